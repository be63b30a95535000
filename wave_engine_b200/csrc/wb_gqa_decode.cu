// wb_gqa_decode.cu -- attention of one new token per sequence over the paged
// key-value cache: for the sequence's query head h over cached positions
// j < len,  out = sum_j softmax_j(scale q . k_j) v_j,  lse = log sum_j
// exp(scale q . k_j); a sequence without positions gives 0 and -inf.
//
// The call reads every cached K and V byte once and does little else with
// it, so HBM bounds it.  All of the batch's keys are one line of 64-key
// units (sequence, key-value head, 8 or 16 query heads, length), which
// the CTAs of one resident wave share out evenly; a CTA's share may begin
// and end inside an item, and the last CTA to finish an item joins its
// pieces in the order of the keys (same bits every run).
//
// One sequence of 131072 positions, 32 heads on 8, head_dim 128, fp16: 89 us,
// 6.0 TB/s, 93% of the measured copy bandwidth (bf16, two products with the
// values: 91 us); 256 sequences of 128 to 4096: int8 189 us, e4m3 192 us, 6.0
// TB/s, bf16 340 us, 6.5 TB/s.  Few keys are bound by latencies (launch,
// lengths and the line 2.5 us, first keys, joins): 32 sequences near 1150, 12
// heads on 4, head_dim 64, e4m3, 14.1 us; one of 257, 7.4 us.  Shares are equal but
// SMs are not equally fast (with 256 sequences they end between 150 and 200
// us); shares cut into six chunks, the later ones dealt out by tickets, all
// ended within 15 us of each other, but 30 us later: a part's start and end
// cost more than the waiting.
//
// In a CTA each of four warps takes every fourth 16-key block, with its own
// running maximum, sum and output, through its own shared-memory ring filled
// by cp.async; the four join at the end of the item.  The products run on
// mma.sync m16n8k16 with the keys (then the dims) as the 16 rows and 8 query
// heads of one key-value head as the columns, so each K and V byte is
// converted once for all of them, and a group of 4 to 8 heads fills the
// columns that it would half fill as rows.  tcgen05 would need every block
// converted to 16 bits and written back to shared memory first, and its 128
// rows would be mostly padding.
//
// Fragments without any transposition of K or V: the dims of q . k and the
// rows of v^T p may be taken in any order as long as both sides use the same
// one, so
//   - lane (r = lane / 4, cc = lane % 4) feeds k . q with whole 16-byte
//     pieces cc, cc + 4, .. of the rows of keys r and r + 8, and
//   - feeds v^T p with piece r of the rows of keys 2cc, 2cc+1, 2cc+8, 2cc+9,
//     two of the piece's dims per product.
// Only the 16 x 8 probabilities change sides (movmatrix).
// 8-bit values become fp16 exactly (e4m3 by cvt, int8 by exponent insertion
// and a subtraction); the K scale multiplies the finished score.  The V
// scale joins the weight, w_j = p_j vscale_j 2^(8 - d2), where d2 is a running
// maximum of its own, of log2 (p_j vscale_j): w_j is then relative to the
// largest weight times scale, so keys with a large probability and small
// values survive the rounding of w to fp16 (as 2^8 w: weights down to
// 2^-32 of the largest count).  With bf16 values p is the sum of two bf16 numbers, each
// with its own product: the tensor pipe has the room, and 8 bits of p would
// cost as much precision as the output's own rounding.  The second one, what
// the first leaves, may be 0 or negative: it meets finite values alone.
#include "wb_gqa.h"

#include <algorithm>
#include <type_traits>

namespace wb {

struct GqaDecodeArgs {
    GqaCacheArgs c;
    const void *q;
    void *out;
    float *lse;
    long long q_ss, q_hs;
    int H;
    float scale;
    unsigned int *counters;  // [grid], zero
    float *part;             // [grid][2] pieces of gqa_piece() floats
};

static constexpr int GD_WARPS = 4, GD_THREADS = GD_WARPS * 32;
static constexpr int GD_UNIT = 64;      // keys per unit: one 16-key block for each warp
static constexpr int GD_ITEM = 2;       // what an item's start and end cost, in units of the line
static constexpr int GD_FEW = 8;        // units per CTA below which items are cut into equal pieces ..
static constexpr int GD_PIECE = 6;      // .. of this many units at least
static constexpr int GD_JOIN = 12;      // pieces that a join loads at a time
static constexpr int GD_SEQS = 256;     // sequences whose lengths a CTA holds in shared memory

enum { GD_NATIVE = 0, GD_INT8 = 1, GD_E4M3 = 2 };

// A key at the running maximum has p = 2^gd_shift, and the maximum is
// followed when p is 2^6 beyond that.  fp16 weights: 2^8, so that 2^-32 of the
// largest still counts.  bf16, which has fp32's range: 2^-26, so that up to
// 2^20 products with the type's largest value add up in fp32 (the definition's
// result is between the values, whatever their size).  8-bit values: 1, as p
// meets their scale before the factor 2^(8 - d2).
__host__ __device__ constexpr float gd_shift(bool quant, bool bf) { return quant ? 0.0f : bf ? -26.0f : 8.0f; }
static constexpr float GD_WEIGHT = 8.0f;    // 8-bit values: the largest weight is 2^8
static constexpr float GD_SMALL = -118.0f;  // least d2: 2^(8 - d2) stays finite
static constexpr float GD_NONE = 3.402823466e38f;  // off before the first key: any finite score replaces it

// CTAs per SM and ring depth: what registers (HDP / 4 NB output and HDP / 8
// NB query registers a thread) and shared memory leave.
template <int KIND, int HDP, int NB>
struct GdConf {
    static constexpr int ESZ = KIND == GD_NATIVE ? 2 : 1;
    static constexpr int RB = HDP * ESZ;  // ring bytes of a row
    static constexpr int CPR = RB / 16;   // 16-byte pieces of a row
    static constexpr int SCALES = KIND == GD_NATIVE ? 0 : 128;
    static constexpr int STAGE = 2 * 16 * RB + SCALES;
    static constexpr int CTAS = NB == 1 ? (HDP == 64 || ESZ == 1 ? 4 : 2) : (HDP == 64 ? 4 : ESZ == 1 ? 3 : 2);
    static constexpr int NST = HDP == 64 ? (ESZ == 2 ? 3 : 5) : (ESZ == 2 ? 3 : NB == 1 ? 3 : 4);
    static constexpr int ROWS = 8 * NB;  // heads of an item
    static constexpr int MST = (ROWS * HDP * 4 + STAGE - 1) / STAGE;  // stages that hold a warp's outputs
    static constexpr int MROWS = ROWS / MST;
    static constexpr int BYTES = GD_WARPS * NST * STAGE;
    static_assert((BYTES + 4096) * CTAS <= 227 * 1024, "shared memory of the resident CTAs");
    static_assert(MROWS * MST == ROWS && MROWS * HDP * 4 <= STAGE && NST - MST >= 1, "the join uses the ring");
};

// Floats of one piece: 16 rows' log2 sum exp, then 16 rows of HDP values
__host__ __device__ constexpr int gqa_piece(int hdp) { return 16 + 16 * hdp; }

template <bool BF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 bytes global -> shared, the bytes past n (0 or 16) as zeros
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void *src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf) {
    uint32_t r;
    if (bf) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// bytes 0, 1 (HI = 0) or 2, 3 (HI = 1) of four 8-bit values as two fp16
template <int KIND, int HI>
__device__ __forceinline__ uint32_t to_f16x2(uint32_t x) {
    uint32_t r;
    if constexpr (KIND == GD_E4M3) {
        const uint16_t h = (uint16_t)(HI ? x >> 16 : x);
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
    } else {
        // 0x6400 | u is 1024 + u; u = value + 128
        const uint32_t m = __byte_perm(x ^ 0x80808080u, 0x64646464u, HI ? 0x4342 : 0x4140);
        const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&m), __half2half2(__ushort_as_half(0x6480)));
        r = *reinterpret_cast<const uint32_t *>(&v);
    }
    return r;
}

// two bf16 magnitudes each: the larger ones, NaN if one is (signs as they come)
__device__ __forceinline__ uint32_t bf16_top(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// over the 8 lanes of one cc
__device__ __forceinline__ float oct_max(float v) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float oct_sum(float v) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// 8 x 8 16-bit values: lane (r, cc) gives row r's columns 2cc, 2cc+1 and gets
// column r's rows 2cc, 2cc+1
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// The sequence's slot and length; a slot or length that does not fit counts
// as empty and is flagged.
__device__ __forceinline__ int gd_len(const GqaCacheArgs &c, int b, int *slot) {
    const int s = c.slots ? c.slots[b] : b;
    const int n = s >= 0 && s < c.n_slots ? c.lens[s] : -1;
    *slot = s;
    if (n < 0 || n > c.max_pages * WB_PAGE) {
        atomicOr(c.dev_err, WB_DERR_BOUNDS);
        return 0;
    }
    return n;
}

// The part of one item that a CTA takes: units ua .. ub-1 of U, keys k0 .. k1-1.
struct GdSeg {
    int b, slot, hk, h0, nrow, ua, ub, U, k0, k1;
    long long first, last;  // the item's first and last position with keys on the line
};

template <class T, int KIND, int HDP, int NB, bool FULL>
__global__ void __launch_bounds__(GD_THREADS, GdConf<KIND, HDP, NB>::CTAS) gqa_decode_kernel(GqaDecodeArgs a) {
    using F = GdConf<KIND, HDP, NB>;
    constexpr bool BF = KIND == GD_NATIVE && __is_same(T, __nv_bfloat16);  // product type
    constexpr bool QUANT = KIND != GD_NATIVE;
    constexpr float SHIFT = gd_shift(QUANT, BF);
    constexpr int NK = HDP / 16;  // products of 16 keys and 8 heads over the dims ..
    constexpr int NV = HDP / 16;  // .. and over the keys
    constexpr int ROWS = F::ROWS;
    constexpr int NST = F::NST, MST = F::MST;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ long long s_scan[GD_WARPS];
    __shared__ long long s_pref, s_at;
    __shared__ GdSeg s_seg[3];
    __shared__ int s_seq;
    __shared__ int s_len[GD_SEQS], s_slot[GD_SEQS];
    __shared__ float s_off[GD_WARPS][16], s_l[GD_WARPS][16], s_f[GD_WARPS][16], s_row[16];
    [[maybe_unused]] __shared__ float s_g[GD_WARPS][16];  // 8-bit values: 2^(d2 - 8)
    __shared__ int s_last, s_stage[GD_WARPS];
    const GqaCacheArgs &c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, cc = lane & 3;
    const int G = a.H / c.Hkv, nch = (G + ROWS - 1) / ROWS, ips = c.Hkv * nch;  // items of a sequence

    gqa_wait();
    // ---- the line of units and this CTA's share s0 .. s1-1
    const int per = (c.n_seq + GD_THREADS - 1) / GD_THREADS;
    long long sum = 0;  // units of a head in this thread's sequences, and how many have any (low 24 bits)
    for (int b = tid * per; b < min((tid + 1) * per, c.n_seq); b++) {
        int slot;
        const int n = gd_len(c, b, &slot);
        if (b < GD_SEQS) {
            s_len[b] = n;
            s_slot[b] = slot;
        }
        sum += (long long)((n + GD_UNIT - 1) / GD_UNIT) << 24 | (n > 0);
    }
    // exclusive sum over the threads, and the total
    auto scan = [&](long long x, long long *all) {
        long long inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) s_scan[warp] = inc;
        __syncthreads();
        long long before = inc - x;
        *all = 0;
#pragma unroll
        for (int w = 0; w < GD_WARPS; w++) {
            if (w < warp) before += s_scan[w];
            *all += s_scan[w];
        }
        return before;
    };
    long long total;
    const long long sums = scan(sum, &total);
    auto length = [&](int b, int *slot) {
        if (b >= GD_SEQS) return gd_len(c, b, slot);
        *slot = s_slot[b];
        return s_len[b];
    };
    for (int b = blockIdx.x; b < c.n_seq; b += gridDim.x) {  // sequences without positions
        int slot;
        if (length(b, &slot)) continue;
        T *op = (T *)a.out + (long long)b * a.H * c.hd;
        for (int i = tid; i < a.H * c.hd; i += GD_THREADS) op[i] = from_f<T>(0.0f);
        for (int h = tid; a.lse && h < a.H; h += GD_THREADS) a.lse[(long long)b * a.H + h] = -INFINITY;
    }
    const long long units = (total >> 24) * ips, items = (total & 0xffffff) * ips;
    // Few units for the CTAs there are: every item in equal pieces of P
    // units, one for each CTA (a piece that ends with its item has one join
    // less; 32 sequences, 12 heads on 4, at 4 units a CTA 13.9 us, 15.4 in
    // equal shares; at 8 units 18.3, 20.6; at 15 units 25.2, 24.6).  P is at
    // least 6: a shorter piece saves less than its join costs (one sequence of
    // 257: 7.5 us, 8.7 with 3, 7.6 with 12; 4 near 1150: 11.5, 10.3, 14.1; 32:
    // 14.1, 14.1, 17.3).  Else positions of one unit, with W more for an
    // item's start and end, in equal shares (256 sequences of 128 to 4096: 189
    // us, 204 without W).
    int P = 1, W = GD_ITEM;
    if (2 * items <= gridDim.x && units <= (long long)gridDim.x * GD_FEW) {
        W = 0;
        P = max(GD_PIECE, (int)((units + (gridDim.x - items) - 1) / (gridDim.x - items)));
    }
    auto item_len = [&](int n) { return n == 0 ? 0 : ((n + GD_UNIT - 1) / GD_UNIT + W + P - 1) / P; };

    long long mine = ((sum >> 24) + W * (sum & 0xffffff)) * ips, before = ((sums >> 24) + W * (sums & 0xffffff)) * ips;
    if (W == 0) {
        mine = 0;
        for (int b = tid * per; b < min((tid + 1) * per, c.n_seq); b++) {
            int slot;
            mine += (long long)item_len(length(b, &slot)) * ips;
        }
        __syncthreads();
        before = scan(mine, &total);
    } else total = units + W * items;
    const long long grid = min((long long)gridDim.x, total);
    if ((long long)blockIdx.x >= grid) return;
    const long long s0 = gqa_quotient(blockIdx.x * total, grid), s1 = gqa_quotient((blockIdx.x + 1) * total, grid);

    // The share's parts with keys, one after another, U = 0 past its end.  One
    // thread finds part x + 2 while part x is joined.
    auto next_seg = [&](GdSeg &g) {
        int nb = s_seq;
        long long pref = s_pref, u = s_at;
        g.U = 0;
        while (u < s1) {
            int slot;
            const int len = length(nb, &slot);
            const int il = item_len(len), U = (len + GD_UNIT - 1) / GD_UNIT;
            if (u >= pref + (long long)il * ips) {
                pref += (long long)il * ips;
                nb++;
                continue;
            }
            const long long rel = u - pref;
            const int item = (int)gqa_quotient(rel, il), o0 = (int)(rel - (long long)item * il);
            const int o1 = (int)min((long long)il, o0 + (s1 - u));
            u += o1 - o0;
            if (o1 * P <= W) continue;
            g.b = nb;
            g.slot = slot;
            g.hk = item / nch;
            const int hc = item - g.hk * nch;
            g.h0 = g.hk * G + hc * ROWS;
            g.nrow = min(ROWS, G - hc * ROWS);
            g.U = U;
            g.ua = max(0, o0 * P - W);
            g.ub = min(U, o1 * P - W);
            g.k0 = g.ua * GD_UNIT;
            g.k1 = min(g.ub * GD_UNIT, len);
            g.first = pref + (long long)item * il + W;
            g.last = pref + (long long)item * il + il - 1;
            break;
        }
        s_seq = nb;
        s_pref = pref;
        s_at = u;
    };
    if (s0 >= before && s0 < before + mine) {  // in this thread's sequences
        s_seq = tid * per;
        s_pref = before;
        s_at = s0;
        next_seg(s_seg[0]);
        next_seg(s_seg[1]);
    }
    __syncthreads();

    uint8_t *ring = sm + warp * (NST * F::STAGE);
    // FULL: rows of HDP values, so that a block's offsets are constants
    const int rowb = FULL ? F::RB : c.row * F::ESZ;
    // This lane's pieces of a block: ch of rows lr, lr + STEP, ..  Piece
    // positions within each 128 bytes of the ring are permuted, K's by row
    // parity and V's by row pair, so that the fragments' reads touch every
    // bank once; all of a lane's places are one base and constants.
    constexpr int STEP = 32 / F::CPR;
    const int ch = lane % F::CPR, lr = lane / F::CPR;
    const bool col = FULL || ch * 16 < rowb;
    const uint32_t src0 = lr * rowb + ch * 16;
    const uint32_t ring0 = ptx::smem_u32(ring);
    auto place = [&](int rr, int ch, int sw) {
        const int pos = (F::RB == 64 ? (rr & 1) * 4 : 0) + ch;
        return (uint32_t)((rr * F::RB / 128 + (F::RB == 256 ? ch / 8 : 0)) * 128 + (((pos & 7) ^ sw) << 4));
    };
    const uint32_t kdst = place(lr, ch, F::RB == 64 ? 0 : (lr & 1) << 2);  // row lr + x STEP: + 512 x
    const uint32_t vdst = 16 * F::RB + place(lr, ch, ((lr >> 1) & 3) << 1);  // and ^ v_flip(x)
    auto v_flip = [](int x) { return (uint32_t)(F::RB == 64 ? 0 : F::RB == 128 ? (x & 1) * 64 : (x & 3) * 32); };
    // reads: piece cc of row r, and of rows 2cc (piece r) for the values
    const uint32_t krd = place(r, cc, F::RB == 64 ? 0 : (r & 1) << 2);
    const uint32_t vrd = 16 * F::RB + (F::RB == 64 ? place(2 * cc, r >> 1, cc << 1) + (r & 1) * 8 : place(2 * cc, r, cc << 1));

    // ---- loads of a part's blocks: this warp's are keys k0 + 16 (warp + 4 i)
    int pbase = 0, pid = -1;  // page ids of pages pbase + lane of the part
    auto pages_of = [&](const GdSeg &g, int p) {
        return p + lane <= (g.k1 - 1) >> WB_PAGE_SHIFT ? c.table[(long long)g.slot * c.max_pages + p + lane] : -1;
    };
    auto key_of = [&](int k0, int i) { return k0 + 16 * (warp + GD_WARPS * i); };
    auto blocks_of = [&](const GdSeg &g) { return (((g.k1 - g.k0 + 15) >> 4) - warp + GD_WARPS - 1) / GD_WARPS; };
    auto issue = [&](const GdSeg &g, int key0, int kend, int stage) {
        const int p = key0 >> WB_PAGE_SHIFT;
        if (p >= pbase + 32) {
            pbase = p;
            pid = pages_of(g, p);
        }
        const int pg = __shfl_sync(0xffffffffu, pid, p - pbase);
        const bool ok = pg >= 0 && pg < c.n_pages;
        const long long row0 = ok ? ((long long)pg * c.Hkv + g.hk) * WB_PAGE + (key0 & (WB_PAGE - 1)) : 0;
        const uint32_t st = ring0 + stage * F::STAGE;
        const uint8_t *kp = (const uint8_t *)c.k_pages + row0 * rowb + src0, *vp = (const uint8_t *)c.v_pages + row0 * rowb + src0;
        if (ok && key0 + 16 <= kend) {
#pragma unroll
            for (int x = 0; x < F::CPR / 2; x++) {
                const uint32_t kd = st + kdst + 512 * x, vd = st + (vdst ^ v_flip(x)) + 512 * x;
                if (FULL) {
                    cp_async16(kd, kp + x * STEP * F::RB);
                    cp_async16(vd, vp + x * STEP * F::RB);
                } else {
                    cp_async16_or_zero(kd, col ? kp + x * STEP * rowb : kp, col ? 16 : 0);
                    cp_async16_or_zero(vd, col ? vp + x * STEP * rowb : vp, col ? 16 : 0);
                }
            }
        } else {
#pragma unroll 1
            for (int x = 0; x < F::CPR / 2; x++) {
                const int n = ok && col && key0 + lr + x * STEP < kend ? 16 : 0;
                const long long o = n ? (long long)x * STEP * rowb : -(long long)src0;
                cp_async16_or_zero(st + kdst + 512 * x, kp + o, n);
                cp_async16_or_zero(st + (vdst ^ v_flip(x)) + 512 * x, vp + o, n);
            }
        }
        if (QUANT && lane < 8) {
            const float *sp = (lane < 4 ? c.k_scale : c.v_scale) + row0 + (lane & 3) * 4;
            cp_async16_or_zero(st + 32 * F::RB + lane * 16, sp, ok ? 16 : 0);
        }
        return ok;
    };
    // a part's queries as loaded: head r of each eight, dims in the order of K's pieces
    const bool q8 = ((a.q_ss | a.q_hs | c.hd) & 3) == 0 && (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
    auto q_dim = [&](int t) { return F::ESZ == 1 ? 16 * (cc + 4 * (t / 4)) + 4 * (t % 4) : 8 * (cc + 4 * (t / 2)) + 4 * (t % 2); };
    uint32_t qf[NB][NK][2];
    auto load_q = [&](const GdSeg &g) {
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            const int row = r + 8 * nb;
            const uint16_t *qp = (const uint16_t *)a.q + g.b * a.q_ss + (long long)(g.h0 + row) * a.q_hs;
#pragma unroll
            for (int t = 0; t < NK; t++) {
                const int d0 = q_dim(t);
                uint2 w = make_uint2(0, 0);
                if (row < g.nrow) {
                    if (q8) {
                        if (d0 < c.hd) w = *reinterpret_cast<const uint2 *>(qp + d0);
                    } else {
                        uint32_t e[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) e[i] = d0 + i < c.hd ? qp[d0 + i] : 0;
                        w = make_uint2(e[0] | e[1] << 16, e[2] | e[3] << 16);
                    }
                }
                qf[nb][t][0] = w.x;
                qf[nb][t][1] = w.y;
            }
        }
    };

    if (s_seg[0].U == 0) return;
    load_q(s_seg[0]);
    pbase = s_seg[0].k0 >> WB_PAGE_SHIFT;
    pid = pages_of(s_seg[0], pbase);
    int stage = 0;  // ring stage of the part's first block
    int cnt = blocks_of(s_seg[0]);
    uint32_t okbits = 0;  // bit of a stage: its block's page is mapped
#pragma unroll
    for (int i = 0; i < NST - MST; i++) {
        if (i < cnt && issue(s_seg[0], key_of(s_seg[0].k0, i), s_seg[0].k1, i)) okbits |= 1u << i;
        ptx::cp_async_commit();
    }
    for (int part = 0;; part++) {
        const GdSeg &g = s_seg[part % 3], &h = s_seg[(part + 1) % 3];
        // ---- the rest of the first loads (the first NST - MST are under way)
#pragma unroll
        for (int i = NST - MST; i < NST - 1; i++) {
            const int sg = (stage + i) % NST;
            okbits &= ~(1u << sg);
            if (i < cnt && issue(g, key_of(g.k0, i), g.k1, sg)) okbits |= 1u << sg;
            ptx::cp_async_commit();
        }
        // the next part's page ids, long before they are needed
        const bool more = h.U != 0;
        const int hpid = more ? pages_of(h, h.k0 >> WB_PAGE_SHIFT) : -1;

        float fac[NB][2];  // score factors of heads 2cc, 2cc+1, log2 e included
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            float f = a.scale * 1.4426950408889634f;
            if (QUANT && !__is_same(T, __half)) {
                // bf16 queries meet fp16 keys: divided by a power of two so
                // that the head's largest is in [1, 2) (exact down to 2^-17
                // of it, 0 below 2^-25)
                uint32_t top = 0;
#pragma unroll
                for (int t = 0; t < NK; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        top = max(top, max((qf[nb][t][e] << 16) & 0x7fffffffu, qf[nb][t][e] & 0x7fff0000u));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e2 = min(max((int)(top >> 23), 1), 253);
                const float down = __uint_as_float((uint32_t)(254 - e2) << 23);
                f *= __uint_as_float((uint32_t)e2 << 23);
#pragma unroll
                for (int t = 0; t < NK; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t x = qf[nb][t][e];
                        qf[nb][t][e] = pack2(__uint_as_float(x << 16) * down, __uint_as_float(x & 0xffff0000u) * down, false);
                    }
            }
            fac[nb][0] = __shfl_sync(0xffffffffu, f, 8 * cc);
            fac[nb][1] = __shfl_sync(0xffffffffu, f, 8 * cc + 4);
        }

        // acc[nb][j]: dims of piece r (two per product), heads 2cc, 2cc+1
        float acc[NB][NV][4] = {};
        // p = 2^(score + off), off = SHIFT - maximum; d2, e2 = 2^(8 - d2): 8-bit values
        float l[NB][2], off[NB][2], d2[NB][2], e2[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                l[nb][e] = 0.0f;
                off[nb][e] = GD_NONE;
                d2[nb][e] = GD_SMALL;
                e2[nb][e] = ex2(GD_WEIGHT - GD_SMALL);
            }
        bool unmapped = false;

        auto block = [&](const uint8_t *st, int n, auto tail) {
            constexpr bool TAIL = decltype(tail)::value;
            // s[nb]: scores of keys r (heads 2cc, 2cc+1) and r + 8 (the same)
            float s[NB][4] = {};
#pragma unroll
            for (int x = 0; x < F::CPR / 4; x++) {
                const uint8_t *kr = st + (krd ^ (x & 1) * 64) + (x >> 1) * 128;
                const uint4 w0 = *reinterpret_cast<const uint4 *>(kr), w1 = *reinterpret_cast<const uint4 *>(kr + 8 * F::RB);
                const uint32_t k0[4] = {w0.x, w0.y, w0.z, w0.w}, k1[4] = {w1.x, w1.y, w1.z, w1.w};
                if constexpr (QUANT) {
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const uint32_t kf[4] = {to_f16x2<KIND, 0>(k0[t]), to_f16x2<KIND, 0>(k1[t]),
                                                to_f16x2<KIND, 1>(k0[t]), to_f16x2<KIND, 1>(k1[t])};
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) mma16816<BF>(s[nb], kf, qf[nb][4 * x + t][0], qf[nb][4 * x + t][1]);
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const uint32_t kf[4] = {k0[2 * t], k1[2 * t], k0[2 * t + 1], k1[2 * t + 1]};
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) mma16816<BF>(s[nb], kf, qf[nb][2 * x + t][0], qf[nb][2 * x + t][1]);
                    }
                }
            }
            float vs[2] = {1.0f, 1.0f};
            if (QUANT) {
                const float *sc = reinterpret_cast<const float *>(st + 32 * F::RB) + r;
                vs[0] = sc[16];
                vs[1] = sc[24];
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[nb][i] *= sc[8 * (i >> 1)];
            }
            // Scores as rounded products: their difference from the largest is
            // then exact, however large they are (the type's lowest value as
            // a mask); as one operation, fac s + off, it would be off by up to
            // half an ulp of the largest.
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[nb][i] = __fmul_rn(s[nb][i], fac[nb][i & 1]);
            // weights of the first n keys (all 16 unless TAIL)
            float pr[NB][4];
            uint32_t pf[NB][2];  // fp16 or bf16: key r, key r + 8
            auto weigh = [&]() {
                float most = 0.0f;
                __half2 top = __half2half2(__ushort_as_half(0));
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        float w[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float &p = pr[nb][2 * g + e];
                            p = ex2(__fadd_rn(s[nb][2 * g + e], off[nb][e]));
                            w[e] = QUANT ? p * vs[g] * e2[nb][e] : p;  // in this order 0 stays 0
                            if (TAIL && r + 8 * g >= n) p = w[e] = 0.0f;
                        }
                        pf[nb][g] = pack2(w[0], w[1], BF);
                        if (!BF) top = __hmax2(top, *reinterpret_cast<const __half2 *>(&pf[nb][g]));
                        most = fmaxf(most, fmaxf(pr[nb][2 * g], pr[nb][2 * g + 1]));  // a NaN hides no other head's
                    }
                }
                // p 2^6 beyond its place, or an fp16 weight above 2^14
                bool far = BF ? most > 9.5367431640625e-7f : QUANT && most > 64.0f;
                if (!BF) far |= __hgt2_mask(top, __half2half2(__ushort_as_half(0x7400))) != 0;
                return far;
            };
            // The references off, d2 stay until then; then they follow the maxima.
            if (__any_sync(0xffffffffu, weigh())) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    float f2[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float mx = -INFINITY, mx2 = GD_SMALL;
#pragma unroll
                        for (int g = 0; g < 2; g++)
                            if (!TAIL || r + 8 * g < n) mx = fmaxf(mx, s[nb][2 * g + e]);
                        mx = oct_max(mx);
                        // SHIFT - mx would be rounded from 2^24 on
                        const float to = fminf(off[nb][e], (fabsf(mx) < 16777216.0f ? SHIFT : 0.0f) - mx), d = to - off[nb][e];
                        l[nb][e] *= ex2(d);
                        off[nb][e] = to;
                        f2[e] = ex2(d);
                        if (QUANT) {
                            // a scale of 0 (a caller's own pages) counts as 2^-118
#pragma unroll
                            for (int g = 0; g < 2; g++)
                                if (!TAIL || r + 8 * g < n) mx2 = fmaxf(mx2, s[nb][2 * g + e] + to + lg2(vs[g]));
                            const float to2 = fmaxf(d2[nb][e] + d, oct_max(mx2));
                            f2[e] = ex2(d + d2[nb][e] - to2);
                            d2[nb][e] = to2;
                            e2[nb][e] = ex2(GD_WEIGHT - to2);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < NV; j++) {
                        acc[nb][j][0] *= f2[0];
                        acc[nb][j][1] *= f2[1];
                        acc[nb][j][2] *= f2[0];
                        acc[nb][j][3] *= f2[1];
                    }
                }
                weigh();
            }
            uint32_t pl[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                l[nb][0] += pr[nb][0] + pr[nb][2];
                l[nb][1] += pr[nb][1] + pr[nb][3];
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    if (BF) {
                        const uint32_t x = pf[nb][g];
                        pl[nb][g] = transposed(pack2(pr[nb][2 * g] - __uint_as_float(x << 16),
                                                     pr[nb][2 * g + 1] - __uint_as_float(x & 0xffff0000u), BF));
                    }
                    pf[nb][g] = transposed(pf[nb][g]);
                }
            }
            auto product = [&](int j, const uint32_t (&p)[NB][2], uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3) {
                const uint32_t vf[4] = {v0, v1, v2, v3};
#pragma unroll
                for (int nb = 0; nb < NB; nb++) mma16816<BF>(acc[nb][j], vf, p[nb][0], p[nb][1]);
            };

            // values: piece r of rows 2cc, 2cc+1, 2cc+8, 2cc+9
            [[maybe_unused]] const uint8_t *sv = st + vrd;
            if constexpr (F::ESZ == 2) {
#pragma unroll
                for (int x = 0; x < HDP / 64; x++) {
                    uint32_t w[4][4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(sv + ((e & 1) + 8 * (e >> 1)) * F::RB + x * 128);
                        w[e][0] = v.x; w[e][1] = v.y; w[e][2] = v.z; w[e][3] = v.w;
                    }
                    auto dims = [&](int d, const uint32_t (&p)[NB][2]) {
                        product(4 * x + d, p, __byte_perm(w[0][d], w[1][d], 0x5410), __byte_perm(w[0][d], w[1][d], 0x7632),
                                __byte_perm(w[2][d], w[3][d], 0x5410), __byte_perm(w[2][d], w[3][d], 0x7632));
                    };
                    if constexpr (!BF) {
#pragma unroll
                        for (int d = 0; d < 4; d++) dims(d, pf);
                    } else {
                        // The second part of p may be 0 or negative, which would
                        // turn an infinite value into a NaN: it gets the values
                        // without what is not finite.
                        uint32_t top = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++)
#pragma unroll
                            for (int d = 0; d < 4; d++) top = bf16_top(top, w[e][d]);
                        const bool bad = (top & 0x7f80u) == 0x7f80u || (top & 0x7f800000u) == 0x7f800000u;
                        if (!__any_sync(0xffffffffu, bad)) {
#pragma unroll
                            for (int d = 0; d < 4; d++) {
                                dims(d, pf);
                                dims(d, pl);
                            }
                        } else {
#pragma unroll
                            for (int d = 0; d < 4; d++) dims(d, pf);
#pragma unroll
                            for (int e = 0; e < 4; e++)
#pragma unroll
                                for (int d = 0; d < 4; d++) {
                                    uint32_t &y = w[e][d];
                                    if ((y & 0x7f80u) == 0x7f80u) y &= 0xffff0000u;
                                    if ((y & 0x7f800000u) == 0x7f800000u) y &= 0xffffu;
                                }
#pragma unroll
                            for (int d = 0; d < 4; d++) dims(d, pl);
                        }
                    }
                }
            } else {
                uint32_t w[4][HDP / 32];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if constexpr (HDP == 128) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(sv + ((e & 1) + 8 * (e >> 1)) * 128);
                        w[e][0] = v.x; w[e][1] = v.y; w[e][2] = v.z; w[e][3] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2 *>(st + (vrd ^ (e & 1) * 64) + (e >> 1) * 512);
                        w[e][0] = v.x; w[e][1] = v.y;
                    }
                }
#pragma unroll
                for (int d = 0; d < HDP / 32; d++) {
                    // (key a byte, key b byte) pairs of dims 4d, 4d+1 and 4d+2, 4d+3
                    const uint32_t a01 = __byte_perm(w[0][d], w[1][d], 0x5140), a23 = __byte_perm(w[0][d], w[1][d], 0x7362);
                    const uint32_t b01 = __byte_perm(w[2][d], w[3][d], 0x5140), b23 = __byte_perm(w[2][d], w[3][d], 0x7362);
                    product(2 * d, pf, to_f16x2<KIND, 0>(a01), to_f16x2<KIND, 1>(a01), to_f16x2<KIND, 0>(b01), to_f16x2<KIND, 1>(b01));
                    product(2 * d + 1, pf, to_f16x2<KIND, 0>(a23), to_f16x2<KIND, 1>(a23), to_f16x2<KIND, 0>(b23), to_f16x2<KIND, 1>(b23));
                }
            }
        };

        int stg = stage, nxs = (stage + NST - 1) % NST;
        const int kbeg = g.k0, kend = g.k1;
        for (int i = 0; i < cnt; i++) {
            ptx::cp_async_wait<NST - 2>();
            __syncwarp();
            const bool ok = (okbits >> stg) & 1;
            okbits &= ~(1u << nxs);
            if (i + NST - 1 < cnt && issue(g, key_of(kbeg, i + NST - 1), kend, nxs)) okbits |= 1u << nxs;
            ptx::cp_async_commit();
            const uint8_t *st = ring + stg * F::STAGE;
            const int key0 = key_of(kbeg, i);
            nxs = stg;
            if (++stg == NST) stg = 0;
            if (ok && key0 + 16 <= kend) {
                block(st, 16, std::false_type{});
            } else {
                unmapped |= !ok;
                block(st, ok ? kend - key0 : 0, std::true_type{});
            }
        }
        // every block of the part has been read: the next part's first loads
        // and queries go out before this one's join
        stage = stg;
        ptx::cp_async_wait<0>();
        int hcnt = 0;
        if (more) {
            hcnt = blocks_of(h);
            pbase = h.k0 >> WB_PAGE_SHIFT;
            pid = hpid;
            okbits = 0;
#pragma unroll
            for (int i = 0; i < NST - MST; i++) {
                const int sg = (stage + i) % NST;
                if (i < hcnt && issue(h, key_of(h.k0, i), h.k1, sg)) okbits |= 1u << sg;
                ptx::cp_async_commit();
            }
            load_q(h);
        }
        if (unmapped && lane == 0) atomicOr(c.dev_err, WB_DERR_BOUNDS);

        // ---- the four warps' outputs into one, through the MST ring stages
        // that hold none of the next part's blocks
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                l[nb][e] = oct_sum(l[nb][e]);
                if (r == 0) {
                    s_off[warp][8 * nb + 2 * cc + e] = off[nb][e];
                    s_l[warp][8 * nb + 2 * cc + e] = l[nb][e];
                    if (QUANT) s_g[warp][8 * nb + 2 * cc + e] = ex2(d2[nb][e] - GD_WEIGHT);
                }
            }
        if (lane == 0) s_stage[warp] = stage;
        auto row_at = [&](int w, int stage_w, int row) {
            const int sg = (stage_w + NST - F::MST + row / F::MROWS) % NST;
            return reinterpret_cast<float *>(sm + (w * NST + sg) * F::STAGE) + row % F::MROWS * HDP;
        };
        __syncwarp();
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int row = 8 * nb + 2 * cc + e;
                if (row < g.nrow) {
                    float *o = row_at(warp, stage, row);
#pragma unroll
                    for (int j = 0; j < NV; j++) {
                        // product j holds dims 2j, 2j+1 of the lane's piece(s)
                        const int d = F::ESZ == 2 ? 64 * (j >> 2) + r * 8 + 2 * (j & 3) : r * (HDP / 8) + 2 * j;
                        *reinterpret_cast<float2 *>(o + d) = make_float2(acc[nb][j][e], acc[nb][j][2 + e]);
                    }
                }
            }
        __syncthreads();
        if (tid == GD_THREADS - 1) next_seg(s_seg[(part + 2) % 3]);
        if (tid < ROWS) {
            float to = GD_NONE, L = 0.0f;
            for (int w = 0; w < GD_WARPS; w++) to = fminf(to, s_off[w][tid]);
            for (int w = 0; w < GD_WARPS; w++) L += s_l[w][tid] * ex2(to - s_off[w][tid]);
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            for (int w = 0; w < GD_WARPS; w++) s_f[w][tid] = ex2(to - s_off[w][tid]) * inv;
            s_row[tid] = L == 0.0f ? -INFINITY : log2f(L) - to;  // log2 sum exp
        }
        __syncthreads();
        const bool whole = g.ua == 0 && g.ub == g.U;
        float *piece = a.part + ((long long)blockIdx.x * 2 + (g.ua == 0 ? 1 : 0)) * gqa_piece(HDP);
        const long long row_out = (long long)g.b * a.H + g.h0;
        auto put = [&](int row, int d, const float (&o)[4]) {
            T *to = (T *)a.out + (row_out + row) * c.hd + d;
#pragma unroll
            for (int y = 0; y < 4; y++)
                if (d + y < c.hd) to[y] = from_f<T>(o[y]);
        };
        for (int i = tid; i < g.nrow * (HDP / 4); i += GD_THREADS) {
            const int row = i / (HDP / 4), d = i % (HDP / 4) * 4;
            float o[4] = {};
#pragma unroll
            for (int w = 0; w < GD_WARPS; w++) {
                const float4 v = *reinterpret_cast<const float4 *>(row_at(w, s_stage[w], row) + d);
                const float f = s_f[w][row], g8 = QUANT ? s_g[w][row] : 1.0f;
                o[0] += v.x * f * g8;
                o[1] += v.y * f * g8;
                o[2] += v.z * f * g8;
                o[3] += v.w * f * g8;
            }
            if (whole) put(row, d, o);
            else __stcg(reinterpret_cast<float4 *>(piece + 16 + 4 * i), make_float4(o[0], o[1], o[2], o[3]));
        }
        if (tid < g.nrow) {
            if (!whole) __stcg(piece + tid, s_row[tid]);
            else if (a.lse) a.lse[row_out + tid] = s_row[tid] * 0.6931471805599453f;
        }
        if (!whole) {
            // ---- the item's last CTA joins the pieces
            const int c0 = (int)gqa_quotient((g.first + 1) * grid - 1, total), c1 = (int)gqa_quotient((g.last + 1) * grid - 1, total);
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicAdd(a.counters + c0, 1) == (unsigned)(c1 - c0);
            __syncthreads();
            if (s_last) {
                __threadfence();
                if (tid == 0) a.counters[c0] = 0;
                const int n = c1 - c0 + 1;
                // piece x of the item: the first CTA's second slot, the others' first
                auto at = [&](int x) { return a.part + ((long long)(c0 + x) * 2 + (x == 0 ? 1 : 0)) * gqa_piece(HDP); };
                // four values a thread, GD_JOIN pieces in one round of loads
                for (int i = tid; i < g.nrow * (HDP / 4); i += GD_THREADS) {
                    const int row = i / (HDP / 4), d = i % (HDP / 4) * 4;
                    float M = -INFINITY, L = 0.0f, o[4] = {};
                    for (int x0 = 0; x0 < n; x0 += GD_JOIN) {
                        float z[GD_JOIN];
                        float4 v[GD_JOIN];
#pragma unroll
                        for (int x = 0; x < GD_JOIN; x++) {
                            z[x] = -INFINITY;
                            v[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (x0 + x < n) {
                                z[x] = __ldcg(at(x0 + x) + row);
                                v[x] = __ldcg(reinterpret_cast<const float4 *>(at(x0 + x) + 16 + 4 * i));
                            }
                        }
                        float top = M;
#pragma unroll
                        for (int x = 0; x < GD_JOIN; x++) top = fmaxf(top, z[x]);
                        const float ref = top == -INFINITY ? 0.0f : top, f = ex2(M - ref);
                        M = top;
                        L *= f;
#pragma unroll
                        for (int y = 0; y < 4; y++) o[y] *= f;
#pragma unroll
                        for (int x = 0; x < GD_JOIN; x++) {
                            const float w = ex2(z[x] - ref);
                            L += w;
                            o[0] += v[x].x * w;
                            o[1] += v[x].y * w;
                            o[2] += v[x].z * w;
                            o[3] += v[x].w * w;
                        }
                    }
#pragma unroll
                    for (int y = 0; y < 4; y++) o[y] = L == 0.0f ? 0.0f : o[y] / L;
                    put(row, d, o);
                    if (d == 0 && a.lse) a.lse[row_out + row] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
                }
            }
        }
        if (!more) return;
        __syncthreads();  // the join's stages are free
        cnt = hcnt;
    }
}

static int gd_grid(const GqaCacheArgs &c, int H, int sm_count, int ctas) {
    const int G = H / c.Hkv;
    const long long most = (long long)c.n_seq * c.Hkv * ((G + 15) / 16) * (c.max_pages * (WB_PAGE / GD_UNIT) + GD_ITEM);
    return (int)std::max(1LL, std::min(most, (long long)std::min(sm_count, 148) * ctas));
}

size_t gqa_decode_scratch(const GqaCacheArgs &c, int H, int sm_count) {
    return (size_t)gd_grid(c, H, sm_count, 4) * 2 * gqa_piece(c.hd <= 64 ? 64 : 128) * sizeof(float);
}

template <class T, int KIND, int HDP, int NB, bool FULL>
static int gd_launch_as(const GqaDecodeArgs &a, int sm_count, cudaStream_t st, std::string *msg) {
    using F = GdConf<KIND, HDP, NB>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t set = gqa_smem_limit(gqa_decode_kernel<T, KIND, HDP, NB, FULL>, F::BYTES, done);
    if (set != cudaSuccess) {
        *msg = std::string("decode kernel attributes: ") + cudaGetErrorString(set);
        return WB_ECUDA;
    }
    ProfScope ps("gqa_decode", st);
    gqa_launch(gqa_decode_kernel<T, KIND, HDP, NB, FULL>, gd_grid(a.c, a.H, sm_count, F::CTAS), GD_THREADS, F::BYTES, st, a);
    return WB_OK;
}

template <class T, int KIND, int HDP>
static int gd_launch(const GqaDecodeArgs &a, int sm_count, cudaStream_t st, std::string *msg) {
    // up to 8 heads on a key-value head: one product's 8 columns; more: two
    // (256 sequences of int8: two for 4 heads 234 us instead of 190, for 8
    // heads 241 instead of 195; 9 heads as two items of one each 372 instead
    // of 246, 16 heads 379 instead of 259)
    const bool full = a.c.row == HDP;
    if (a.H / a.c.Hkv <= 8)
        return full ? gd_launch_as<T, KIND, HDP, 1, true>(a, sm_count, st, msg)
                    : gd_launch_as<T, KIND, HDP, 1, false>(a, sm_count, st, msg);
    return full ? gd_launch_as<T, KIND, HDP, 2, true>(a, sm_count, st, msg)
                : gd_launch_as<T, KIND, HDP, 2, false>(a, sm_count, st, msg);
}

int launch_gqa_decode(const GqaCacheArgs &c, int dtype, int H, const void *q, long long q_ss, long long q_hs,
                      float scale, void *out, float *lse, unsigned int *counters, void *scratch, int sm_count,
                      cudaStream_t st, std::string *msg) {
    GqaDecodeArgs a{c, q, out, lse, q_ss, q_hs, H, scale, counters, (float *)scratch};
    auto by_store = [&](auto t) {
        using T = decltype(t);
        // rows of up to 64 in 64 columns (in 128: 17.8 us instead of 14.1, 32
        // sequences near 1150)
        const bool wide = c.hd > 64;
        if (c.store == WB_INT8)
            return wide ? gd_launch<T, GD_INT8, 128>(a, sm_count, st, msg) : gd_launch<T, GD_INT8, 64>(a, sm_count, st, msg);
        if (c.store == WB_E4M3)
            return wide ? gd_launch<T, GD_E4M3, 128>(a, sm_count, st, msg) : gd_launch<T, GD_E4M3, 64>(a, sm_count, st, msg);
        return wide ? gd_launch<T, GD_NATIVE, 128>(a, sm_count, st, msg) : gd_launch<T, GD_NATIVE, 64>(a, sm_count, st, msg);
    };
    return dtype == WB_BF16 ? by_store(__nv_bfloat16{}) : by_store(__half{});
}

}  // namespace wb
