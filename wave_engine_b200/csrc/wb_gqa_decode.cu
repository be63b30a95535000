// wb_gqa_decode.cu -- attention of one new token per sequence over the paged
// key-value cache: for the sequence's query head h over cached positions
// j < len,  out = sum_j softmax_j(scale q . k_j) v_j,  lse = log sum_j
// exp(scale q . k_j); a sequence without positions gives 0 and -inf.
//
// The call reads every cached K and V byte once and does little else with
// it, so HBM bounds it.  All of the batch's keys are one line of 64-key
// units (sequence, key-value head, group of 16 query heads, length), which
// the CTAs of one resident wave share out evenly; a CTA's share may begin
// and end inside an item, and the last CTA to finish an item joins its
// pieces in the order of the keys (same bits every run).
//
// In a CTA each of four warps takes every fourth 16-key block, with its own
// running maximum, sum and output, through its own shared-memory ring filled
// by cp.async; the four join at the end of the item.  The products run on
// mma.sync m16n8k16 with the (up to 16) query heads of one key-value head as
// the rows: each K and V byte is converted once for all of them.  tcgen05
// would need every block converted to 16 bits and written back to shared
// memory first, and its 128 rows would be mostly padding.
//
// Fragments without any transposition: the dims of q . k and the columns of
// p v may be taken in any order as long as both sides use the same one, so
//   - lane (r = lane / 4, c = lane % 4) feeds q . k with whole 16-byte
//     pieces c, c + 4, .. of key r's row (and of key r + 8's), and
//   - feeds p v with piece r of the rows of keys 2c, 2c+1, 2c+8, 2c+9, one
//     product per dim of the piece -- the keys whose probabilities the lane
//     already holds.
// 8-bit values become fp16 exactly (e4m3 by cvt, int8 by exponent insertion
// and a subtraction); the K scale multiplies the finished score.  The V
// scale s_j joins the exponent, w_j = exp2(s_j + log2 vscale_j - m2), with
// its own running maximum m2: w_j is then relative to the largest weight
// times scale, so keys with a large probability and small values survive
// the rounding of w to fp16 (scaled by 2^8: weights down to 2^-32 of the
// largest count).  With bf16 values p is the sum of two bf16 numbers, each
// with its own product: the tensor pipe has the room, and 8 bits of p would
// cost as much precision as the output's own rounding.
#include "wb_gqa.h"
#include "wb_ptx.cuh"

#include <algorithm>

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
static constexpr float GD_SHIFT = 8.0f; // weights are kept as 2^8 exp2(s - m): see above
static constexpr float GD_LAZY = 6.0f;  // m follows the maximum once it is this far behind (2^14 < 65504)

enum { GD_NATIVE = 0, GD_INT8 = 1, GD_E4M3 = 2 };

// CTAs per SM and ring depth: three CTAs of 168 registers at 128 columns
// (64 output + 32 query registers a thread), four at 64; the ring takes what
// shared memory leaves.
template <int KIND, int HDP>
struct GdConf {
    static constexpr int ESZ = KIND == GD_NATIVE ? 2 : 1;
    static constexpr int RB = HDP * ESZ;  // ring bytes of a row
    static constexpr int CPR = RB / 16;   // 16-byte pieces of a row
    static constexpr int SCALES = KIND == GD_NATIVE ? 0 : 128;
    static constexpr int STAGE = 2 * 16 * RB + SCALES;
    static constexpr int CTAS = HDP == 64 ? 4 : (ESZ == 2 ? 2 : 3);
    static constexpr int NST = HDP == 64 ? (ESZ == 2 ? 3 : 6) : (ESZ == 2 ? 3 : 4);
    static constexpr int BYTES = GD_WARPS * NST * STAGE;
    static_assert(BYTES * CTAS <= 224 * 1024, "shared memory of the resident CTAs");
    static_assert(BYTES >= GD_WARPS * 16 * HDP * 4 && BYTES >= 148 * CTAS * 64, "the joins reuse the ring");
};

// floats of one piece: 16 rows' log2 sum exp, then 16 rows of HDP values
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
__device__ __forceinline__ void cp_async16_or_zero(void *dst, const void *src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src), "r"(n)
                 : "memory");
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
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// The sequence's slot and length; a slot or length that does not fit counts
// as empty and is flagged.
__device__ __forceinline__ int gd_len(const GqaCacheArgs &c, int b, int *slot) {
    const int s = c.slots ? __ldg(c.slots + b) : b;
    const int n = s >= 0 && s < c.n_slots ? __ldg(c.lens + s) : -1;
    *slot = s;
    if (n < 0 || n > c.max_pages * WB_PAGE) {
        atomicOr(c.dev_err, WB_DERR_BOUNDS);
        return 0;
    }
    return n;
}

template <class T, int KIND, int HDP>
__global__ void __launch_bounds__(GD_THREADS, GdConf<KIND, HDP>::CTAS) gqa_decode_kernel(GqaDecodeArgs a) {
    using F = GdConf<KIND, HDP>;
    constexpr bool BF = KIND == GD_NATIVE && sizeof(T) == 2 && __is_same(T, __nv_bfloat16);  // product type
    constexpr bool QUANT = KIND != GD_NATIVE;
    constexpr int NK = HDP / 16;  // q . k products per 8 keys
    constexpr int NV = HDP / 8;   // p v products per 16 keys
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ long long s_scan[GD_WARPS];
    __shared__ long long s_pref;
    __shared__ int s_seq;
    __shared__ float s_m[GD_WARPS][16], s_l[GD_WARPS][16], s_m2[GD_WARPS][16], s_f[GD_WARPS][16], s_row[16];
    __shared__ int s_last;
    const GqaCacheArgs &c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, cc = lane & 3;
    const int G = a.H / c.Hkv, nch = (G + 15) / 16, ips = c.Hkv * nch;  // items of a sequence

    // ---- the line of units and this CTA's share
    const int per = (c.n_seq + GD_THREADS - 1) / GD_THREADS;
    long long mine = 0;
    for (int b = tid * per; b < min((tid + 1) * per, c.n_seq); b++) {
        int slot;
        const int n = gd_len(c, b, &slot);
        mine += (long long)((n + GD_UNIT - 1) / GD_UNIT) * ips;
        if (n == 0 && b % (int)gridDim.x == (int)blockIdx.x) {
            T *op = (T *)a.out + (long long)b * a.H * c.hd;
            for (int i = 0; i < a.H * c.hd; i++) op[i] = from_f<T>(0.0f);
            if (a.lse)
                for (int h = 0; h < a.H; h++) a.lse[(long long)b * a.H + h] = -INFINITY;
        }
    }
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    long long total = 0, before = inc - mine;
#pragma unroll
    for (int w = 0; w < GD_WARPS; w++) {
        if (w < warp) before += s_scan[w];
        total += s_scan[w];
    }
    const long long grid = min((long long)gridDim.x, total);
    if ((long long)blockIdx.x >= grid) return;
    const long long s0 = blockIdx.x * total / grid, s1 = (blockIdx.x + 1) * total / grid;
    if (s0 >= before && s0 < before + mine) {
        int b = tid * per;
        for (;; b++) {
            int slot;
            const long long n = (long long)((gd_len(c, b, &slot) + GD_UNIT - 1) / GD_UNIT) * ips;
            if (s0 < before + n) break;
            before += n;
        }
        s_seq = b;
        s_pref = before;
    }
    __syncthreads();
    int b = s_seq;
    long long pref = s_pref;

    uint8_t *ring = sm + warp * (F::NST * F::STAGE);
    const int rowb = c.row * F::ESZ;
    for (long long u = s0; u < s1;) {
        int slot;
        const int len = gd_len(c, b, &slot);
        const int U = (len + GD_UNIT - 1) / GD_UNIT;
        if (U == 0) {
            b++;
            continue;
        }
        const long long rel = u - pref;
        const int item = (int)(rel / U), ua = (int)(rel - (long long)item * U);
        const int ub = (int)min((long long)U, ua + (s1 - u));
        const int hk = item / nch, hc = item - hk * nch;
        const int h0 = hk * G + hc * 16, nrow = min(16, G - hc * 16);
        const int k0 = ua * GD_UNIT, k1 = min(ub * GD_UNIT, len);

        // ---- loads of this warp's blocks k0 + 16 (warp + 4 i)
        const int nblk = (k1 - k0 + 15) >> 4;
        const int cnt = (nblk - warp + GD_WARPS - 1) / GD_WARPS;
        const int32_t *trow = c.table + (long long)slot * c.max_pages;
        const int last_page = (k1 - 1) >> WB_PAGE_SHIFT;
        int pbase = k0 >> WB_PAGE_SHIFT;
        int pid = pbase + lane <= last_page ? __ldg(trow + pbase + lane) : -1;
        auto issue = [&](int i) {
            const int key0 = k0 + 16 * (warp + GD_WARPS * i);
            const int p = key0 >> WB_PAGE_SHIFT;
            if (p >= pbase + 32) {
                pbase = p;
                pid = pbase + lane <= last_page ? __ldg(trow + pbase + lane) : -1;
            }
            const int pg = __shfl_sync(0xffffffffu, pid, p - pbase);
            const bool ok = pg >= 0 && pg < c.n_pages;
            const long long row0 = ok ? ((long long)pg * c.Hkv + hk) * WB_PAGE + (key0 & (WB_PAGE - 1)) : 0;
            uint8_t *st = ring + (i % F::NST) * F::STAGE;
            const uint8_t *kp = (const uint8_t *)c.k_pages + row0 * rowb, *vp = (const uint8_t *)c.v_pages + row0 * rowb;
            const int ch = lane % F::CPR;
#pragma unroll
            for (int x = 0; x < F::CPR / 2; x++) {
                const int rr = lane / F::CPR + x * (32 / F::CPR);
                const int n = ok && key0 + rr < k1 && ch * 16 < rowb ? 16 : 0;
                const long long off = n ? (long long)rr * rowb + ch * 16 : 0;
                // piece positions within each 128 bytes: K's by row parity, V's
                // by row pair, so that the fragments' reads below touch every
                // bank once
                const int pos = (F::RB == 64 ? (rr & 1) * 4 : 0) + ch, line = rr * F::RB / 128 + (F::RB == 256 ? ch / 8 : 0);
                const int kpos = F::RB == 64 ? pos : (pos & 7) ^ ((rr & 1) << 2);
                const int vpos = (pos & 7) ^ (((rr >> 1) & 3) << 1);
                cp_async16_or_zero(st + line * 128 + kpos * 16, kp + off, n);
                cp_async16_or_zero(st + 16 * F::RB + line * 128 + vpos * 16, vp + off, n);
            }
            if (QUANT && lane < 8) {
                const float *sp = (lane < 4 ? c.k_scale : c.v_scale) + row0 + (lane & 3) * 4;
                cp_async16_or_zero(st + 32 * F::RB + lane * 16, sp, ok ? 16 : 0);
            }
            return ok;
        };
        uint32_t okbits = 0;  // bit i % NST: block i's page is mapped
#pragma unroll
        for (int i = 0; i < F::NST - 1; i++) {
            if (i < cnt && issue(i)) okbits |= 1u << i;
            ptx::cp_async_commit();
        }

        // ---- queries: rows r and r + 8 of the 16, dims in the order of K's pieces
        uint32_t qf[NK][4];
        float fac[2];  // score factor of the two rows, log2 e included
        {
            float amax[2] = {0.0f, 0.0f};
            float qv[2][NK * 4];
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int row = r + 8 * hf;
                const T *qp = (const T *)a.q + b * a.q_ss + (long long)(h0 + row) * a.q_hs;
#pragma unroll
                for (int t = 0; t < NK; t++) {
                    const int d0 = F::ESZ == 1 ? 16 * (cc + 4 * (t / 4)) + 4 * (t % 4) : 8 * (cc + 4 * (t / 2)) + 4 * (t % 2);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float x = row < nrow && d0 + e < c.hd ? to_f(qp[d0 + e]) : 0.0f;
                        qv[hf][t * 4 + e] = x;
                        amax[hf] = fmaxf(amax[hf], fabsf(x));
                    }
                }
                fac[hf] = a.scale * 1.4426950408889634f;
                if (QUANT && !__is_same(T, __half)) {
                    // bf16 queries meet fp16 keys: divided by a power of two
                    // so that the row's largest is in [1, 2) (exact down to
                    // 2^-14 of it)
                    const int e = min(max((int)(__float_as_uint(quad_max(amax[hf])) >> 23), 1), 253);
                    const float f = __uint_as_float((uint32_t)(254 - e) << 23);
                    fac[hf] *= __uint_as_float((uint32_t)e << 23);
#pragma unroll
                    for (int i = 0; i < NK * 4; i++) qv[hf][i] *= f;
                }
            }
#pragma unroll
            for (int t = 0; t < NK; t++) {
                qf[t][0] = pack2(qv[0][t * 4], qv[0][t * 4 + 1], BF);
                qf[t][1] = pack2(qv[1][t * 4], qv[1][t * 4 + 1], BF);
                qf[t][2] = pack2(qv[0][t * 4 + 2], qv[0][t * 4 + 3], BF);
                qf[t][3] = pack2(qv[1][t * 4 + 2], qv[1][t * 4 + 3], BF);
            }
        }

        float acc[NV][4];
#pragma unroll
        for (int j = 0; j < NV; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
        // finite stand-ins for -inf: the first visible score replaces them
        float m[2] = {-1e30f, -1e30f}, m2[2] = {-1e30f, -1e30f}, l[2] = {0.0f, 0.0f};
        bool unmapped = false;

        for (int i = 0; i < cnt; i++) {
            ptx::cp_async_wait<F::NST - 2>();
            __syncwarp();
            const int stg = i % F::NST;
            const bool ok = (okbits >> stg) & 1;
            const int nx = i + F::NST - 1;
            if (nx < cnt) {
                okbits &= ~(1u << (nx % F::NST));
                if (issue(nx)) okbits |= 1u << (nx % F::NST);
            }
            ptx::cp_async_commit();
            const uint8_t *st = ring + stg * F::STAGE;
            const int key0 = k0 + 16 * (warp + GD_WARPS * i);

            // scores of keys 0-7 (s[0]) and 8-15 (s[1])
            float s[2][4] = {};
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const int rr = r + 8 * g;
#pragma unroll
                for (int x = 0; x < F::CPR / 4; x++) {
                    const int ch = cc + 4 * x;
                    const int pos = (F::RB == 64 ? (rr & 1) * 4 : 0) + ch;
                    const int line = rr * F::RB / 128 + (F::RB == 256 ? ch / 8 : 0);
                    const int kpos = F::RB == 64 ? pos : (pos & 7) ^ ((rr & 1) << 2);
                    const uint4 w = *reinterpret_cast<const uint4 *>(st + line * 128 + kpos * 16);
                    if constexpr (QUANT) {
                        mma16816<BF>(s[g], qf[4 * x], to_f16x2<KIND, 0>(w.x), to_f16x2<KIND, 1>(w.x));
                        mma16816<BF>(s[g], qf[4 * x + 1], to_f16x2<KIND, 0>(w.y), to_f16x2<KIND, 1>(w.y));
                        mma16816<BF>(s[g], qf[4 * x + 2], to_f16x2<KIND, 0>(w.z), to_f16x2<KIND, 1>(w.z));
                        mma16816<BF>(s[g], qf[4 * x + 3], to_f16x2<KIND, 0>(w.w), to_f16x2<KIND, 1>(w.w));
                    } else {
                        mma16816<BF>(s[g], qf[2 * x], w.x, w.y);
                        mma16816<BF>(s[g], qf[2 * x + 1], w.z, w.w);
                    }
                }
            }
            // this lane's keys: 2cc, 2cc+1 (g = 0) and 2cc+8, 2cc+9 (g = 1)
            float lv[2][2];
#pragma unroll
            for (int g = 0; g < 2; g++) {
                float2 ks = make_float2(1.0f, 1.0f), vs = ks;
                if (QUANT) {
                    ks = *reinterpret_cast<const float2 *>(st + 32 * F::RB + (2 * cc + 8 * g) * 4);
                    vs = *reinterpret_cast<const float2 *>(st + 32 * F::RB + 64 + (2 * cc + 8 * g) * 4);
                    lv[g][0] = lg2(vs.x);
                    lv[g][1] = lg2(vs.y);
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const bool vis = ok && key0 + 2 * cc + 8 * g + e < k1;
                    const float kf = e ? ks.y : ks.x;
                    s[g][e] = vis ? s[g][e] * fac[0] * kf : -INFINITY;
                    s[g][2 + e] = vis ? s[g][2 + e] * fac[1] * kf : -INFINITY;
                    if (QUANT && !vis) lv[g][e] = 0.0f;
                }
            }
            unmapped |= !ok;
            float mx[2], mx2[2];
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                mx[hf] = quad_max(fmaxf(fmaxf(s[0][2 * hf], s[0][2 * hf + 1]), fmaxf(s[1][2 * hf], s[1][2 * hf + 1])));
                if (QUANT)
                    mx2[hf] = quad_max(fmaxf(fmaxf(s[0][2 * hf] + lv[0][0], s[0][2 * hf + 1] + lv[0][1]),
                                             fmaxf(s[1][2 * hf] + lv[1][0], s[1][2 * hf + 1] + lv[1][1])));
                else mx2[hf] = mx[hf];
            }
            // the references follow the maxima when one is far ahead
            const bool far = mx[0] > m[0] + GD_LAZY || mx[1] > m[1] + GD_LAZY ||
                             (QUANT && (mx2[0] > m2[0] + GD_LAZY || mx2[1] > m2[1] + GD_LAZY));
            if (__any_sync(0xffffffffu, far)) {
                float f2[2];
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const float mn = fmaxf(m[hf], mx[hf]), mn2 = fmaxf(m2[hf], mx2[hf]);
                    l[hf] *= ex2(m[hf] - mn);
                    f2[hf] = ex2(m2[hf] - mn2);
                    m[hf] = mn;
                    m2[hf] = mn2;
                }
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    acc[j][0] *= f2[0];
                    acc[j][1] *= f2[0];
                    acc[j][2] *= f2[1];
                    acc[j][3] *= f2[1];
                }
            }
            uint32_t pf[4], pl[4];
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const float p0 = ex2(s[g][2 * hf] - m[hf] + GD_SHIFT), p1 = ex2(s[g][2 * hf + 1] - m[hf] + GD_SHIFT);
                    l[hf] += p0 + p1;
                    if (QUANT)
                        pf[2 * g + hf] = pack2(ex2(s[g][2 * hf] + lv[g][0] - m2[hf] + GD_SHIFT),
                                               ex2(s[g][2 * hf + 1] + lv[g][1] - m2[hf] + GD_SHIFT), BF);
                    else pf[2 * g + hf] = pack2(p0, p1, BF);
                    if (BF) {
                        const uint32_t x = pf[2 * g + hf];
                        pl[2 * g + hf] = pack2(p0 - __uint_as_float(x << 16), p1 - __uint_as_float(x & 0xffff0000u), BF);
                    }
                }

            // values: piece r of rows 2cc, 2cc+1, 2cc+8, 2cc+9
            const uint8_t *sv = st + 16 * F::RB;
            if constexpr (F::ESZ == 2) {
#pragma unroll
                for (int x = 0; x < HDP / 64; x++) {
                    uint4 w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int rr = 2 * cc + (e & 1) + 8 * (e >> 1);
                        w[e] = *reinterpret_cast<const uint4 *>(sv + (rr * F::RB / 128 + x) * 128 +
                                                                ((r ^ (((rr >> 1) & 3) << 1)) * 16));
                    }
                    const uint32_t *w0 = &w[0].x, *w1 = &w[1].x, *w2 = &w[2].x, *w3 = &w[3].x;
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        const uint32_t a0 = __byte_perm(w0[d], w1[d], 0x5410), b0 = __byte_perm(w2[d], w3[d], 0x5410);
                        const uint32_t a1 = __byte_perm(w0[d], w1[d], 0x7632), b1 = __byte_perm(w2[d], w3[d], 0x7632);
                        mma16816<BF>(acc[8 * x + 2 * d], pf, a0, b0);
                        mma16816<BF>(acc[8 * x + 2 * d + 1], pf, a1, b1);
                        if (BF) {
                            mma16816<BF>(acc[8 * x + 2 * d], pl, a0, b0);
                            mma16816<BF>(acc[8 * x + 2 * d + 1], pl, a1, b1);
                        }
                    }
                }
            } else {
                uint32_t w[4][HDP / 32];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int rr = 2 * cc + (e & 1) + 8 * (e >> 1);
                    if constexpr (HDP == 128) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(sv + rr * 128 + ((r ^ (((rr >> 1) & 3) << 1)) * 16));
                        w[e][0] = v.x; w[e][1] = v.y; w[e][2] = v.z; w[e][3] = v.w;
                    } else {
                        const int pos = ((rr & 1) * 4 + (r >> 1)) ^ (((rr >> 1) & 3) << 1);
                        const uint2 v = *reinterpret_cast<const uint2 *>(sv + (rr >> 1) * 128 + pos * 16 + (r & 1) * 8);
                        w[e][0] = v.x; w[e][1] = v.y;
                    }
                }
#pragma unroll
                for (int d = 0; d < HDP / 32; d++) {
                    // (key a byte, key b byte) pairs of dims 4d, 4d+1 and 4d+2, 4d+3
                    const uint32_t a01 = __byte_perm(w[0][d], w[1][d], 0x5140), a23 = __byte_perm(w[0][d], w[1][d], 0x7362);
                    const uint32_t b01 = __byte_perm(w[2][d], w[3][d], 0x5140), b23 = __byte_perm(w[2][d], w[3][d], 0x7362);
                    mma16816<BF>(acc[4 * d], pf, to_f16x2<KIND, 0>(a01), to_f16x2<KIND, 0>(b01));
                    mma16816<BF>(acc[4 * d + 1], pf, to_f16x2<KIND, 1>(a01), to_f16x2<KIND, 1>(b01));
                    mma16816<BF>(acc[4 * d + 2], pf, to_f16x2<KIND, 0>(a23), to_f16x2<KIND, 0>(b23));
                    mma16816<BF>(acc[4 * d + 3], pf, to_f16x2<KIND, 1>(a23), to_f16x2<KIND, 1>(b23));
                }
            }
        }
        ptx::cp_async_wait<0>();
        if (unmapped && lane == 0) atomicOr(c.dev_err, WB_DERR_BOUNDS);

        // ---- the four warps' outputs into one
        l[0] = quad_sum(l[0]);
        l[1] = quad_sum(l[1]);
        if (cc == 0) {
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                s_m[warp][r + 8 * hf] = m[hf];
                s_l[warp][r + 8 * hf] = l[hf];
                s_m2[warp][r + 8 * hf] = QUANT ? m2[hf] : m[hf];
            }
        }
        __syncthreads();  // the rings have been read
        float *buf = reinterpret_cast<float *>(sm);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            // column n of product j is dim n * 16 + j (8-bit, 128 columns), n * 8 + j % 8 + 64 (j / 8) (else)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = r + 8 * (e >> 1), n = 2 * cc + (e & 1);
                const int d = F::ESZ == 1 && HDP == 128 ? n * 16 + j : n * 8 + (j & 7) + 64 * (j >> 3);
                if (row < nrow) buf[(warp * 16 + row) * HDP + d] = acc[j][e];
            }
        }
        if (tid < 16) {
            float M = -1e30f, M2 = -1e30f, L = 0.0f;
            for (int w = 0; w < GD_WARPS; w++) {
                M = fmaxf(M, s_m[w][tid]);
                M2 = fmaxf(M2, s_m2[w][tid]);
            }
            for (int w = 0; w < GD_WARPS; w++) L += s_l[w][tid] * ex2(s_m[w][tid] - M);
            const float inv = L == 0.0f ? 0.0f : ex2(M2 - M) / L;
            for (int w = 0; w < GD_WARPS; w++) s_f[w][tid] = ex2(s_m2[w][tid] - M2) * inv;
            s_row[tid] = L == 0.0f ? -INFINITY : M - GD_SHIFT + log2f(L);  // log2 sum exp
        }
        __syncthreads();
        const bool whole = ua == 0 && ub == U;
        float *piece = a.part + ((long long)blockIdx.x * 2 + (ua == 0 ? 1 : 0)) * gqa_piece(HDP);
        for (int i = tid; i < nrow * c.hd; i += GD_THREADS) {
            const int row = i / c.hd, d = i - row * c.hd;
            float o = 0.0f;
#pragma unroll
            for (int w = 0; w < GD_WARPS; w++) o += buf[(w * 16 + row) * HDP + d] * s_f[w][row];
            if (whole) ((T *)a.out)[((long long)b * a.H + h0 + row) * c.hd + d] = from_f<T>(o);
            else __stcg(piece + 16 + row * HDP + d, o);
        }
        if (tid < nrow) {
            if (!whole) __stcg(piece + tid, s_row[tid]);
            else if (a.lse) a.lse[(long long)b * a.H + h0 + tid] = s_row[tid] * 0.6931471805599453f;
        }
        if (!whole) {
            // ---- the last CTA of the item's joins the pieces
            const long long i0 = pref + (long long)item * U;
            const int c0 = (int)(((i0 + 1) * grid - 1) / total), c1 = (int)(((i0 + U) * grid - 1) / total);
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
                float *wt = reinterpret_cast<float *>(sm);  // [n][16] weights
                for (int row = warp; row < nrow; row += GD_WARPS) {
                    float M = -INFINITY, L = 0.0f;
                    for (int x = lane; x < n; x += 32) M = fmaxf(M, __ldcg(at(x) + row));
                    M = warp_max(M);
                    const float M0 = M == -INFINITY ? 0.0f : M;
                    for (int x = lane; x < n; x += 32) {
                        const float w = ex2(__ldcg(at(x) + row) - M0);
                        wt[x * 16 + row] = w;
                        L += w;
                    }
                    L = warp_sum(L);
                    if (lane == 0) {
                        s_f[0][row] = L == 0.0f ? 0.0f : 1.0f / L;
                        s_row[row] = L == 0.0f ? -INFINITY : M0 + log2f(L);
                    }
                }
                __syncthreads();
                for (int i = tid; i < nrow * c.hd; i += GD_THREADS) {
                    const int row = i / c.hd, d = i - row * c.hd;
                    float o = 0.0f;
#pragma unroll 4
                    for (int x = 0; x < n; x++) o += __ldcg(at(x) + 16 + row * HDP + d) * wt[x * 16 + row];
                    ((T *)a.out)[((long long)b * a.H + h0 + row) * c.hd + d] = from_f<T>(o * s_f[0][row]);
                }
                if (tid < nrow && a.lse) a.lse[(long long)b * a.H + h0 + tid] = s_row[tid] * 0.6931471805599453f;
            }
        }
        __syncthreads();  // shared memory is free for the next item
        u += ub - ua;
        if (rel + (ub - ua) == (long long)U * ips) {
            pref += (long long)U * ips;
            b++;
        }
    }
}

static int gd_grid(const GqaCacheArgs &c, int H, int sm_count, int ctas) {
    const int G = H / c.Hkv;
    const long long most = (long long)c.n_seq * c.Hkv * ((G + 15) / 16) * c.max_pages * (WB_PAGE / GD_UNIT);
    return (int)std::max(1LL, std::min(most, (long long)std::min(sm_count, 148) * ctas));
}

size_t gqa_decode_scratch(const GqaCacheArgs &c, int H, int sm_count) {
    return (size_t)gd_grid(c, H, sm_count, 4) * 2 * gqa_piece(c.hd <= 64 ? 64 : 128) * sizeof(float);
}

template <class T, int KIND, int HDP>
static int gd_launch(const GqaDecodeArgs &a, int sm_count, cudaStream_t st, std::string *msg) {
    using F = GdConf<KIND, HDP>;
    static const cudaError_t set =
        cudaFuncSetAttribute(gqa_decode_kernel<T, KIND, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::BYTES);
    if (set != cudaSuccess) {
        *msg = std::string("decode kernel attributes: ") + cudaGetErrorString(set);
        return WB_ECUDA;
    }
    ProfScope ps("gqa_decode", st);
    gqa_decode_kernel<T, KIND, HDP><<<gd_grid(a.c, a.H, sm_count, F::CTAS), GD_THREADS, F::BYTES, st>>>(a);
    return WB_OK;
}

int launch_gqa_decode(const GqaCacheArgs &c, int dtype, int H, const void *q, long long q_ss, long long q_hs,
                      float scale, void *out, float *lse, unsigned int *counters, void *scratch, int sm_count,
                      cudaStream_t st, std::string *msg) {
    GqaDecodeArgs a{c, q, out, lse, q_ss, q_hs, H, scale, counters, (float *)scratch};
    auto by_store = [&](auto t) {
        using T = decltype(t);
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
