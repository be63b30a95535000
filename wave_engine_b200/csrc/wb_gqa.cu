// wb_gqa.cu -- grouped-head dot-product attention over packed prompts.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij) / sum_j exp(s_ij),
//   s_ij = scale q_i . k_j  over the keys j <= i + (n_k - n_q) of the
//   query's own sequence (all of them when not causal);
//   lse_i = log sum_j exp(s_ij); a query without keys, or whose scores are all
//   -infinity, gives 0 and -inf.
//
// One pass over the keys per query tile with the running maximum m and sum
// l of the softmax: S = Q K^T on tcgen05 into TMEM, P = 2^(c S - m) in
// registers (c = scale log2 e), P back to TMEM as the left operand of
// O += P V, O in TMEM until the end.  m follows the row's maximum only when
// that is more than 2^8 ahead (O and l are then rescaled), so most tiles
// touch O on the tensor cores alone.  P is rounded to the type of q, k and v:
// in 32 bits (tf32) its product would take twice as long.  l sums what P was
// before; the output is off by up to that type's unit roundoff times
// sum_j p_ij |v_j|, as much as the rounding of an output of that size.
//
// Tiles.  The query heads that share a key-value head are rows of the same
// tile: row = token * G + g, 128 / G tokens of G heads, which TMA gathers as
// one box.  A CTA has two such tiles, one softmax warpgroup each: while the
// tensor cores work for one, the other's warps take exponentials, and both
// read the same K and V tiles (128 keys).  P is handed over in two halves,
// so that its product begins while the second is computed.
//
// What bounds it.  A pair of tiles costs 2048 cycles of the tensor cores at
// head_dim 128 (1024 at 64) and, at 16 ex2 per cycle and SM, 2048 of the
// exponential unit.  It takes about 3400 (3050): a tile's chain is 400 to 600
// cycles for the maximum, 1350 to 1700 for the exponentials (the other tile's
// among them), then 700 (400) to issue and run P V and the next Q K^T and 350
// until the scores are seen.  One sequence of 8192 tokens, 32 heads on 8,
// head_dim 128, causal: 437 us, 1258 TFLOP/s, 75% of the measured cuBLAS
// burst rate, in bursts of a few calls; call after call for seconds 509 to 520
// us at 1590 to 1640 of 1965 MHz, 75% of the sustained rate: there the chip is
// at its power limit (with the two tiles half a period apart a pair takes
// 3310 cycles at a clock 4% lower: the same time).
// Short sequences pay the start and end of an item, about 4000 cycles: 32
// sequences of 1 to 1024 tokens, 12 heads on 4, head_dim 64: 61.3 us.
//
// Measured and not kept: exponentials by a polynomial on the FMA pipe (a
// quarter of them cost 4% at 8192 tokens, three eighths 7%); eight softmax
// warps a tile (+10%); a warp for each tile's products (+25%); a third S
// buffer at head_dim 64, so that Q K^T runs ahead (+12%: more barriers and
// registers than it hides); the next item's first Q K^T issued before this
// one's epilogue (+4% at head_dim 64, with Q in two buffers +5%: it goes in
// front of the other tile's last products).
#include "wb_gqa.h"
#include "wb_tc.h"

#include <algorithm>

namespace wb {

static constexpr int GA_ROWS = 128, GA_KEYS = 128;  // rows of a query tile, keys of a K/V tile
static constexpr int GA_EDGES = 4;  // most key tiles that some row of a CTA sees in part

struct GaArgs {
    GqaAttnArgs a;
    float c;      // |scale| log2 e, at least the smallest subnormal
    float c_two;  // the largest power of two that is not above c
    int G, TT;    // heads per key-value head, tokens of a query tile
    int vec;      // out rows take 16-byte stores
    long long items;  // no more than this many (sequence, tiles) items
};

// A work item: two query tiles of one key-value head.
struct GaItem {
    int q0, nq, k0, nk;      // the sequence's rows; q0 < 0: no more work
    int tok0, hk;            // first token of the first tile, key-value head
    int nt[2], edge;         // key tiles of each query tile, the first that some row sees in part
    uint32_t any_bad, bad[GA_EDGES][GA_KEYS / 32];  // keys from tile `edge` on with values that are not finite
};
static constexpr int GA_SLOTS = 4;  // items known to the CTA's roles at a time

template <int HDP>
struct GaConf {
    static constexpr int NT = 2;  // query tiles of a CTA
    static constexpr int W_TMA = 4 * NT, W_MMA = W_TMA + 1, W_FIX = W_MMA + 1;  // warps before: softmax
    static constexpr int THREADS = (W_FIX + 2) * 32;
    // registers: the softmax warps take what the other four give up
    static constexpr int R_SOFTMAX = 208, R_OTHER = 88;
    static constexpr int TMEM = NT * 256, O_COL = NT * 128;  // columns: S of each tile, then O of each
    static constexpr int NC = HDP / 64;              // 64-column swizzle atoms of a row
    static constexpr int Q_BYTES = GA_ROWS * HDP * 2;
    static constexpr int KV_BYTES = GA_KEYS * HDP * 2;
    static constexpr int ST = HDP == 64 ? 4 : 2;  // K/V stages
    static constexpr int OFF_K = NT * Q_BYTES, OFF_V = OFF_K + ST * KV_BYTES;
    static constexpr int OFF_OUT = OFF_V + ST * KV_BYTES, OUT_WARP = 32 * 64;  // a warp's 32 rows of 32 outputs
    static constexpr int OFF_BAR = OFF_OUT + 4 * NT * OUT_WARP;
    static constexpr int NBAR = 4 * ST + 4 * NT + 3 + 3 * GA_SLOTS;
    static constexpr int OFF_ITEM = OFF_BAR + NBAR * 8;
    static constexpr int BYTES = OFF_ITEM + GA_SLOTS * (int)sizeof(GaItem) + 1024;
    static_assert(BYTES + 1280 <= 227 * 1024, "shared memory");
    static_assert(OFF_OUT % 128 == 0 && OFF_BAR % 16 == 0, "alignment");
};

// Bounded mbarrier wait that also gives up once another role has: a timeout
// then does not chain into one per barrier.  Lanes may give up apart from each
// other, so no lane leaves a loop on its own answer: after a timeout a role
// goes on to the item's end for nothing (every wait returns at once), where
// the warp leaves as one (a vote in every wait: 62.3 us instead of 60.8, packed
// 768-wide batch).
__device__ __forceinline__ bool ga_wait(uint64_t *bar, uint32_t parity, volatile int *gave_up) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (true) {
        if (ptx::mbar_try_wait_sleep(bar, parity, 20000)) return true;
        if (*gave_up) return false;
        if (clock64() - t0 > 4000000000LL) {
            *gave_up = 1;
            return false;
        }
    }
}

__device__ __forceinline__ float ga_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// one lane of a converged warp, in the form that the compiler knows to be one:
// MMAs behind it are issued faster than behind `lane == 0` (8192 tokens,
// 32 heads x 128: 450 -> 438 us)
__device__ __forceinline__ bool ga_elect() {
    uint32_t y;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(y));
    return y != 0;
}

// the largest; NaN if one is
__device__ __forceinline__ float ga_max(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

template <class T>
__device__ __forceinline__ uint32_t ga_pack(float lo, float hi) {
    uint32_t r;
    if (__is_same(T, __nv_bfloat16)) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// tcgen05.mma with A from shared memory or TMEM; descriptors as low and high
// words
template <bool ACC>
__device__ __forceinline__ void ga_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}\n" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "n"(ACC ? 1 : 0)
        : "memory");
}
__device__ __forceinline__ void ga_mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 b;\n mov.b64 b, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
        "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}

// Items (NT query tiles each) of a sequence; 0, flagged, when its rows do
// not lie inside the tensors.
__device__ __forceinline__ int ga_items(const GqaAttnArgs &a, int b, int per_item) {
    const int q0 = __ldg(a.cu_q + b), q1 = __ldg(a.cu_q + b + 1), k0 = __ldg(a.cu_k + b), k1 = __ldg(a.cu_k + b + 1);
    if (q0 < 0 || q1 < q0 || q1 > a.total_q || k0 < 0 || k1 < k0 || k1 > a.total_k) {
        atomicOr(a.dev_err, WB_DERR_BOUNDS);
        return 0;
    }
    return (q1 - q0 + per_item - 1) / per_item;
}

// Finds the sequence and tiles of ascending item indexes; one warp.  Up to
// 64 sequences: tiles late in their sequences (with the most keys) first --
// the largest t with more than `index` items at or behind place t, then by
// sequence -- so that long items are dealt out first (8 sequences up to 4096:
// 135 us, 164 in the sequences' order; 32 up to 1024: 61.3, 68; 64 up to 600:
// 62, 66).  More: in the order of the sequences, one pass over them for all
// items of the CTA (65 up to 600: 65 us both ways; 255 up to 400: 125 us, 140
// with the longest first).
struct GaFinder {
    static constexpr int N = 2;
    int n[N];                // items of sequences lane + 32 x (or of sequences b0 + lane, in n[0])
    int top = 0, b0 = 0;
    long long before = 0;    // items of sequences before b0
    __device__ __forceinline__ void start(const GqaAttnArgs &a, int per_item, int lane) {
#pragma unroll
        for (int x = 0; x < N; x++) {
            n[x] = lane + 32 * x < a.n_seq ? ga_items(a, lane + 32 * x, per_item) : 0;
            top = max(top, n[x]);
        }
        top = __reduce_max_sync(0xffffffffu, top);
    }
    __device__ __forceinline__ int behind(int t) const {  // items at places >= t
        int sum = 0;
#pragma unroll
        for (int x = 0; x < N; x++) sum += max(0, n[x] - t);
        return __reduce_add_sync(0xffffffffu, sum);
    }
    __device__ __forceinline__ bool find(const GqaAttnArgs &a, int per_item, long long index, int lane, int *seq, int *place) {
        if (a.n_seq > 32 * N) {
            for (;;) {
                int inc = n[0];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += y;
                }
                const uint32_t past = __ballot_sync(0xffffffffu, before + inc > index);
                if (past) {
                    const int at = __ffs(past) - 1;
                    *seq = b0 + at;
                    *place = (int)(index - before) - __shfl_sync(0xffffffffu, inc - n[0], at);
                    return true;
                }
                before += __shfl_sync(0xffffffffu, inc, 31);
                b0 += 32;
                if (b0 >= a.n_seq) return false;
                n[0] = b0 + lane < a.n_seq ? ga_items(a, b0 + lane, per_item) : 0;
            }
        }
        if (a.n_seq == 1) {
            *place = top - 1 - (int)index;
            return index < top;
        }
        if (index >= behind(0)) return false;
        int lo = 0, hi = top;  // behind(lo) > index >= behind(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (behind(mid) > index) lo = mid;
            else hi = mid;
        }
        int rank = (int)(index - behind(hi));
        *place = lo;
#pragma unroll
        for (int x = 0; x < N; x++) {
            const uint32_t has = __ballot_sync(0xffffffffu, n[x] > lo);
            if (rank >= 0 && rank < __popc(has)) *seq = 32 * x + (int)__fns(has, 0, rank + 1);
            rank -= __popc(has);
        }
        return true;
    }
};

// Persistent: one CTA per SM takes the items in rounds, every second round
// backwards (the items come largest first), and its roles run ahead of each
// other from item to item: warps 0-3 and 4-7 softmax and epilogue of tiles 0
// and 1 (thread = row); warp 8 finds the items and loads; warp 9 issues the
// MMAs and owns TMEM; warps 10, 11 look through the V tiles at the rows'
// edges.
//
// Edges.  A key that a row does not see gets probability 0, but 0 times an
// infinity or NaN among its values would reach the row through the MMA.  So
// in the tiles that some row sees in part (at the diagonal and at the
// sequence's end) warps 10 and 11 set values that are not finite, and all
// values past the sequence's last key, to 0 before the MMA may read them, and
// note the key; the epilogue adds such values to the rows that do see them.
template <class T, int HDP>
__global__ void __launch_bounds__(GaConf<HDP>::THREADS, 1)
    gqa_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const GaArgs ga) {
    using F = GaConf<HDP>;
    constexpr int ST = F::ST, NC = F::NC, NT = F::NT;
    constexpr bool BF = __is_same(T, __nv_bfloat16);
    const GqaAttnArgs &a = ga.a;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm + F::OFF_BAR);
    uint64_t *full = bars, *free_ = full + ST, *vok = free_ + ST, *vgo = vok + ST;
    uint64_t *qfull = vgo + ST, *qfree = qfull + 1, *done = qfree + 1;
    uint64_t *sfull = done + 1, *pready = sfull + NT, *ofull = pready + 2 * NT;
    uint64_t *itemfull = ofull + NT, *itemfree = itemfull + GA_SLOTS, *fixed = itemfree + GA_SLOTS;
    GaItem *items = reinterpret_cast<GaItem *>(sm + F::OFF_ITEM);
    __shared__ uint32_t tmem_slot;
    __shared__ int s_gave_up;
    volatile int *gave_up = &s_gave_up;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = ga.G, TT = ga.TT;

    GaFinder finder;  // warp W_TMA's
    int seq = 0, place = 0;
    bool any = false;
    if (warp == F::W_TMA) {
        if (lane == 0) {
            ptx::prefetch_tmap(&tm_q);
            ptx::prefetch_tmap(&tm_k);
            ptx::prefetch_tmap(&tm_v);
        }
        finder.start(a, NT * TT, lane);
        any = finder.find(a, NT * TT, blockIdx.x / a.Hkv, lane, &seq, &place);
    }
    if (warp == 0) {
        for (int i = lane; i < F::NBAR; i += 32) {
            uint64_t *b = bars + i;
            int n = 1;
            if (b >= vok && b < vok + ST) n = 2;
            else if (b >= pready && b < pready + 2 * NT) n = 4;
            else if (b >= itemfree && b < itemfree + GA_SLOTS) n = 4 * NT + 3;
            else if (b >= fixed) n = 2;
            ptx::mbar_init(b, n);
        }
        ptx::fence_mbar_init();
        if (lane == 0) s_gave_up = 0;
    }
    if (warp == F::W_MMA) {
        ptx::tmem_alloc(&tmem_slot, F::TMEM);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // keys that token t of an item's sequence sees
    auto visible = [&](int nq, int nk, int t) {
        const long long n = a.causal ? (long long)t + 1 + nk - nq : nk;
        return (int)max(0LL, min((long long)nk, n));
    };

    uint32_t g = 0, nq_loads = 0;  // warp W_TMA, lane 0: ring stages and Q pairs loaded
    if (warp >= F::W_TMA) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::R_OTHER));
        if (warp == F::W_TMA) {
            // ---- items and loads
            bool ok = true;
            for (int k = 0;; k++) {
                const long long index = (long long)k * gridDim.x + ((k & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                if (k > 0) any = index < ga.items * a.Hkv && finder.find(a, NT * TT, index / a.Hkv, lane, &seq, &place);
                GaItem *it = items + k % GA_SLOTS;
                if (k >= GA_SLOTS &&
                    !__all_sync(0xffffffffu, ga_wait(itemfree + k % GA_SLOTS, (uint32_t)(k / GA_SLOTS - 1) & 1, gave_up))) {
                    if (lane == 0) atomicOr(a.dev_err, WB_DERR_TIMEOUT_TMA);
                    ok = false;
                    break;
                }
                if (lane <= GA_EDGES * GA_KEYS / 32) (&it->any_bad)[lane] = 0;
                const int q0 = any ? __ldg(a.cu_q + seq) : -1, nq = any ? __ldg(a.cu_q + seq + 1) - q0 : 0;
                const int k0 = any ? __ldg(a.cu_k + seq) : 0, nk = any ? __ldg(a.cu_k + seq + 1) - k0 : 0;
                const int hk = (int)(index % a.Hkv), tok0 = place * NT * TT;
                int nt[NT], nmax = 0;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const int last = min(tok0 + (t + 1) * TT, nq) - 1;
                    nt[t] = tok0 + t * TT < nq ? (visible(nq, nk, last) + GA_KEYS - 1) / GA_KEYS : 0;
                    nmax = max(nmax, nt[t]);
                }
                const int edge = visible(nq, nk, tok0) / GA_KEYS;
                __syncwarp();
                if (lane == 0) {
                    it->q0 = q0;
                    it->nq = nq;
                    it->k0 = k0;
                    it->nk = nk;
                    it->tok0 = tok0;
                    it->hk = hk;
                    it->nt[0] = nt[0];
                    it->nt[1] = nt[1];
                    it->edge = edge;
                    ptx::mbar_arrive(itemfull + k % GA_SLOTS);
                }
                if (!any) break;
                if (lane == 0 && nmax > 0) {
                    // Stage g of the ring holds K of the item's tile x and V
                    // of tile x - 1, what one round of the products needs.
                    for (int x = 0; ok && x <= nmax; x++) {
                        const int st = (int)(g % ST);
                        if (g >= ST && !ga_wait(free_ + st, (g / ST - 1) & 1, gave_up)) {
                            ok = false;
                            break;
                        }
                        // warps 10, 11 come to a stage out of step with its
                        // phases: this one lets them at the tile's own
                        if (x > edge) ptx::mbar_arrive(vgo + st);
                        ptx::mbar_arrive_expect_tx(full + st, ((x < nmax) + (x > 0)) * F::KV_BYTES);
                        g++;
                        for (int c = 0; x < nmax && c < NC; c++)
                            ptx::tma_load_3d(sm + F::OFF_K + st * F::KV_BYTES + c * (GA_KEYS * 128), &tm_k, full + st,
                                             c * 64, hk, k0 + x * GA_KEYS);
                        for (int c = 0; x > 0 && c < NC; c++)
                            ptx::tma_load_3d(sm + F::OFF_V + st * F::KV_BYTES + c * (GA_KEYS * 128), &tm_v, full + st,
                                             c * 64, hk, k0 + (x - 1) * GA_KEYS);
                        if (x > 0) continue;
                        if (nq_loads > 0) ok = ga_wait(qfree, (nq_loads - 1) & 1, gave_up);
                        if (!ok) break;
                        int tiles = 0;
#pragma unroll
                        for (int t = 0; t < NT; t++) tiles += nt[t] > 0;
                        ptx::mbar_arrive_expect_tx(qfull, (uint32_t)(tiles * NC * G * TT * 128));
#pragma unroll
                        for (int t = 0; t < NT; t++)
                            for (int c = 0; nt[t] > 0 && c < NC; c++)
                                ptx::tma_load_4d(sm + t * F::Q_BYTES + c * (GA_ROWS * 128), &tm_q, qfull, c * 64, 0, hk,
                                                 q0 + tok0 + t * TT);
                        nq_loads++;
                    }
                    if (!ok) atomicOr(a.dev_err, WB_DERR_TIMEOUT_TMA);
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
            }
        } else if (warp == F::W_MMA) {
            // ---- products.  The whole warp goes through the loop, one lane
            // issues: counters and stages then stay in uniform registers,
            // where the MMAs want their descriptors.
            {
                constexpr uint32_t ID_QK = BF ? ptx::idesc_bf16(128, 128, 0, 0) : ptx::idesc_f16(128, 128, 0, 0);
                constexpr uint32_t ID_PV = BF ? ptx::idesc_bf16(128, HDP, 0, 1) : ptx::idesc_f16(128, HDP, 0, 1);
                // Descriptors: the low words change, by constants within a
                // product; few instructions stand between a barrier and the
                // first product behind it.
                const uint32_t hi = 1024 / 16 | 1u << 14 | ptx::UMMA_SW128 << 29;
                const uint32_t q_lo = ptx::smem_u32(sm) >> 4 | 1u << 16, k_lo = ptx::smem_u32(sm + F::OFF_K) >> 4 | 1u << 16;
                const uint32_t v_lo = ptx::smem_u32(sm + F::OFF_V) >> 4 | (GA_KEYS * 128 / 16) << 16;
                auto qk = [&](int t, int st) {
                    const uint32_t q = q_lo + t * (F::Q_BYTES / 16), kd = k_lo + st * (F::KV_BYTES / 16);
                    if (ga_elect()) {
#pragma unroll
                        for (int kk = 0; kk < HDP / 16; kk++) {
                            const uint32_t o = (kk >> 2) * (GA_ROWS * 8) + (kk & 3) * 2;
                            if (kk == 0) ga_mma_ss<false>(tmem + t * 128, q + o, kd + o, hi, ID_QK);
                            else ga_mma_ss<true>(tmem + t * 128, q + o, kd + o, hi, ID_QK);
                        }
                        ptx::mma_commit(sfull + t);
                    }
                    __syncwarp();
                };
                auto pv = [&](int t, int st, int part, bool first) {  // keys 64 part ..
                    const uint32_t v = v_lo + st * (F::KV_BYTES / 16), S = tmem + t * 128, O = tmem + F::O_COL + t * HDP;
                    if (ga_elect()) {
#pragma unroll
                        for (int kk = 4 * part; kk < 4 * part + 4; kk++) {
                            if (kk == 0) ga_mma_ts(O, S, v, hi, ID_PV, !first);
                            else ga_mma_ts(O, S + kk * 8, v + kk * (2048 / 16), hi, ID_PV, true);
                        }
                    }
                    __syncwarp();
                };
                auto commit = [&](uint64_t *bar) {
                    if (ga_elect()) ptx::mma_commit(bar);
                    __syncwarp();
                };
                auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
                uint32_t g = 0, n_q = 0, n_p[NT] = {}, vok_ph = 0;
                bool ok = true;
                for (int k = 0;; k++) {
                    ok = __all_sync(0xffffffffu, ok && ga_wait(itemfull + k % GA_SLOTS, (uint32_t)(k / GA_SLOTS) & 1, gave_up));
                    if (!ok) break;
                    const GaItem *it = items + k % GA_SLOTS;
                    if ((int)uniform(it->q0) < 0) break;
                    const int nt[NT] = {(int)uniform(it->nt[0]), (int)uniform(it->nt[1])};
                    const int nmax = max(nt[0], nt[1]), edge = uniform(it->edge);
                    if (lane == 0) ptx::mbar_arrive(itemfree + k % GA_SLOTS);
                    __syncwarp();
                    if (nmax == 0) continue;
                    g = uniform(g);
                    vok_ph = uniform(vok_ph);
                    ok = ga_wait(qfull, n_q++ & 1, gave_up) && ga_wait(full + g % ST, (g / ST) & 1, gave_up);
#pragma unroll
                    for (int t = 0; t < NT; t++) n_p[t] = uniform(n_p[t]);
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        continue;  // and out
                    }
                    ptx::tc_fence_after();
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        if (nt[t] > 0) qk(t, (int)(g % ST));
                    commit(free_ + g % ST);
                    g++;
                    if (nmax == 1) commit(qfree);
                    for (int j = 0; j < nmax; j++, g++) {
                        const int st = (int)(g % ST);
                        ok = ok && ga_wait(full + st, (g / ST) & 1, gave_up);
                        if (j >= edge) {
                            ok = ok && ga_wait(vok + st, (vok_ph >> st) & 1, gave_up);
                            vok_ph ^= 1u << st;
                        }
                        // after a timeout the products go on for nothing to
                        // the item's end: every wait returns at once
#pragma unroll
                        for (int t = 0; t < NT; t++)
                            if (j < nt[t]) {
                                ok = ok && ga_wait(pready + 2 * t, n_p[t] & 1, gave_up);
                                ptx::tc_fence_after();
                                pv(t, st, 0, j == 0);  // the warps that gave P have read the item's before O
                                ok = ok && ga_wait(pready + 2 * t + 1, n_p[t]++ & 1, gave_up);
                                ptx::tc_fence_after();
                                pv(t, st, 1, j == 0);
                                if (j + 1 == nt[t]) commit(ofull + t);
                                else qk(t, st);  // in order behind the product that reads P from S's columns
                            }
                        commit(free_ + st);
                        if (j + 2 == nmax) commit(qfree);
                    }
                }
                if (!ok && lane == 0) atomicOr(a.dev_err, WB_DERR_TIMEOUT_MMA);
                // Every product and its arrivals, also those that no other
                // role waits for, come before TMEM and shared memory are given
                // back (off the softmax warps' path: it costs nothing).
                commit(done);
                ptx::mbar_wait(done, 0, 200000000LL);
            }
        } else {
            // ---- V tiles at the edges: 8 threads per row, one 16-byte piece
            // of each swizzle atom each
            const int x = tid - F::W_FIX * 32;
            const uint32_t step = BF ? 0x00800080u : 0x04000400u;  // carries out of a full exponent field
            auto bad = [&](uint32_t w) { return ((w & 0x7fff7fffu) + step) & 0x80008000u; };
            auto clean = [&](uint32_t w) {
                const uint32_t m = bad(w);
                return w & ~((m & 0x8000u ? 0xffffu : 0u) | (m & 0x80000000u ? 0xffff0000u : 0u));
            };
            uint32_t g = 0, vgo_ph = 0;
            bool ok = true;
            for (int k = 0;; k++) {
                GaItem *it = items + k % GA_SLOTS;
                ok = __all_sync(0xffffffffu, ok && ga_wait(itemfull + k % GA_SLOTS, (uint32_t)(k / GA_SLOTS) & 1, gave_up));
                if (!ok || it->q0 < 0) break;
                const int nmax = max(it->nt[0], it->nt[1]), edge = it->edge, nk = it->nk;
                for (int j = edge; j < nmax; j++) {
                    const uint32_t gj = g + 1 + j;
                    const int st = (int)(gj % ST), left = nk - j * GA_KEYS;
                    ok = ok && ga_wait(vgo + st, (vgo_ph >> st) & 1, gave_up) && ga_wait(full + st, (gj / ST) & 1, gave_up);
                    vgo_ph ^= 1u << st;
                    uint8_t *v0 = sm + F::OFF_V + st * F::KV_BYTES + (x >> 3) * 128 + (x & 7) * 16;
                    for (int i0 = 0; ok && i0 < NC * 16; i0 += 8) {  // rows x / 8 + 8 i of an atom
                        uint4 v[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) v[i] = *reinterpret_cast<const uint4 *>(v0 + (i0 + i) * 1024);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int row = (x >> 3) + 8 * ((i0 + i) & 15);
                            const bool past = row >= left;
                            if (past || (bad(v[i].x) | bad(v[i].y) | bad(v[i].z) | bad(v[i].w))) {
                                *reinterpret_cast<uint4 *>(v0 + (i0 + i) * 1024) =
                                    past ? make_uint4(0, 0, 0, 0)
                                         : make_uint4(clean(v[i].x), clean(v[i].y), clean(v[i].z), clean(v[i].w));
                                if (!past) {
                                    atomicOr(&it->bad[j - edge][row >> 5], 1u << (row & 31));
                                    it->any_bad = 1;
                                }
                            }
                        }
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(vok + st);
                }
                if (nmax > 0) g += nmax + 1;
                __syncwarp();
                if (lane == 0) {
                    ptx::mbar_arrive(fixed + k % GA_SLOTS);
                    ptx::mbar_arrive(itemfree + k % GA_SLOTS);
                }
            }
            if (!ok && lane == 0) atomicOr(a.dev_err, WB_DERR_TIMEOUT_TMA);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F::R_SOFTMAX));
        // ---- softmax of tile t: thread = row
        // fp16 probabilities: 2^5 times, up to 2^13, down to 2^-29.  bf16, which
        // has fp32's range: 2^-28 times, so that up to 2^20 products with the
        // type's largest value add up in fp32.
        constexpr float SHIFT = BF ? -28.0f : 5.0f;
        const int t = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(row & 96) << 16;
        const uint32_t S = tmem + t * 128 + lanes, O = tmem + F::O_COL + t * HDP + lanes;
        const int row_tok = t * TT + row / G, row_g = row % G;
        uint32_t n_s = 0, n_o = 0;
        bool ok = true;
        for (int k = 0;; k++) {
            const GaItem *it = items + k % GA_SLOTS;
            if (!__all_sync(0xffffffffu, ga_wait(itemfull + k % GA_SLOTS, (uint32_t)(k / GA_SLOTS) & 1, gave_up))) {
                ok = false;
                break;
            }
            const int q0 = it->q0;
            if (q0 < 0) break;
            const int mine = it->nt[t], edge = it->edge, nq = it->nq, k0 = it->k0, hk = it->hk, tok = it->tok0 + row_tok;
            const bool real = row < TT * G && tok < nq;
            // rows past the tile's last query: what they hold goes nowhere, they
            // cost no masking (2 of 128 rows with 3 heads: 430 cycles a tile)
            const int vis = real ? visible(nq, it->nk, tok) : 0x7fffffff;
            float m = -INFINITY, off = 0.0f;  // reference of the exponents, and what is added to c s
            // c s + off in one operation differs from the difference of the
            // rounded c s and m by up to half an ulp of m: a factor without
            // bounds for large scores (the type's lowest value as a mask).
            // From |m| = BIG on the row's scores, whose differences are then
            // 0, an ulp's noise, or too large for the smaller key to count,
            // are multiplied by a power of two up to c instead, which is
            // exact (scores times c first, in the rows that need it: 3%
            // slower than this, 16 x 512 tokens, 8 heads of 48).
            constexpr float BIG = BF ? 268435456.0f : 16777216.0f;  // half an ulp: 2^3, 2^-1
            float shift = SHIFT;
            uint64_t c2 = ptx::f2_pack(ga.c, ga.c);
            uint64_t l2[2] = {0, 0};
            for (int j = 0; j < mine; j++, n_s++) {
                ga_wait(sfull + t, n_s & 1, gave_up);
                ptx::tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int x = 0; x < 4; x++) ptx::tmem_ld32(S + 32 * x, s[x]);
                ptx::tmem_ld_wait();
                const int lim = vis - j * GA_KEYS;
                if (__any_sync(0xffffffffu, lim < GA_KEYS)) {
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const int n = min(32, max(0, lim - 32 * x));  // columns of this piece that the row sees
                        const uint32_t seen = n == 32 ? 0xffffffffu : (1u << n) - 1;
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (!(seen & 1u << i)) s[x][i] = 0xff800000u;
                    }
                }
                float mx[4];
#pragma unroll
                for (int i = 0; i < 32; i += 2)
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const float u = __uint_as_float(s[x][i]), v = __uint_as_float(s[x][i + 1]);
                        mx[x] = i == 0 ? ga_max(u, u, v) : ga_max(mx[x], u, v);
                    }
                // a row that sees a NaN or +infinity is NaN from here on
                const float most = ga_max(ga_max(mx[0], mx[1], mx[2]), mx[3], mx[3]);
                float top = most * ga.c;
                const bool far = real && !(top <= m + 8.0f);
                if (__any_sync(0xffffffffu, far)) {
                    if (!(top < INFINITY)) top = NAN;
                    float f = 1.0f;
                    if (far) {
                        const bool big = fabsf(top) >= BIG && top > -INFINITY;
                        const float to = big ? 0.0f : SHIFT, c = big ? ga.c_two : ga.c;
                        f = m == -INFINITY ? 0.0f : ga_ex2(m - top + (to - shift));
                        m = top;
                        shift = to;
                        off = m == -INFINITY ? 0.0f : to - (big ? most * c : m);
                        c2 = ptx::f2_pack(c, c);
                    }
                    const uint64_t f2 = ptx::f2_pack(f, f);
                    l2[0] = ptx::f2_fma(l2[0], f2, 0);
                    l2[1] = ptx::f2_fma(l2[1], f2, 0);
                    if (j > 0) {
                        // S of this tile is complete, so the product before it is
#pragma unroll 1
                        for (int x = 0; x < HDP / 16; x++) {
                            uint32_t o[16];
                            ptx::tmem_ld16(O + 16 * x, o);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            ptx::tmem_st16(O + 16 * x, o);
                        }
                    }
                }
                const uint64_t off2 = ptx::f2_pack(off, off);
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        float e0, e1;
                        ptx::f2_unpack(
                            ptx::f2_fma(ptx::f2_pack(__uint_as_float(s[x][2 * i]), __uint_as_float(s[x][2 * i + 1])), c2, off2),
                            e0, e1);
                        e0 = ga_ex2(e0);
                        e1 = ga_ex2(e1);
                        l2[i & 1] = ptx::f2_add(l2[i & 1], ptx::f2_pack(e0, e1));
                        p[i] = ga_pack<T>(e0, e1);
                    }
                    ptx::tmem_st16(S + 16 * x, p);
                    if (x & 1) {  // half of the keys: their product may begin
                        ptx::tmem_st_wait();
                        ptx::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) ptx::mbar_arrive(pready + 2 * t + (x >> 1));
                    }
                }
            }
            // ---- epilogue: O / l
            float l0, l1;
            ptx::f2_unpack(ptx::f2_add(l2[0], l2[1]), l0, l1);
            // l is 0 where no key is visible or every visible score is -infinity
            const float l = l0 + l1, inv = l == 0.0f ? 0.0f : 1.0f / l;
            const bool none = vis == 0;
            const int h = hk * G + row_g;
            const long long at = (long long)(q0 + tok) * a.o_ts + (long long)h * a.o_hs;  // the row's place in out
            const uint32_t rows = __ballot_sync(0xffffffffu, real);
            // keys noted at the edges that this row may see
            ga_wait(fixed + k % GA_SLOTS, (uint32_t)(k / GA_SLOTS) & 1, gave_up);
            if (mine > 0) ga_wait(ofull + t, n_o++ & 1, gave_up);
            // 1 by now if any of the item's waits gave up
            if (__any_sync(0xffffffffu, *gave_up)) {
                ok = false;
                break;
            }
            ptx::tc_fence_after();
            const bool noted = it->any_bad;
            const int edges = max(0, mine - edge);
            // 32 columns at a time through shared memory, so that a store
            // instruction writes 64 bytes of eight rows (a thread per row
            // took 4 us): 16-byte piece c of a row at place c ^ (row / 2 & 3).
            // The loops are short: this code runs once an item and is fetched
            // anew each time (unrolled it took 1 us of an item's 3).
            uint8_t *stage = sm + F::OFF_OUT + warp * F::OUT_WARP;
#pragma unroll 1
            for (int x = 0; x < HDP / 16 && 16 * x < a.hd; x++) {
                uint32_t o[16];
                if (mine > 0) {
                    ptx::tmem_ld16(O + 16 * x, o);
                    ptx::tmem_ld_wait();
                }
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    w[i] = ga_pack<T>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                    if (none) w[i] = 0;
                }
#pragma unroll
                for (int i = 0; i < 2; i++)
                    *reinterpret_cast<uint4 *>(stage + lane * 64 + ((2 * (x & 1) + i) ^ (lane >> 1 & 3)) * 16) =
                        make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                if (!(x & 1) && 16 * x + 16 < a.hd) continue;
                __syncwarp();
                const int x0 = 32 * (x >> 1);
                if (ga.vec) {
                    const int d = x0 + 8 * (lane & 3);
#pragma unroll 1
                    for (int r = lane >> 2; r < 32; r += 8) {
                        const long long to = __shfl_sync(0xffffffffu, at, r);
                        if ((rows >> r & 1) && d < a.hd)
                            *reinterpret_cast<uint4 *>((T *)a.out + to + d) =
                                *reinterpret_cast<const uint4 *>(stage + r * 64 + ((lane & 3) ^ (r >> 1 & 3)) * 16);
                    }
                } else {
#pragma unroll 8
                    for (int r = 0; r < 32; r++) {
                        const long long to = __shfl_sync(0xffffffffu, at, r);
                        if ((rows >> r & 1) && x0 + lane < a.hd)
                            ((T *)a.out)[to + x0 + lane] =
                                *reinterpret_cast<const T *>(stage + r * 64 + ((lane >> 3) ^ (r >> 1 & 3)) * 16 + (lane & 7) * 2);
                    }
                }
                __syncwarp();
            }
            // Values at the edges that are not finite: the sum is whatever
            // they make of it.
            if (noted && real) {
#pragma unroll 1
                for (int i = 0; i < edges * GA_KEYS; i++) {
                    const int key = edge * GA_KEYS + i;
                    if (key >= vis || !(it->bad[i / GA_KEYS][(i >> 5) & 3] >> (i & 31) & 1)) continue;
                    const T *v = (const T *)a.v + (long long)(k0 + key) * a.v_ts + (long long)hk * a.v_hs;
                    T *o = (T *)a.out + at;
#pragma unroll 1
                    for (int d = 0; d < a.hd; d++) {
                        const float y = to_f(v[d]);
                        if (!isfinite(y)) o[d] = from_f<T>(to_f(o[d]) + (l == 0.0f ? l * y : y));
                    }
                }
            }
            if (real && a.lse)
                a.lse[(long long)h * a.total_q + q0 + tok] = none ? -INFINITY : (log2f(l) - shift + m) * 0.6931471805599453f;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(itemfree + k % GA_SLOTS);
        }
        if (!ok && lane == 0) atomicOr(a.dev_err, WB_DERR_TIMEOUT_SOFTMAX);
    }
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    // When some role gave up, copies may be under way, whichever it was and
    // whether or not warp W_TMA had finished: they land before the shared
    // memory is given back.  (Else the products have waited for each of them.)
    if (*gave_up && warp == F::W_TMA && lane == 0) {
        if (nq_loads > 0) ptx::mbar_wait(qfull, (nq_loads - 1) & 1, 200000000LL);
        for (uint32_t i = g > ST ? g - ST : 0; i < g; i++) ptx::mbar_wait(full + i % ST, (i / ST) & 1, 200000000LL);
    }
    __syncwarp();
    if (warp == F::W_MMA) ptx::tmem_dealloc(tmem, F::TMEM);
}

// ---- rows that TMA cannot read --------------------------------------------
// A tensor map wants a 16-byte aligned base and strides of whole 16 bytes.
// Other rows (odd offsets, head_dim 42 back to back, heads spread by a zero
// stride) are first copied to rows of 8-element multiples; a negative scale
// is moved into the queries there.
static bool ga_aligned(const void *p, long long ts, long long hs, int heads) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ts > 0 && ts % 8 == 0 && (heads == 1 || (hs > 0 && hs % 8 == 0));
}
static long long ga_copy_elems(long long rows, int heads, int hd) { return rows * heads * ((hd + 7) & ~7); }
struct GaCopies {
    bool q, k, v;
    size_t oq, ok, ov, bytes;
};
static GaCopies ga_copies(const GqaAttnArgs &a) {
    GaCopies c{};
    c.q = a.scale < 0.0f || !ga_aligned(a.q, a.q_ts, a.q_hs, a.H);
    c.k = a.total_k && !ga_aligned(a.k, a.k_ts, a.k_hs, a.Hkv);
    c.v = a.total_k && !ga_aligned(a.v, a.v_ts, a.v_hs, a.Hkv);
    Carve cv;
    c.oq = c.q ? cv.take<uint16_t>(ga_copy_elems(a.total_q, a.H, a.hd)) : 0;
    c.ok = c.k ? cv.take<uint16_t>(ga_copy_elems(a.total_k, a.Hkv, a.hd)) : 0;
    c.ov = c.v ? cv.take<uint16_t>(ga_copy_elems(a.total_k, a.Hkv, a.hd)) : 0;
    c.bytes = cv.off;
    return c;
}

size_t gqa_attention_scratch(const GqaAttnArgs &a, int) { return ga_copies(a).bytes; }

struct GaCopyJob {
    const uint16_t *src;
    uint4 *dst;
    long long ts, hs, n;  // n: pieces of 8 elements
    int heads;
    uint32_t flip;        // 0x8000 changes the sign
};
struct GaCopyJobs {
    GaCopyJob job[3];
    int hd;
};
// One thread per 8 output elements, all the rows to copy in one launch.
__global__ void __launch_bounds__(256) gqa_rows_kernel(GaCopyJobs js) {
    const int per = (js.hd + 7) / 8;
    long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    int which = 0;
    while (which < 3 && i >= js.job[which].n) i -= js.job[which++].n;
    if (which == 3) return;
    const GaCopyJob &j = js.job[which];
    const long long rh = gqa_quotient(i, per), row = gqa_quotient(rh, j.heads);
    const int d0 = (int)(i - rh * per) * 8;
    const uint16_t *p = j.src + row * j.ts + (rh - row * j.heads) * j.hs;
    uint32_t w[4];
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const uint32_t lo = d0 + 2 * x < js.hd ? p[d0 + 2 * x] ^ j.flip : 0;
        const uint32_t hi = d0 + 2 * x + 1 < js.hd ? p[d0 + 2 * x + 1] ^ j.flip : 0;
        w[x] = lo | hi << 16;
    }
    j.dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
}

template <class T, int HDP>
static int ga_launch(const GaArgs &ga, int sm_count, cudaStream_t st, std::string *msg) {
    using F = GaConf<HDP>;
    const GqaAttnArgs &a = ga.a;
    const CUtensorMapDataType dt =
        __is_same(T, __nv_bfloat16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap tq, tk, tv;
    int rc;
    const uint64_t q_hs = a.H == 1 ? 16 : (uint64_t)a.q_hs * 2, q_gs = ga.G == 1 ? 16 : q_hs;
    const uint64_t qd[4] = {(uint64_t)a.hd, (uint64_t)ga.G, (uint64_t)a.Hkv, (uint64_t)a.total_q};
    const uint64_t qs[3] = {q_gs, a.Hkv == 1 ? 16 : q_hs * ga.G, (uint64_t)a.q_ts * 2};
    const uint32_t qb[4] = {64, (uint32_t)ga.G, 1, (uint32_t)ga.TT};
    if ((rc = make_tmap(&tq, a.q, dt, 4, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B, msg))) return rc;
    if (a.total_k) {
        const uint64_t kd[3] = {(uint64_t)a.hd, (uint64_t)a.Hkv, (uint64_t)a.total_k};
        const uint32_t kb[3] = {64, 1, GA_KEYS};
        const uint64_t ks[2] = {a.Hkv == 1 ? 16 : (uint64_t)a.k_hs * 2, (uint64_t)a.k_ts * 2};
        const uint64_t vs[2] = {a.Hkv == 1 ? 16 : (uint64_t)a.v_hs * 2, (uint64_t)a.v_ts * 2};
        if ((rc = make_tmap(&tk, a.k, dt, 3, kd, ks, kb, CU_TENSOR_MAP_SWIZZLE_128B, msg))) return rc;
        if ((rc = make_tmap(&tv, a.v, dt, 3, kd, vs, kb, CU_TENSOR_MAP_SWIZZLE_128B, msg))) return rc;
    } else {  // never loaded from
        tk = tv = tq;
    }
    static std::atomic<uint64_t> done{0};
    const cudaError_t set = gqa_smem_limit(gqa_attn_kernel<T, HDP>, F::BYTES, done);
    if (set != cudaSuccess) {
        *msg = std::string("attention kernel attributes: ") + cudaGetErrorString(set);
        return WB_ECUDA;
    }
    ProfScope ps("gqa_attn", st);
    const unsigned grid = (unsigned)std::min<long long>(ga.items * a.Hkv, sm_count);
    gqa_attn_kernel<T, HDP><<<grid, F::THREADS, F::BYTES, st>>>(tq, tk, tv, ga);
    return WB_OK;
}

int launch_gqa_attention(const GqaAttnArgs &args, int dtype, void *scratch, int sm_count, cudaStream_t st,
                         std::string *msg) {
    GaArgs ga{args, 0.0f, 0.0f, args.H / args.Hkv, 0, 0, 0};
    GqaAttnArgs &a = ga.a;
    ga.TT = GA_ROWS / ga.G;
    // at most this many, whatever the sequences' lengths are
    ga.items = std::min(a.total_q, a.total_q / (2 * ga.TT) + a.n_seq);
    // 0 would turn a hidden key's -inf into NaN; times the smallest subnormal
    // every finite score is 0, to 2^-21
    ga.c = std::max(fabsf(a.scale) * 1.4426950408889634f, 1.40129846e-45f);
    int up;
    frexpf(ga.c, &up);  // c / 2^up is in [0.5, 1)
    ga.c_two = ldexpf(0.5f, up);
    ga.vec = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.o_ts % 8 == 0 && a.o_hs % 8 == 0 && a.hd % 8 == 0;
    const GaCopies cp = ga_copies(args);
    if (cp.q || cp.k || cp.v) {
        GaCopyJobs js{};
        js.hd = a.hd;
        long long n = 0;
        auto job = [&](GaCopyJob &j, const void *&p, long long &ts, long long &hs, long long rows, int heads, uint32_t flip,
                       size_t off) {
            j = GaCopyJob{(const uint16_t *)p, (uint4 *)((char *)scratch + off), ts, hs, ga_copy_elems(rows, heads, a.hd) / 8,
                          heads, flip};
            n += j.n;
            p = j.dst;
            hs = (a.hd + 7) & ~7;
            ts = hs * heads;
        };
        if (cp.q) job(js.job[0], a.q, a.q_ts, a.q_hs, a.total_q, a.H, a.scale < 0.0f ? 0x8000 : 0, cp.oq);
        if (cp.k) job(js.job[1], a.k, a.k_ts, a.k_hs, a.total_k, a.Hkv, 0, cp.ok);
        if (cp.v) job(js.job[2], a.v, a.v_ts, a.v_hs, a.total_k, a.Hkv, 0, cp.ov);
        if ((n + 255) / 256 > 0x7fffffffLL) {
            *msg = "too many rows to copy";
            return WB_EINVAL;
        }
        ProfScope ps("gqa_rows", st);
        gqa_rows_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(js);
    }
    // rows of up to 64 in 64 columns (in 128: 71.5 us instead of 61.3, packed
    // 768-wide batch; 26.4 instead of 21.2, 16 x 512 tokens of 48)
    if (dtype == WB_BF16)
        return a.hd <= 64 ? ga_launch<__nv_bfloat16, 64>(ga, sm_count, st, msg) : ga_launch<__nv_bfloat16, 128>(ga, sm_count, st, msg);
    return a.hd <= 64 ? ga_launch<__half, 64>(ga, sm_count, st, msg) : ga_launch<__half, 128>(ga, sm_count, st, msg);
}

}  // namespace wb
