// wb_gqa_cache.cu -- the paged key-value cache of the grouped-head
// attention: writing (with quantisation to 8 bits) and reading back.
//
// A position's head of hd values x is stored as they are, or with one scale
//   scale = max(max|x| * (1 / top), 2^-126),  top = 127 (int8), 448 (e4m3),
//   stored = round(x / scale) to the nearest representable, ties to even
//            (saturating),
// in fp32 (an IEEE division, 1 / top the nearest float), and reads back as
// stored * scale.  The lower limit keeps a head of zeros (and of the smallest
// subnormals) off 0 / 0.
//
// Both directions move bytes: a lane takes 16 values of a row when writing
// (the row's scale and place cost as much as its values with 8), 8 when
// reading, four rows a thread under way at once.  The rows of a
// block are loaded before their places in the cache are looked up (sequence,
// slot, start, page: dependent loads that take as long as the data).
// 8 x 4096 positions of 8 heads x 128, fp16 to e4m3 and back: 43.4 + 35.1 us
// apart, 75 us in a row (203 MB each way, 5.4 TB/s of 6.5; below it stays what
// a warp has to do a row: the maximum over its lanes, the quotients); as they
// are 48.5 + 44.2 us apart, 93 in a row (5.8 TB/s).  One
// position of 32 sequences: 7.2 us for both, launches and the dependent loads.
#include "wb_gqa.h"

#include <algorithm>

namespace wb {

struct GqaMove {
    GqaCacheArgs c;
    const int32_t *cu, *start;
    void *k, *v;
    long long k_ts, k_hs, v_ts, v_hs, total;
    int append;  // start == nullptr: from the slots' lengths (1) or from position 0 (0)
    int vec;     // rows of k and v take 16-byte accesses
    unsigned int *ticket;  // zero; the append's last block sets the lengths
    uint32_t inv;          // 2^32 / Hkv rounded up
};

static constexpr int GM_THREADS = 128, GM_ROWS = 4;  // rows of a thread
static constexpr int GM_CTAS = 8;  // write blocks per SM (256 threads and 4 blocks: 77 us instead of 75, 64 and 16: 82)

// Row `local` of a block (counted from its first token's first head): token
// and head.  inv = 2^32 / Hkv rounded up, so the quotient is right or one
// too large.
__device__ __forceinline__ void gm_row(uint32_t local, int Hkv, uint32_t inv, int *t, int *h) {
    uint32_t q = Hkv == 1 ? local : __umulhi(local, inv);
    if (q * Hkv > local) q--;
    *t = (int)q;
    *h = (int)(local - q * Hkv);
}

__device__ __forceinline__ long long gqa_start(const GqaMove &m, int b, int slot) {
    return m.start ? m.start[b] : m.append ? m.c.lens[slot] : 0;
}

// Sequence b's rows lie inside the tensors.
__device__ __forceinline__ bool gqa_rows_fit(const GqaMove &m, int b) {
    const int r0 = m.cu[b], r1 = m.cu[b + 1];
    return r0 >= 0 && r1 >= r0 && r1 <= m.total;
}

// The row index of packed token t's position (page, head 0), or -1 outside
// the cache or when the sequence's rows do not all lie inside the tensors.
__device__ __forceinline__ long long gqa_place(const GqaMove &m, long long t) {
    const GqaCacheArgs &c = m.c;
    int b = (int)t;
    long long i = 0, end = t + 1;
    if (m.cu) {
        b = gqa_find_seq(m.cu, c.n_seq, t);
        i = t - m.cu[b];
        end = m.cu[b + 1];
    }
    const int slot = c.slots ? c.slots[b] : b;
    if (slot < 0 || slot >= c.n_slots || i < 0 || t >= end || end > m.total) return -1;
    const long long s0 = gqa_start(m, b, slot);
    const long long pos = s0 + i;
    if (s0 < 0 || pos >= (long long)c.max_pages * WB_PAGE) return -1;
    const int pg = c.table[(long long)slot * c.max_pages + (pos >> WB_PAGE_SHIFT)];
    if (pg < 0 || pg >= c.n_pages) return -1;
    return (long long)pg * c.Hkv * WB_PAGE + (pos & (WB_PAGE - 1));
}

// lens[slot] = the position after sequence b's last token, when its rows are
// there and all its positions have a page.
__device__ __forceinline__ void gqa_set_len(const GqaMove &m, int b) {
    const GqaCacheArgs &c = m.c;
    if (m.cu && !gqa_rows_fit(m, b)) {
        atomicOr(c.dev_err, WB_DERR_BOUNDS);  // no row of it may have been looked at
        return;
    }
    const long long n = m.cu ? (long long)m.cu[b + 1] - m.cu[b] : 1;
    const int slot = c.slots ? c.slots[b] : b;
    if (slot < 0 || slot >= c.n_slots) return;
    const long long s0 = gqa_start(m, b, slot), end = s0 + n;
    if (s0 < 0 || end > (long long)c.max_pages * WB_PAGE) return;
    for (long long p = s0 >> WB_PAGE_SHIFT; p << WB_PAGE_SHIFT < end; p++) {
        const int pg = c.table[(long long)slot * c.max_pages + p];
        if (pg < 0 || pg >= c.n_pages) return;
    }
    c.lens[slot] = (int)end;
}

// 8 values of 16 bits as four pairs of fp32
template <class T>
__device__ __forceinline__ void gm_floats(const uint4 &x, uint64_t *f) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (__is_same(T, __nv_bfloat16)) {
            f[i] = ptx::f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        } else {
            const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            f[i] = ptx::f2_pack(v.x, v.y);
        }
    }
}

// 8 values y, a pair's low one first, rounded to S
template <class S>
__device__ __forceinline__ uint2 gm_round(const uint64_t *y) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        float a, b, c, d;
        ptx::f2_unpack(y[2 * i], a, b);
        ptx::f2_unpack(y[2 * i + 1], c, d);
        if constexpr (__is_same(S, int8_t)) {
            // y + 1.5 2^23 has the integer in its low bits
            const uint64_t big = ptx::f2_pack(12582912.0f, 12582912.0f);
            ptx::f2_unpack(ptx::f2_add(y[2 * i], big), a, b);
            ptx::f2_unpack(ptx::f2_add(y[2 * i + 1], big), c, d);
            w[i] = __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                               __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
        } else {
            uint16_t lo, hi;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
            w[i] = lo | (uint32_t)hi << 16;
        }
    }
    return make_uint2(w[0], w[1]);
}

// The 16 values x / scale rounded to S.  The quotient's rounding to fp32 counts
// (ties are frequent among 8- and 11-bit inputs): with r = 1 / scale rounded
// to nearest and q = x r, the remainder x - q scale is exact in a fused
// multiply-add and q + (x - q scale) r rounds to the quotient (P. Markstein,
// IBM J. Res. Dev. 34, 1990), three packed operations a pair.  Scales so
// small that the remainder could underflow, or not finite, take the division
// instruction sequence.
template <class S>
__device__ __forceinline__ void gm_quantise(const uint64_t (&x)[8], float scale, uint2 (&w)[2]) {
    uint64_t y[8];
    if (scale > 1e-30f && scale < 1e35f) {
        const float r = __frcp_rn(scale);
        const uint64_t r2 = ptx::f2_pack(r, r), n2 = ptx::f2_pack(-scale, -scale);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint64_t q = ptx::f2_mul(x[i], r2);
            y[i] = ptx::f2_fma(ptx::f2_fma(q, n2, x[i]), r2, q);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float a, b;
            ptx::f2_unpack(x[i], a, b);
            a = __fdiv_rn(a, scale);
            b = __fdiv_rn(b, scale);
            // a head with a value that is not finite: its scale makes the
            // others NaN when read, whatever is stored
            if (__is_same(S, int8_t)) {
                a = isfinite(a) ? a : 0.0f;
                b = isfinite(b) ? b : 0.0f;
            }
            y[i] = ptx::f2_pack(a, b);
        }
    }
    w[0] = gm_round<S>(y);
    w[1] = gm_round<S>(y + 4);
}

// the larger of 16-bit pairs
__device__ __forceinline__ uint32_t gm_max16(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("max.u16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}

// two stored values (bytes 2 i, 2 i + 1 of w) as fp32
template <class S>
__device__ __forceinline__ uint64_t gm_stored(uint32_t w, int i) {
    if constexpr (__is_same(S, int8_t)) {
        // 2^23 + (value + 128), less 2^23 + 128
        const uint32_t u = w ^ 0x80808080u;
        return ptx::f2_add(ptx::f2_pack(__uint_as_float(__byte_perm(u, 0x4b000000u, i ? 0x7652 : 0x7650)),
                                        __uint_as_float(__byte_perm(u, 0x4b000000u, i ? 0x7653 : 0x7651))),
                           ptx::f2_pack(-8388736.0f, -8388736.0f));
    } else {
        uint32_t h;
        const uint16_t b = (uint16_t)(i ? w >> 16 : w);
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(b));
        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&h));
        return ptx::f2_pack(v.x, v.y);
    }
}

template <class T>
__device__ __forceinline__ uint32_t gm_pack(uint64_t v) {
    float a, b;
    ptx::f2_unpack(v, a, b);
    uint32_t r;
    if (__is_same(T, __nv_bfloat16)) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// One block: GM_THREADS / LPR x GM_ROWS rows (token, head) of k (blockIdx.y = 0)
// or v; a lane has 16 values of a row.
template <class T, class S, int LPR>
__global__ void __launch_bounds__(GM_THREADS, GM_CTAS) gqa_write_kernel(GqaMove m) {
    const GqaCacheArgs &c = m.c;
    constexpr int SIDE = GM_THREADS / LPR, ROWS = SIDE * GM_ROWS;
    __shared__ long long s_place[ROWS + 1];
    __shared__ int s_last;
    const int tid = threadIdx.x, piece = tid % LPR, d0 = piece * 16;
    const bool v = blockIdx.y;
    const long long r0 = (long long)blockIdx.x * ROWS, t0 = gqa_quotient(r0, c.Hkv), rest = m.total * c.Hkv - t0 * c.Hkv;
    // rows from t0's first on: this thread's first, and how many there are
    const uint32_t l0 = (uint32_t)(r0 - t0 * c.Hkv) + tid / LPR, left = (uint32_t)min(rest, 1LL << 30);
    const long long ts = v ? m.v_ts : m.k_ts, hs = v ? m.v_hs : m.k_hs;
    const uint16_t *in = (const uint16_t *)(v ? m.v : m.k) + t0 * ts + d0;
    gqa_wait();
    // ---- loads
    uint4 x[GM_ROWS][2];
#pragma unroll
    for (int u = 0; u < GM_ROWS; u++) {
        int t, h;
        gm_row(l0 + u * SIDE, c.Hkv, m.inv, &t, &h);
        x[u][0] = x[u][1] = make_uint4(0, 0, 0, 0);
        if (l0 + u * SIDE < left && d0 < c.hd) {
            const uint16_t *p = in + t * ts + h * hs;
            if (m.vec && d0 + 16 <= c.hd) {
                x[u][0] = __ldcs(reinterpret_cast<const uint4 *>(p));
                x[u][1] = __ldcs(reinterpret_cast<const uint4 *>(p) + 1);
            } else {
                uint32_t e[16];
#pragma unroll
                for (int i = 0; i < 16; i++) e[i] = d0 + i < c.hd ? p[i] : 0;
#pragma unroll
                for (int i = 0; i < 2; i++)
                    x[u][i] = make_uint4(e[8 * i] | e[8 * i + 1] << 16, e[8 * i + 2] | e[8 * i + 3] << 16,
                                         e[8 * i + 4] | e[8 * i + 5] << 16, e[8 * i + 6] | e[8 * i + 7] << 16);
            }
        }
    }
    // ---- places of the block's tokens
    const int nt = (int)min(m.total - t0, (long long)(((uint32_t)(r0 - t0 * c.Hkv) + ROWS + c.Hkv - 1) / (uint32_t)c.Hkv));
    for (int i = tid; i < nt; i += GM_THREADS) {
        const long long p = gqa_place(m, t0 + i);
        s_place[i] = p;
        if (p < 0) atomicOr(c.dev_err, WB_DERR_BOUNDS);
    }
    __syncthreads();
    S *pages = (S *)(v ? c.v_pages : c.k_pages) + d0;
    float *scales = v ? c.v_scale : c.k_scale;
#pragma unroll
    for (int u = 0; u < GM_ROWS; u++) {
        int t, h;
        gm_row(l0 + u * SIDE, c.Hkv, m.inv, &t, &h);
        const long long place = l0 + u * SIDE < left ? s_place[t] : -1;
        const long long row = place + h * WB_PAGE;
        S *dst = pages + row * c.row;
        if constexpr (sizeof(S) == 2) {
            if (place >= 0 && d0 < c.row) {
                *reinterpret_cast<uint4 *>(dst) = x[u][0];
                *reinterpret_cast<uint4 *>(dst + 8) = x[u][1];
            }
        } else {
            // |x| as integers, 16 bits each: NaN above infinity above the rest
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint4 &w = x[u][i];
                const uint32_t a16 = 0x7fff7fffu;
                top = gm_max16(top, gm_max16(gm_max16(w.x & a16, w.y & a16), gm_max16(w.z & a16, w.w & a16)));
            }
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) top = gm_max16(top, __shfl_xor_sync(0xffffffffu, top, o));
            const uint16_t most = (uint16_t)max(top & 0xffffu, top >> 16);
            float scale = __fmul_rn(to_f(*reinterpret_cast<const T *>(&most)), __is_same(S, int8_t) ? 1.0f / 127.0f : 1.0f / 448.0f);
            scale = scale < 1.17549435e-38f ? 1.17549435e-38f : scale;
            if (place >= 0 && d0 < c.row) {
                uint64_t f[8];
                gm_floats<T>(x[u][0], f);
                gm_floats<T>(x[u][1], f + 4);
                uint2 w[2];
                gm_quantise<S>(f, scale, w);
                *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
                if (piece == 0) scales[row] = scale;
            }
        }
    }
    // ---- lengths: with given starts by the first block, else by the last to
    // get here, when every block has read them
    int last = blockIdx.x == 0 && blockIdx.y == 0;
    if (!m.start) {
        __syncthreads();
        if (tid == 0) s_last = atomicAdd(m.ticket, 1) == gridDim.x * gridDim.y - 1;
        __syncthreads();
        last = s_last;
        if (last && tid == 0) *m.ticket = 0;
    }
    if (last)
        for (int b = tid; b < c.n_seq; b += GM_THREADS) gqa_set_len(m, b);
}

template <class T, class S, int LPR>
__global__ void __launch_bounds__(GM_THREADS) gqa_read_kernel(GqaMove m) {
    const GqaCacheArgs &c = m.c;
    constexpr int SIDE = GM_THREADS / LPR, ROWS = SIDE * GM_ROWS;
    __shared__ long long s_place[ROWS + 1];
    const int tid = threadIdx.x, piece = tid % LPR, d0 = piece * 8;
    const bool v = blockIdx.y;
    const long long r0 = (long long)blockIdx.x * ROWS, t0 = gqa_quotient(r0, c.Hkv), rest = m.total * c.Hkv - t0 * c.Hkv;
    const uint32_t l0 = (uint32_t)(r0 - t0 * c.Hkv) + tid / LPR, left = (uint32_t)min(rest, 1LL << 30);
    const int nt = (int)min(m.total - t0, (long long)(((uint32_t)(r0 - t0 * c.Hkv) + ROWS + c.Hkv - 1) / (uint32_t)c.Hkv));
    gqa_wait();
    for (int i = tid; i < nt; i += GM_THREADS) {
        const long long p = gqa_place(m, t0 + i);
        s_place[i] = p;
        if (p < 0) atomicOr(c.dev_err, WB_DERR_BOUNDS);
    }
    // starts that leave out rows, or sequences that no row belongs to
    if (m.cu && blockIdx.x + blockIdx.y == 0 && tid == GM_THREADS - 1 && (m.cu[0] != 0 || m.cu[c.n_seq] != m.total))
        atomicOr(c.dev_err, WB_DERR_BOUNDS);
    __syncthreads();
    const S *pages = (const S *)(v ? c.v_pages : c.k_pages) + d0;
    const float *scales = v ? c.v_scale : c.k_scale;
    uint4 x[GM_ROWS];
    float scale[GM_ROWS];
#pragma unroll
    for (int u = 0; u < GM_ROWS; u++) {
        int t, h;
        gm_row(l0 + u * SIDE, c.Hkv, m.inv, &t, &h);
        x[u] = make_uint4(0, 0, 0, 0);
        scale[u] = 0.0f;
        const long long place = l0 + u * SIDE < left ? s_place[t] : -1;
        if (place < 0 || d0 >= c.hd) continue;
        const long long row = place + h * WB_PAGE;
        if constexpr (sizeof(S) == 2) {
            x[u] = *reinterpret_cast<const uint4 *>(pages + row * c.row);
        } else {
            const uint2 q = *reinterpret_cast<const uint2 *>(pages + row * c.row);
            x[u].x = q.x;
            x[u].y = q.y;
            scale[u] = scales[row];
        }
    }
    uint16_t *out = (uint16_t *)(v ? m.v : m.k) + (r0 + tid / LPR) * c.hd + d0;
#pragma unroll
    for (int u = 0; u < GM_ROWS; u++) {
        if (l0 + u * SIDE >= left || d0 >= c.hd) continue;
        uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
        if constexpr (sizeof(S) == 1) {
            // a position outside the pages reads 0
            const uint64_t sc = ptx::f2_pack(scale[u], scale[u]);
            const uint32_t q[2] = {w[0], w[1]};
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = gm_pack<T>(ptx::f2_mul(gm_stored<S>(q[i >> 1], i & 1), sc));
        }
        uint16_t *dst = out + u * SIDE * c.hd;
        if (m.vec && d0 + 8 <= c.hd) {
            __stcs(reinterpret_cast<uint4 *>(dst), make_uint4(w[0], w[1], w[2], w[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (d0 + i < c.hd) dst[i] = (uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1]);
        }
    }
}

template <class F>
static void by_types(int dtype, int store, F &&f) {
    if (dtype == WB_BF16) {
        if (store == WB_INT8) f(__nv_bfloat16{}, int8_t{});
        else if (store == WB_E4M3) f(__nv_bfloat16{}, __nv_fp8_e4m3{});
        else f(__nv_bfloat16{}, __nv_bfloat16{});
    } else {
        if (store == WB_INT8) f(__half{}, int8_t{});
        else if (store == WB_E4M3) f(__half{}, __nv_fp8_e4m3{});
        else f(__half{}, __half{});
    }
}

// lanes of a row (16 values each in the write, 8 in the read) and blocks of a
// move
static int gm_lanes(int row) { return row <= 32 ? 2 : row <= 64 ? 4 : 8; }
static long long gm_blocks(const GqaMove &m, int lanes) {
    const long long per = (long long)GM_THREADS / lanes * GM_ROWS;
    return (m.total * m.c.Hkv + per - 1) / per;
}
static uint32_t gm_inv(int n) { return (uint32_t)((((unsigned long long)1 << 32) + n - 1) / n); }
static bool gm_vec(const void *p, long long ts, long long hs) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ts % 8 == 0 && hs % 8 == 0;
}

int launch_gqa_cache_write(const GqaCacheArgs &c, int dtype, const int32_t *cu, long long total, const int32_t *start,
                           const void *k, const void *v, long long k_ts, long long k_hs, long long v_ts, long long v_hs,
                           unsigned int *ticket, cudaStream_t st, std::string *msg) {
    GqaMove m{c, cu, start, (void *)k, (void *)v, k_ts, k_hs, v_ts, v_hs, total, 1,
              gm_vec(k, k_ts, k_hs) && gm_vec(v, v_ts, v_hs), ticket, gm_inv(c.Hkv)};
    const int l = gm_lanes(c.row);
    const long long blocks = std::max(1LL, gm_blocks(m, l));  // one for the lengths at least
    if (blocks > 0x7fffffffLL) {
        *msg = "too many cache rows";
        return WB_EINVAL;
    }
    ProfScope ps("gqa_write", st);
    by_types(dtype, c.store, [&](auto t, auto s) {
        using T = decltype(t);
        using S = decltype(s);
        if (l == 2) gqa_launch(gqa_write_kernel<T, S, 2>, dim3((unsigned)blocks, 2), GM_THREADS, 0, st, m);
        else if (l == 4) gqa_launch(gqa_write_kernel<T, S, 4>, dim3((unsigned)blocks, 2), GM_THREADS, 0, st, m);
        else gqa_launch(gqa_write_kernel<T, S, 8>, dim3((unsigned)blocks, 2), GM_THREADS, 0, st, m);
    });
    return WB_OK;
}

int launch_gqa_cache_read(const GqaCacheArgs &c, int dtype, const int32_t *cu, long long total, const int32_t *start,
                          void *k, void *v, cudaStream_t st, std::string *msg) {
    GqaMove m{c, cu, start, k, v, 0, 0, 0, 0, total, 0, gm_vec(k, c.hd, c.hd) && gm_vec(v, c.hd, c.hd), nullptr, gm_inv(c.Hkv)};
    const int l = 2 * gm_lanes(c.row);
    const long long blocks = gm_blocks(m, l);
    if (blocks > 0x7fffffffLL) {
        *msg = "too many cache rows";
        return WB_EINVAL;
    }
    if (blocks == 0) return WB_OK;
    ProfScope ps("gqa_read", st);
    by_types(dtype, c.store, [&](auto t, auto s) {
        using T = decltype(t);
        using S = decltype(s);
        if (l == 4) gqa_launch(gqa_read_kernel<T, S, 4>, dim3((unsigned)blocks, 2), GM_THREADS, 0, st, m);
        else if (l == 8) gqa_launch(gqa_read_kernel<T, S, 8>, dim3((unsigned)blocks, 2), GM_THREADS, 0, st, m);
        else gqa_launch(gqa_read_kernel<T, S, 16>, dim3((unsigned)blocks, 2), GM_THREADS, 0, st, m);
    });
    return WB_OK;
}

}  // namespace wb
