// wb_gqa_cache.cu -- the paged key-value cache of the grouped-head
// attention: writing (with quantisation to 8 bits) and reading back.
//
// A position's head of hd values x is stored as they are, or with one scale
//   scale = max(max|x| * (1 / top), 2^-126),  top = 127 (int8), 448 (e4m3),
//   stored = round(x / scale) to the nearest representable, ties to even
//            (saturating),
// in fp32 (an IEEE division, 1 / top the nearest float), and reads back as
// stored * scale.  The
// lower limit keeps a head of zeros (and of the smallest subnormals) off
// 0 / 0.
#include "wb_gqa.h"

namespace wb {

struct GqaMove {
    GqaCacheArgs c;
    const int32_t *cu, *start;
    void *k, *v;
    long long k_ts, k_hs, v_ts, v_hs, total;
    int append;  // start == nullptr: from the slots' lengths (1) or from position 0 (0)
};

__device__ __forceinline__ long long gqa_start(const GqaMove &m, int b, int slot) {
    return m.start ? m.start[b] : m.append ? m.c.lens[slot] : 0;
}

// Sequence and cache position of packed token t; the flat row index of
// (page, head 0, position) in units of rows, or -1 (flagged) outside the
// cache.
__device__ __forceinline__ long long gqa_place(const GqaMove &m, long long t, int *len_out) {
    const GqaCacheArgs &c = m.c;
    int b = (int)t;
    long long i = 0, n = 1;
    if (m.cu) {
        b = gqa_find_seq(m.cu, c.n_seq, t);
        i = t - m.cu[b];
        n = (long long)m.cu[b + 1] - m.cu[b];
    }
    const int slot = c.slots ? c.slots[b] : b;
    *len_out = -1;
    if (slot < 0 || slot >= c.n_slots || i < 0 || i >= n) return -1;
    const long long s0 = gqa_start(m, b, slot);
    const long long pos = s0 + i;
    if (s0 < 0 || pos >= (long long)c.max_pages * WB_PAGE) return -1;
    const int pg = c.table[(long long)slot * c.max_pages + (pos >> WB_PAGE_SHIFT)];
    if (pg < 0 || pg >= c.n_pages) return -1;
    if (i == n - 1) *len_out = (int)(pos + 1);
    return (long long)pg * c.Hkv * WB_PAGE + (pos & (WB_PAGE - 1));
}

__device__ __forceinline__ uint32_t warp_max_u(uint32_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// One warp per (token, key-value head).
template <class T, class S>
__global__ void __launch_bounds__(128) gqa_write_kernel(GqaMove m) {
    const GqaCacheArgs &c = m.c;
    const long long wid = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (wid >= m.total * c.Hkv) return;
    const long long t = wid / c.Hkv;
    const int h = (int)(wid - t * c.Hkv);
    int len;
    const long long place = gqa_place(m, t, &len);
    if (place < 0) {
        if (lane == 0) atomicOr(c.dev_err, WB_DERR_BOUNDS);
        return;
    }
    const long long r = place + (long long)h * WB_PAGE;
    constexpr bool quant = sizeof(S) == 1;
    for (int which = 0; which < 2; which++) {
        const T *x = which ? (const T *)m.v + t * m.v_ts + h * m.v_hs : (const T *)m.k + t * m.k_ts + h * m.k_hs;
        S *d = (S *)(which ? c.v_pages : c.k_pages) + r * c.row;
        float f[4];
        uint32_t top = 0;  // |x| as bits: orders NaN above infinity above the rest
        for (int i = 0; i < 4; i++) {
            f[i] = lane + 32 * i < c.hd ? to_f(x[lane + 32 * i]) : 0.0f;
            top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
        }
        float scale = 1.0f;
        if (quant) {
            const float amax = __uint_as_float(warp_max_u(top));
            scale = __fmul_rn(amax, c.store == WB_INT8 ? 1.0f / 127.0f : 1.0f / 448.0f);
            scale = scale < 1.17549435e-38f ? 1.17549435e-38f : scale;
            if (lane == 0) (which ? c.v_scale : c.k_scale)[r] = scale;
        }
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < c.row) d[lane + 32 * i] = from_f<S>(quant ? __fdiv_rn(f[i], scale) : f[i]);
    }
}

// lens[slot] = the position after each sequence's last token.
__global__ void gqa_len_kernel(GqaMove m) {
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= m.c.n_seq) return;
    const long long n = m.cu ? (long long)m.cu[b + 1] - m.cu[b] : 1;
    const int slot = m.c.slots ? m.c.slots[b] : b;
    if (slot < 0 || slot >= m.c.n_slots || n < 0) return;
    const long long s0 = gqa_start(m, b, slot);
    const long long end = s0 + n;
    if (s0 < 0 || end > (long long)m.c.max_pages * WB_PAGE) return;
    for (long long p = s0 >> WB_PAGE_SHIFT; p << WB_PAGE_SHIFT < end; p++) {
        const int pg = m.c.table[(long long)slot * m.c.max_pages + p];
        if (pg < 0 || pg >= m.c.n_pages) return;
    }
    m.c.lens[slot] = (int)end;
}

template <class T, class S>
__global__ void __launch_bounds__(128) gqa_read_kernel(GqaMove m) {
    const GqaCacheArgs &c = m.c;
    const long long wid = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (wid >= m.total * c.Hkv) return;
    const long long t = wid / c.Hkv;
    const int h = (int)(wid - t * c.Hkv);
    int len;
    const long long place = gqa_place(m, t, &len);
    if (place < 0 && lane == 0) atomicOr(c.dev_err, WB_DERR_BOUNDS);
    const long long r = place + (long long)h * WB_PAGE;
    for (int which = 0; which < 2; which++) {
        T *x = (which ? (T *)m.v : (T *)m.k) + (t * c.Hkv + h) * c.hd;
        const S *d = (const S *)(which ? c.v_pages : c.k_pages) + r * c.row;
        float scale = 1.0f;
        if (sizeof(S) == 1 && place >= 0) scale = (which ? c.v_scale : c.k_scale)[r];
        for (int i = lane; i < c.hd; i += 32) x[i] = from_f<T>(place < 0 ? 0.0f : __fmul_rn(to_f(d[i]), scale));
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

int launch_gqa_cache_write(const GqaCacheArgs &c, int dtype, const int32_t *cu, long long total, const int32_t *start,
                           const void *k, const void *v, long long k_ts, long long k_hs, long long v_ts, long long v_hs,
                           cudaStream_t st, std::string *msg) {
    GqaMove m{c, cu, start, (void *)k, (void *)v, k_ts, k_hs, v_ts, v_hs, total, 1};
    const long long blocks = (total * c.Hkv + 3) / 4;
    if (blocks > 0x7fffffffLL) {
        *msg = "too many cache rows";
        return WB_EINVAL;
    }
    ProfScope ps("gqa_write", st);
    if (blocks > 0)
        by_types(dtype, c.store, [&](auto t, auto s) {
            gqa_write_kernel<decltype(t), decltype(s)><<<(unsigned)blocks, 128, 0, st>>>(m);
        });
    gqa_len_kernel<<<(c.n_seq + 127) / 128, 128, 0, st>>>(m);
    return WB_OK;
}

int launch_gqa_cache_read(const GqaCacheArgs &c, int dtype, const int32_t *cu, long long total, const int32_t *start,
                          void *k, void *v, cudaStream_t st, std::string *msg) {
    GqaMove m{c, cu, start, k, v, 0, 0, 0, 0, total, 0};
    const long long blocks = (total * c.Hkv + 3) / 4;
    if (blocks > 0x7fffffffLL) {
        *msg = "too many cache rows";
        return WB_EINVAL;
    }
    if (blocks == 0) return WB_OK;
    ProfScope ps("gqa_read", st);
    by_types(dtype, c.store, [&](auto t, auto s) {
        gqa_read_kernel<decltype(t), decltype(s)><<<(unsigned)blocks, 128, 0, st>>>(m);
    });
    return WB_OK;
}

}  // namespace wb
