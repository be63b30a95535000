// wb_gqa.h -- grouped-head dot-product attention in 16 bits: attention over
// packed prompts, a paged key-value cache of 16- or 8-bit values, and the
// attention of one new token over it.
#pragma once
#include "wave_b200.h"
#include "wb_internal.h"
#ifdef __CUDACC__
#include "wb_ptx.cuh"
#endif

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>
#include <string>

namespace wb {

static constexpr int GQA_MAX_HD = 128;
static constexpr int GQA_MAX_GROUP = 128;

// columns of a stored cache row: head_dim up to whole 16s, so that rows of
// either width are whole 16-byte pieces
__host__ __device__ inline int gqa_row(int hd) { return (hd + 15) & ~15; }

// Packed prompts (device pointers; strides in elements).
struct GqaAttnArgs {
    const void *q, *k, *v;
    void *out;
    float *lse;  // nullable, [H][total_q]
    long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;
    const int32_t *cu_q, *cu_k;
    long long total_q, total_k;
    int H, Hkv, hd, n_seq, causal;
    float scale;
    uint32_t *dev_err;
};

// One layer's paged cache and the sequences of a call (device pointers).
struct GqaCacheArgs {
    void *k_pages, *v_pages;
    float *k_scale, *v_scale;
    const int32_t *table;
    int32_t *lens;
    const int32_t *slots;  // [n_seq], nullptr = 0, 1, ..
    int store, Hkv, hd, row, n_pages, n_slots, max_pages, n_seq;
    uint32_t *dev_err;
};

// A stream's scratch begins with counters that every call finds and leaves
// zero.
static constexpr size_t GQA_WS_HEAD = 16384;
static constexpr int GQA_WS_TICKET = 4095;  // the cache write's counter (the decode's are the first, one per CTA)

// scratch bytes (after the counters and index arrays) of the calls below
size_t gqa_attention_scratch(const GqaAttnArgs &a, int dtype);
size_t gqa_decode_scratch(const GqaCacheArgs &c, int H, int sm_count);

int launch_gqa_attention(const GqaAttnArgs &a, int dtype, void *scratch, int sm_count, cudaStream_t st,
                         std::string *msg);
// cu: nullptr = one token per sequence; start: nullptr = the slots' lengths
int launch_gqa_cache_write(const GqaCacheArgs &c, int dtype, const int32_t *cu, long long total, const int32_t *start,
                           const void *k, const void *v, long long k_ts, long long k_hs, long long v_ts, long long v_hs,
                           unsigned int *ticket, cudaStream_t st, std::string *msg);
int launch_gqa_cache_read(const GqaCacheArgs &c, int dtype, const int32_t *cu, long long total, const int32_t *start,
                          void *k, void *v, cudaStream_t st, std::string *msg);
int launch_gqa_decode(const GqaCacheArgs &c, int dtype, int H, const void *q, long long q_ss, long long q_hs,
                      float scale, void *out, float *lse, unsigned int *counters, void *scratch, int sm_count,
                      cudaStream_t st, std::string *msg);

#ifdef __CUDACC__
// The cache's kernels and the decode may be brought up while the stream's
// previous kernel ends (a token written and read back 8.3 -> 7.0 us).  They
// call gqa_wait() before they read or write memory, and by that call let the
// next one be brought up in turn (by then everything before them has
// completed).  What earlier kernels may have written is read by plain loads:
// the read-only path wants memory that stays as it is while the kernel runs.
// The prompt attention is launched plainly: let in early, the next one cost it 2
// to 6 us of 70 (packed 768-wide batch).
template <typename... KArgs, typename... Args>
static void gqa_launch(void (*kernel)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t st, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, args...);  // an error stays for the caller's check
}
// A kernel's shared memory limit, once per device (`done`: a bit each).
template <typename K>
static cudaError_t gqa_smem_limit(K *kernel, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (e != cudaSuccess || (done.load(std::memory_order_relaxed) & bit)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}
__device__ __forceinline__ void gqa_wait() {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
}

// The last sequence b with cu[b] <= t (cu[0] = 0, n sequences).  Empty
// sequences share their start with the next one and are never found.
__device__ __forceinline__ int gqa_find_seq(const int32_t *cu, int n, long long t) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// a / b, by a 32-bit division where that does
__device__ __forceinline__ long long gqa_quotient(long long a, long long b) {
    return (unsigned long long)(a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}

__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
#endif

}  // namespace wb
