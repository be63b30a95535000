// wb_gqa.cu -- grouped-head dot-product attention over packed prompts.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij) / sum_j exp(s_ij),
//   s_ij = scale q_i . k_j  over the keys j <= i + (n_k - n_q) of the
//   query's own sequence (all of them when not causal);
//   lse_i = log sum_j exp(s_ij); a query without keys gives 0 and -inf.
#include "wb_gqa.h"

namespace wb {

// One warp per (query token, head): a running maximum m, sum l and weighted
// values, one key at a time; the lanes hold 4 interleaved dims each.
template <class T>
__global__ void __launch_bounds__(128) gqa_attn_simple_kernel(GqaAttnArgs a) {
    const long long wid = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (wid >= a.total_q * a.H) return;
    const long long t = wid / a.H;
    const int h = (int)(wid - t * a.H), hk = h / (a.H / a.Hkv);
    const int b = gqa_find_seq(a.cu_q, a.n_seq, t);
    const long long q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
    if (q0 < 0 || t < q0 || t >= q1 || q1 > a.total_q || k0 < 0 || k1 < k0 || k1 > a.total_k) {
        if (lane == 0) atomicOr(a.dev_err, WB_DERR_BOUNDS);
        return;
    }
    const long long nk = k1 - k0;
    long long vis = a.causal ? (t - q0) + nk - (q1 - q0) + 1 : nk;
    vis = vis < nk ? vis : nk;
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
    const T *qp = (const T *)a.q + t * a.q_ts + (long long)h * a.q_hs;
    for (int i = 0; i < 4; i++) q[i] = lane + 32 * i < a.hd ? to_f(qp[lane + 32 * i]) : 0.0f;
    float m = -INFINITY, l = 0.0f, le = 0.0f;  // l's rounding so far in le
    for (long long j = 0; j < vis; j++) {
        const T *kp = (const T *)a.k + (k0 + j) * a.k_ts + (long long)hk * a.k_hs;
        const T *vp = (const T *)a.v + (k0 + j) * a.v_ts + (long long)hk * a.v_hs;
        float s = 0.0f;
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < a.hd) s = fmaf(q[i], to_f(kp[lane + 32 * i]), s);
        s = warp_sum(s) * a.scale;
        const float mn = fmaxf(m, s);
        const float c = m == mn ? 1.0f : expf(m - mn), p = s == mn ? 1.0f : expf(s - mn);
        const float y = p - le * c, ln = l * c + y;
        le = (ln - l * c) - y;
        l = ln;
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < a.hd) o[i] = o[i] * c + p * to_f(vp[lane + 32 * i]);
        m = mn;
    }
    T *op = (T *)a.out + t * a.o_ts + (long long)h * a.o_hs;
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    for (int i = 0; i < 4; i++)
        if (lane + 32 * i < a.hd) op[lane + 32 * i] = from_f<T>(o[i] * inv);
    if (a.lse && lane == 0) a.lse[(long long)h * a.total_q + t] = m + logf(l);
}

size_t gqa_attention_scratch(const GqaAttnArgs &, int) { return 0; }

int launch_gqa_attention(const GqaAttnArgs &a, int dtype, void *, int, cudaStream_t st, std::string *msg) {
    const long long blocks = (a.total_q * a.H + 3) / 4;
    if (blocks > 0x7fffffffLL) {
        *msg = "too many query rows";
        return WB_EINVAL;
    }
    ProfScope ps("gqa_attn", st);
    if (dtype == WB_BF16) gqa_attn_simple_kernel<__nv_bfloat16><<<(unsigned)blocks, 128, 0, st>>>(a);
    else gqa_attn_simple_kernel<__half><<<(unsigned)blocks, 128, 0, st>>>(a);
    return WB_OK;
}

}  // namespace wb
