// wb_gqa_decode.cu -- attention of one new token per sequence over the paged
// key-value cache: for the sequence's query head h over cached positions
// j < len,  out = sum_j softmax_j(scale q . k_j) v_j,  lse = log sum_j
// exp(scale q . k_j); a sequence without positions gives 0 and -inf.
#include "wb_gqa.h"

namespace wb {

struct GqaDecodeArgs {
    GqaCacheArgs c;
    const void *q;
    void *out;
    float *lse;
    long long q_ss, q_hs;
    int H;
    float scale;
};

// One warp per (sequence, query head), one position at a time.
template <class T, class S>
__global__ void __launch_bounds__(128) gqa_decode_simple_kernel(GqaDecodeArgs a) {
    const GqaCacheArgs &c = a.c;
    const long long wid = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (wid >= (long long)c.n_seq * a.H) return;
    const int b = (int)(wid / a.H), h = (int)(wid - (long long)b * a.H), hk = h / (a.H / c.Hkv);
    const int slot = c.slots ? c.slots[b] : b;
    const T *qp = (const T *)a.q + b * a.q_ss + h * a.q_hs;
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < 4; i++) q[i] = lane + 32 * i < c.hd ? to_f(qp[lane + 32 * i]) : 0.0f;
    float m = -INFINITY, l = 0.0f, le = 0.0f;  // l's rounding so far in le
    bool bad = slot < 0 || slot >= c.n_slots;
    const int len = bad ? 0 : c.lens[slot];
    if (len < 0 || len > c.max_pages * WB_PAGE) bad = true;
    for (int j = 0; !bad && j < len; j++) {
        const int pg = c.table[(long long)slot * c.max_pages + (j >> WB_PAGE_SHIFT)];
        if (pg < 0 || pg >= c.n_pages) {
            bad = true;
            break;
        }
        const long long r = ((long long)pg * c.Hkv + hk) * WB_PAGE + (j & (WB_PAGE - 1));
        const S *kp = (const S *)c.k_pages + r * c.row, *vp = (const S *)c.v_pages + r * c.row;
        float s = 0.0f, vs = 1.0f;
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < c.hd) s = fmaf(q[i], to_f(kp[lane + 32 * i]), s);
        s = warp_sum(s) * a.scale;
        if (sizeof(S) == 1) {
            s *= c.k_scale[r];
            vs = c.v_scale[r];
        }
        const float mn = fmaxf(m, s);
        const float f = m == mn ? 1.0f : expf(m - mn), p = s == mn ? 1.0f : expf(s - mn);
        const float y = p - le * f, ln = l * f + y;
        le = (ln - l * f) - y;
        l = ln;
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < c.hd) o[i] = o[i] * f + p * (vs * to_f(vp[lane + 32 * i]));
        m = mn;
    }
    if (bad && lane == 0) atomicOr(c.dev_err, WB_DERR_BOUNDS);
    T *op = (T *)a.out + ((long long)b * a.H + h) * c.hd;
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    for (int i = 0; i < 4; i++)
        if (lane + 32 * i < c.hd) op[lane + 32 * i] = from_f<T>(o[i] * inv);
    if (a.lse && lane == 0) a.lse[(long long)b * a.H + h] = m + logf(l);
}

size_t gqa_decode_scratch(const GqaCacheArgs &, int, int) { return 0; }

int launch_gqa_decode(const GqaCacheArgs &c, int dtype, int H, const void *q, long long q_ss, long long q_hs,
                      float scale, void *out, float *lse, unsigned int *, void *, int, cudaStream_t st,
                      std::string *msg) {
    GqaDecodeArgs a{c, q, out, lse, q_ss, q_hs, H, scale};
    const long long blocks = ((long long)c.n_seq * H + 3) / 4;
    if (blocks > 0x7fffffffLL) {
        *msg = "too many query rows";
        return WB_EINVAL;
    }
    ProfScope ps("gqa_decode", st);
    const unsigned g = (unsigned)blocks;
    if (dtype == WB_BF16) {
        if (c.store == WB_INT8) gqa_decode_simple_kernel<__nv_bfloat16, int8_t><<<g, 128, 0, st>>>(a);
        else if (c.store == WB_E4M3) gqa_decode_simple_kernel<__nv_bfloat16, __nv_fp8_e4m3><<<g, 128, 0, st>>>(a);
        else gqa_decode_simple_kernel<__nv_bfloat16, __nv_bfloat16><<<g, 128, 0, st>>>(a);
    } else {
        if (c.store == WB_INT8) gqa_decode_simple_kernel<__half, int8_t><<<g, 128, 0, st>>>(a);
        else if (c.store == WB_E4M3) gqa_decode_simple_kernel<__half, __nv_fp8_e4m3><<<g, 128, 0, st>>>(a);
        else gqa_decode_simple_kernel<__half, __half><<<g, 128, 0, st>>>(a);
    }
    return WB_OK;
}

}  // namespace wb
