"""Plain 64-bit forms of the grouped-head attention and its cache, and the
tolerances of the tests that compare with them.

Tolerance of an attention output o = sum_j p_j v_j of dtype T with half unit
in the last place u (2^-9 for bf16, 2^-12 for fp16, relative): the output is
rounded once (u |o|, and half the smallest subnormal, 2^-25, for an fp16
output below its normal range) and each unnormalised probability is rounded once to T
(at most u p_j |v_j| each, so u A with A = sum_j p_j |v_j|).  Everything else
is fp32: a score's sum of hd products is off by at most hd 2^-24 sum|q k|
scale, about 1e-4 at hd 128 and inputs of unit size, which moves o by that
times A, as does the log sum exp itself."""
from __future__ import annotations

import torch

HALF_ULP = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}
FP32_REL = 1e-4  # scores, exponentials and sums in fp32
LSE_ABS = 1e-4
SUBNORMAL = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def attention(q, k, v, cu_q, cu_k, causal, scale):
    """(out, A, lse) in float64: A = attention over |v|."""
    H, Hkv = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full((H, q.shape[0]), -float("inf"), dtype=torch.float64, device=q.device)
    for b in range(len(cu_q) - 1):
        qs, ks = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        n, m = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if n == 0 or m == 0:
            continue
        see = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if causal:
            see = see.tril(m - n)
        for h in range(H):
            g = h // (H // Hkv)
            s = (q[qs, h].double() @ k[ks, g].double().T * scale).masked_fill(~see, -float("inf"))
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - torch.where(z == -float("inf"), 0.0, z)[:, None])
            vv = v[ks, g].double()
            out[qs, h], mag[qs, h], lse[h, qs] = p @ vv, p @ vv.abs(), z
    return out, mag, lse


def check(got, lse, ref, mag, ref_lse):
    u = HALF_ULP[got.dtype]
    bound = 1.01 * u * (ref.abs() + mag) + FP32_REL * mag + SUBNORMAL[got.dtype] + 1e-30
    err = (got.double() - ref).abs()
    worst = (err - bound).max().item()
    assert worst <= 0, f"worst excess {worst}, at a bound of {bound.flatten()[(err - bound).argmax()].item()}"
    if lse is not None:
        empty = ref_lse == -float("inf")
        assert torch.equal(lse == -float("inf"), empty)
        off = (lse.double() - ref_lse)[~empty].abs().max().item() if (~empty).any() else 0.0
        assert off <= LSE_ABS, f"lse off by {off}"
    assert not got[(mag == 0) & (ref == 0)].any()


def quantise(x, store):
    """(stored, scale) of rows x [...][hd], as the cache's definition: fp32, 1 / top the nearest float."""
    top = 127.0 if store == torch.int8 else 448.0
    scale = (x.float().abs().amax(-1) * (1.0 / top)).clamp(min=2.0 ** -126)
    y = x.float() / scale[..., None]
    return (y.round() if store == torch.int8 else y).to(store), scale


def values(stored, scale, dtype):
    """What quantised rows read back as."""
    return (stored.float() * scale[..., None]).to(dtype)


def starts(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu
