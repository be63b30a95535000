"""Plain 64-bit forms of the grouped-head attention and its cache, and the
tolerances of the tests that compare with them.

Tolerance of an attention output o = sum_j p_j v_j of dtype T with unit
roundoff u (2^-8 for bf16's 8 significant bits, 2^-11 for fp16's 11): the
output is rounded once (u |o|, and half the smallest subnormal, 2^-25, for an
fp16 output below its normal range) and each unnormalised probability is
rounded once to the type of its product with v, whose unit roundoff is u_p
(at most u_p p_j |v_j| each, so u_p A with A = sum_j p_j |v_j|): T in the
prompt attention; in the one-token attention fp16, or the sum of two bf16
numbers with bf16 values.  An fp16 probability, kept as 2^8 times its ratio
to the largest (2^5 in the prompt attention), is below its normal range off by
up to 2^-25 2^-8 of the largest: ``floor``, 2^-33 (2^-30) n max|v| over the n
keys.  Everything else is fp32: a score's sum of hd
products is off by at most hd 2^-24 sum|q k| scale -- about 1e-4 at hd 128 and
inputs of unit size, and computed where that is more -- which moves o by that
times A, and the log sum exp by as much."""
from __future__ import annotations

import torch

FP32_REL = 1e-4  # scores, exponentials and sums in fp32, at inputs of unit size
ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SUBNORMAL = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def attention(q, k, v, cu_q, cu_k, causal, scale):
    """(out, A, (lse, off)) in float64: A = attention over |v|, off = what fp32 scores may be off by."""
    H, Hkv = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full((H, q.shape[0]), -float("inf"), dtype=torch.float64, device=q.device)
    off = torch.full((H, q.shape[0]), FP32_REL, dtype=torch.float64, device=q.device)
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
            most = (q[qs, h].double().abs() @ k[ks, g].double().abs().T).masked_fill(~see, 0.0).amax(1)
            off[h, qs] = (q.shape[2] * 2.0 ** -24 * abs(scale) * most).clamp(min=FP32_REL)
            p = torch.exp(s - torch.where(z == -float("inf"), 0.0, z)[:, None])
            vv = v[ks, g].double()
            out[qs, h], mag[qs, h], lse[h, qs] = p @ vv, p @ vv.abs(), z
    return out, mag, (lse, off)


def floor(n, v, shift=8):
    """What fp16 probabilities below their normal range may move an output of n keys by."""
    return 2.0 ** (-25 - shift) * n * v.abs().max().item() if n and v.numel() else 0.0


def check(got, lse, ref, mag, ref_lse, u_p=None, floor=0.0):
    """u_p None: probabilities rounded to the output's type."""
    u = ROUNDOFF[got.dtype]
    u_p = u if u_p is None else u_p
    ref_lse, off = ref_lse
    score = off.T[:, :, None]
    bound = 1.01 * (u * ref.abs() + u_p * mag) + score * mag + SUBNORMAL[got.dtype] + floor + 1e-30
    err = (got.double() - ref).abs()
    worst = (err - bound).max().item()
    assert worst <= 0, f"worst excess {worst}, at a bound of {bound.flatten()[(err - bound).argmax()].item()}"
    if lse is not None:
        empty = ref_lse == -float("inf")
        assert torch.equal(lse == -float("inf"), empty)
        past = ((lse.double() - ref_lse).abs() - off)[~empty]
        assert past.numel() == 0 or past.max().item() <= 0, f"lse off by {past.max().item()} over {off.max().item()}"
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
