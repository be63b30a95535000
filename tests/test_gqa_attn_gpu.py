"""Attention over packed prompts (wb_gqa_attention) against its definition in
64 bits: types, head layouts, lengths from one token, odd sizes, strides,
rows without keys, values that must not leak, refusals."""
from __future__ import annotations

import pytest

from tests import gqa_ref as ref

pytestmark = pytest.mark.gpu


def _inputs(seed, dtype, H, Hkv, hd, Tq, Tk):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    mk = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return mk(Tq, H, hd), mk(Tk, Hkv, hd), mk(Tk, Hkv, hd)


def _check(out, lse, want, v):
    import torch
    ref.check(out, lse, *want, floor=ref.floor(v.shape[0], v, 5) if out.dtype == torch.float16 else 0.0)


def _run(dtype, H, Hkv, hd, lens, past=None, causal=True, scale=None, host=False, seed=0):
    import torch
    import wave_engine_b200 as wb
    dtype = getattr(torch, dtype)
    keys = [n + (past[i] if past else 0) for i, n in enumerate(lens)]
    cq, ck = ref.starts(lens), ref.starts(keys)
    q, k, v = _inputs(seed, dtype, H, Hkv, hd, cq[-1], ck[-1])
    ix = (lambda c: c) if host else (lambda c: torch.tensor(c, dtype=torch.int32, device="cuda"))
    out, lse = wb.gqa_attention(q, k, v, ix(cq), None if past is None else ix(ck), causal=causal, scale=scale,
                                return_lse=True)
    o, m, z = ref.attention(q, k, v, cq, ck, causal, hd ** -0.5 if scale is None else scale)
    _check(out, lse, (o, m, z), v)
    assert wb.default_context(0).take_device_error() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("H,Hkv,hd", [(4, 2, 42), (8, 8, 48), (12, 4, 64), (12, 2, 64), (4, 1, 80), (10, 2, 104),
                                      (32, 8, 128), (7, 1, 128), (3, 3, 1), (5, 5, 8), (128, 1, 32), (33, 3, 24)])
def test_heads(dtype, H, Hkv, hd):
    _run(dtype, H, Hkv, hd, [150, 1, 0, 37, 260])


@pytest.mark.parametrize("lens", [[1], [2], [127], [128], [129], [255], [256], [257], [1023], [1500], [0, 0, 5, 0],
                                  [1] * 70, [31, 33, 64, 65, 16, 15, 300, 2]])
@pytest.mark.parametrize("H,Hkv,hd", [(2, 2, 64), (8, 1, 128)])
def test_lengths(lens, H, Hkv, hd):
    _run("bfloat16", H, Hkv, hd, lens, seed=len(lens))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hkv,hd", [(4, 4, 128), (6, 2, 64)])
def test_continued(causal, H, Hkv, hd):
    """Key counts above and below the query counts; rows that see no key."""
    _run("float16", H, Hkv, hd, [5, 130, 1, 200, 64, 3, 300], [700, 129, 1000, -150, -64, -3, 0], causal=causal)


def test_non_causal():
    _run("bfloat16", 4, 2, 128, [300, 1, 129], causal=False)


def test_many_keys():
    _run("bfloat16", 2, 1, 128, [3], [9000])


def test_host_starts_and_scale():
    _run("float16", 4, 2, 64, [50, 0, 200], causal=True, scale=0.3, host=True)
    _run("float16", 4, 2, 64, [50, 0, 200], [3, 5, 7], causal=True, scale=-0.2, host=True)
    _run("bfloat16", 2, 2, 32, [200], scale=0.0)


def test_large_scores():
    """Scores of hundreds: the running maximum rises over the tiles, one key takes all."""
    _run("bfloat16", 2, 2, 128, [700], scale=8.0)
    _run("float16", 2, 2, 64, [700], scale=6.0)


@pytest.mark.parametrize("rising", [True, False])
def test_drifting_scores(rising):
    """Scores that rise (or fall) steadily with the key's position."""
    import torch
    import wave_engine_b200 as wb
    T, H, hd = 1200, 2, 64
    q, k, v = _inputs(3, torch.float16, H, H, hd, T, T)
    q[:, :, 0] = 4.0
    ramp = torch.linspace(-40, 40, T, device="cuda").to(torch.float16)
    k[:, :, 0] = (ramp if rising else -ramp)[:, None]
    cu = [0, T]
    out, lse = wb.gqa_attention(q, k, v, cu, return_lse=True, scale=1.0)
    _check(out, lse, ref.attention(q, k, v, cu, cu, True, 1.0), v)


@pytest.mark.parametrize("hd", [64, 128, 42])
@pytest.mark.parametrize("layout", ["heads_first", "fused", "odd_offset", "broadcast", "odd_stride"])
def test_strides(layout, hd):
    import torch
    import wave_engine_b200 as wb
    H, Hkv, T = 6, 2, 333
    q, k, v = _inputs(5, torch.bfloat16, H, Hkv, hd, T, T)
    if layout == "heads_first":
        q, k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    elif layout == "fused":
        rows = torch.cat([q, k, v], 1)
        q, k, v = rows[:, :H], rows[:, H:H + Hkv], rows[:, H + Hkv:]
    elif layout == "odd_offset":
        def shift(x):
            buf = torch.full((x.numel() + 1,), float("nan"), dtype=x.dtype, device="cuda")
            buf[1:] = x.reshape(-1)
            return buf[1:].view(x.shape)
        q, k, v = shift(q), shift(k), shift(v)
    elif layout == "broadcast":
        k, v = k[:, :1].expand(T, Hkv, hd), v[:, :1].expand(T, Hkv, hd)
    else:
        def widen(x):
            buf = torch.full((x.shape[0], x.shape[1], hd + 3), float("nan"), dtype=x.dtype, device="cuda")
            buf[:, :, :hd] = x
            return buf[:, :, :hd]
        q, k, v = widen(q), widen(k), widen(v)
    cu = torch.tensor([0, 100, T], dtype=torch.int32, device="cuda")
    buf = torch.full((H, T, hd), 7.0, dtype=q.dtype, device="cuda")
    out, lse = wb.gqa_attention(q, k, v, cu, return_lse=True, out=buf.transpose(0, 1))
    _check(out, lse, ref.attention(q, k, v, [0, 100, T], [0, 100, T], True, hd ** -0.5), v)
    out2 = wb.gqa_attention(q, k, v, cu)
    assert torch.equal(out2, out)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("H,Hkv,hd", [(2, 2, 64), (8, 1, 128), (4, 2, 42)])
def test_unseen_values_do_not_leak(bad, H, Hkv, hd):
    """Infinities and NaN in keys and values of other sequences and of later
    positions; queries that do see such a value are not finite in that column."""
    import torch
    import wave_engine_b200 as wb
    lens = [70, 1, 300]
    cu = ref.starts(lens)
    T = cu[-1]
    q, k, v = _inputs(11, torch.bfloat16, H, Hkv, hd, T, T)
    clean = wb.gqa_attention(q, k, v, cu)
    v2, k2 = v.clone(), k.clone()
    v2[69, 0, 3 % hd] = bad      # last position of the first sequence
    v2[70, 0, 5 % hd] = bad      # the second sequence (one position)
    v2[71 + 200, 0, 7 % hd] = bad
    k2[71 + 250, 0, 0] = float("nan")
    got = wb.gqa_attention(q, k2, v2, cu)
    rows = torch.arange(T, device="cuda")
    hit = torch.zeros(T, H, hd, dtype=torch.bool, device="cuda")
    G = H // Hkv
    hit[69, :G, 3 % hd] = True
    hit[70, :G, 5 % hd] = True
    hit[(rows >= 271), :G, 7 % hd] = True
    hit[(rows >= 321), :G, :] = True
    assert torch.equal(got[~hit], clean[~hit])
    assert not torch.isfinite(got[hit]).any()
    # non-causal: only the own sequence's values
    got = wb.gqa_attention(q, k, v2, cu, causal=False)
    clean = wb.gqa_attention(q, k, v, cu, causal=False)
    own = torch.zeros(T, H, hd, dtype=torch.bool, device="cuda")
    own[:70, :G, 3 % hd] = True
    own[70, :G, 5 % hd] = True
    own[71:, :G, 7 % hd] = True
    assert torch.equal(got[~own], clean[~own]) and not torch.isfinite(got[own]).any()


@pytest.mark.parametrize("n", [63, 64, 65, 200])
def test_many_sequences(n):
    """Both orders in which items are dealt out: sequences of no tokens up to several items."""
    _run("bfloat16", 6, 2, 64, [(i * 37) % 211 if i % 5 else 0 for i in range(n)], seed=n)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("H,Hkv,hd", [(6, 2, 64), (8, 1, 128), (6, 2, 42)])
def test_queries_do_not_reach_each_other(bad, H, Hkv, hd):
    """A query that is not finite makes its own head NaN; rows of the same
    tile (the next sequence's among them) stay as they are."""
    import torch
    import wave_engine_b200 as wb
    cu = ref.starts([70, 1, 300])
    q, k, v = _inputs(12, torch.bfloat16, H, Hkv, hd, cu[-1], cu[-1])
    clean, clean_lse = wb.gqa_attention(q, k, v, cu, return_lse=True)
    q2 = q.clone()
    hit = torch.zeros(cu[-1], H, dtype=torch.bool, device="cuda")
    for t, h in ((70, 1), (71, 0), (71 + 41, H - 1), (370, 2)):
        q2[t, h, 0] = bad
        hit[t, h] = True
    got, lse = wb.gqa_attention(q2, k, v, cu, return_lse=True)
    assert torch.equal(got[~hit], clean[~hit]) and torch.equal(lse.T[~hit], clean_lse.T[~hit])
    if bad != bad:
        assert got[hit].isnan().all() and lse.T[hit].isnan().all()


def test_same_bits_and_streams():
    import torch
    import wave_engine_b200 as wb
    q, k, v = _inputs(2, torch.bfloat16, 8, 2, 128, 700, 700)
    cu = torch.tensor([0, 300, 700], dtype=torch.int32, device="cuda")
    a = wb.gqa_attention(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = wb.gqa_attention(q, k, v, cu)
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    c = torch.empty_like(a)
    with torch.cuda.graph(graph):
        wb.gqa_attention(q, k, v, cu, out=c)
    q2 = torch.randn_like(q)
    want = wb.gqa_attention(q2, k, v, cu)
    q.copy_(q2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, want)


def test_bad_device_starts_are_flagged():
    """Starts outside the buffers, on the device: flagged, nothing outside is touched."""
    import torch
    import wave_engine_b200 as wb
    q, k, v = _inputs(1, torch.bfloat16, 2, 2, 64, 200, 200)
    ctx = wb.Context(0)
    for cu, ck in ([[0, 100, 300], None], [[0, 100, 200], [0, 400, 500]], [[0, 100, 200], [0, 150, 100]],
                   [[-5, 100, 200], None]):
        i = lambda c: None if c is None else torch.tensor(c, dtype=torch.int32, device="cuda")  # noqa: E731
        wb.gqa_attention(q, k, v, i(cu), i(ck), ctx=ctx)
        assert ctx.take_device_error() & 0x8
    ctx.close()


def test_refusals():
    import torch
    import wave_engine_b200 as wb
    q, k, v = _inputs(1, torch.bfloat16, 4, 2, 64, 10, 10)
    bad = [
        lambda: wb.gqa_attention(q, k, v, [0, 5, 9]),                       # last start is not the rows' number
        lambda: wb.gqa_attention(q, k, v, [0, 6, 5, 10]),                   # descends
        lambda: wb.gqa_attention(q, k, v, [1, 10]),
        lambda: wb.gqa_attention(q, k, v, [0, 10], [0, 5, 10]),             # another number of sequences
        lambda: wb.gqa_attention(q[:, :3], k, v, [0, 10]),                  # heads not a multiple
        lambda: wb.gqa_attention(q, k.half(), v, [0, 10]),                  # mixed types
        lambda: wb.gqa_attention(q.float(), k.float(), v.float(), [0, 10]),
        lambda: wb.gqa_attention(q.cpu(), k, v, [0, 10]),
        lambda: wb.gqa_attention(q, k[:, :, :32], v[:, :, :32], [0, 10]),
        lambda: wb.gqa_attention(q, k, v[:9], [0, 10]),
        lambda: wb.gqa_attention(q[0], k, v, [0, 10]),
        lambda: wb.gqa_attention(q, k, v, [0, 10], scale=float("nan")),
        lambda: wb.gqa_attention(q, k, v, torch.tensor([0, 10], device="cuda")),  # int64
        lambda: wb.gqa_attention(q, k[:9], v[:9], [0, 10]),                 # cu_k needed
        lambda: wb.gqa_attention(q, k, v, [0, 10], out=torch.empty(10, 4, 64, device="cuda")),
        lambda: wb.gqa_attention(q.repeat(1, 1, 3), k.repeat(1, 1, 3), v.repeat(1, 1, 3), [0, 10]),  # head_dim 192
        lambda: wb.gqa_attention(q.repeat(1, 65, 1), k[:, :1], v[:, :1], [0, 10]),  # 260 heads on one
    ]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, wb.WaveB200Error)):
            f()
            print("case", i, "was taken")
    assert wb.gqa_attention(q[:0], k[:0], v[:0], [0]).shape == (0, 4, 64)
