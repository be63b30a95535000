"""Edges of the grouped-head attention and its cache: infinities in visible
values, values and scores at the ends of the range, index arrays that do not
fit their rows, scratch under memory pressure and under graph captures."""
from __future__ import annotations

import pytest

from tests import gqa_ref as ref

pytestmark = pytest.mark.gpu


def _ints(*values):
    import torch
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rows(seed, dtype, T, Hkv, hd):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    return tuple(torch.randn(T, Hkv, hd, generator=g, device="cuda").to(dtype) for _ in range(2))


def _cache(k, v, lens, store="native"):
    """Slots 0.. of one layer that hold the packed rows."""
    import wave_engine_b200 as wb
    c = wb.GqaCache(1, k.shape[1], k.shape[2], len(lens), max(lens), sum(-(-n // 128) for n in lens), dtype=k.dtype, store=store)
    for i, n in enumerate(lens):
        c.reserve(i, n)
    c.write(0, k, v, list(range(len(lens))), ref.starts(lens))
    return c


def _held(x, store):
    """What the cache's rows stand for, in 64 bits."""
    import torch
    if store == "native":
        return x.double()
    q, s = ref.quantise(x, {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}[store])
    return q.double() * s.double()[..., None]


def _check_decode(c, q, k, v, lens, store, scale):
    """The cache's decode against 64 bits."""
    import torch
    import wave_engine_b200 as wb
    out, lse = c.decode(0, q, return_lse=True, scale=scale)
    vv = _held(v, store)
    o, m, z = ref.attention(q, _held(k, store), vv, list(range(len(lens) + 1)), ref.starts(lens), True, scale)
    pair = store == "native" and q.dtype == torch.bfloat16
    ref.check(out, lse.T, o, m, z, 2.0 ** -16 if pair else 2.0 ** -11, 0.0 if pair else ref.floor(max(lens), vv))
    assert wb.default_context(0).take_device_error() == 0
    return out, lse


@pytest.mark.parametrize("op", ["prompt", "decode"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("H,Hkv,hd", [(4, 2, 64), (24, 2, 128), (3, 1, 42)])
def test_visible_infinities_in_values(op, dtype, H, Hkv, hd):
    """An infinity or NaN among the values of visible keys reaches its column as in 64 bits (opposite infinities are
    NaN), whatever the weights round to, and no other column."""
    import torch
    import wave_engine_b200 as wb
    dtype = getattr(torch, dtype)
    lens = [300, 2000, 1, 40]
    cu = ref.starts(lens)
    k, v = _rows(1, dtype, cu[-1], Hkv, hd)
    q = _rows(2, dtype, len(lens), H, hd)[0] * 0.25
    bad = v.clone()
    for key, col, x in ((5, 0, "inf"), (17, 3, "-inf"), (130, 4, "nan"), (255, 9, "inf"), (299, 9, "-inf"), (299, 10, "inf"),
                        (300 + 64, 1, "inf"), (300 + 65, 2, "-inf"), (300 + 1999, 20, "inf"), (2300, 7, "-inf"),
                        (2301 + 39, 8, "inf"), (2301, 8, "inf")):
        bad[key, 0, col] = float(x)
    if op == "decode":
        clean, got = (_cache(k, x, lens).decode(0, q) for x in (v, bad))
    else:
        starts = _ints(*range(len(lens) + 1)), _ints(*cu)
        clean, got = (wb.gqa_attention(q, k, x, *starts) for x in (v, bad))
    want = ref.attention(q, k, bad, list(range(len(lens) + 1)), cu, True, hd ** -0.5)[0]
    hit = ~torch.isfinite(want)
    assert hit.sum() == 10 * (H // Hkv) and torch.equal(got[~hit], clean[~hit])
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[hit].double().nan_to_num(7.0), want[hit].nan_to_num(7.0))


@pytest.mark.parametrize("store", ["native", "int8"])
def test_starts_past_the_rows_are_flagged(store):
    """Starts on the device that end behind the rows at hand: flagged, no length changes for what was not written."""
    import torch
    import wave_engine_b200 as wb
    ctx = wb.Context(0)
    c = wb.GqaCache(1, 2, 64, 3, 256, 6, store=store, ctx=ctx)
    for i in range(3):
        c.reserve(i, 256)
    k, v = _rows(11, torch.bfloat16, 5, 2, 64)
    for slots, cu, start, lens in (((0,), (0, 8), None, [0, 0, 0]), ((0, 1, 2), (0, 3, 5, 9), None, [3, 2, 0]),
                                   ((0, 1, 2), (0, 5, 200, 300), (7, 0, 0), [12, 2, 0]), ((1,), (0, 9), (4,), [12, 2, 0]),
                                   ((2,), (0, -3), None, [12, 2, 0]), ((1, 2), (0, 5, 4), (0, 9), [12, 5, 0])):
        c.write(0, k, v, _ints(*slots), _ints(*cu), None if start is None else _ints(*start))
        assert ctx.take_device_error() & 0x8, cu
        assert c.lens[0].tolist() == lens, cu
    for cu, total in (((0, 8), 5), ((0, 5, 9), 5), ((0, 5, 4), 5)):
        c.read(0, _ints(*range(len(cu) - 1)), _ints(*cu), total)
        assert ctx.take_device_error() & 0x8, cu
    c.read(0, _ints(0, 1), _ints(0, 3, 5), 5)
    assert ctx.take_device_error() == 0
    ctx.close()


@pytest.mark.parametrize("store", ["int8", "e4m3"])
@pytest.mark.parametrize("upto", [64, 70, 300])
def test_decode_value_scales_of_zero(store, upto):
    """Pages that the caller filled: rows whose value scale is 0 are values of 0, at the start of every warp's keys too."""
    import torch
    lens = [300]
    k, v = _rows(5, torch.bfloat16, 300, 1, 64)
    q = _rows(6, torch.bfloat16, 1, 4, 64)[0]
    c = _cache(k, v, lens, store)
    for key in range(upto):
        c.v_scale[0, c.table[0, key // 128], 0, key % 128] = 0.0
    v = v.clone()
    v[:upto] = 0
    _check_decode(c, q, k, v, lens, store, 0.125)


@pytest.mark.parametrize("store", ["native", "int8", "e4m3"])
@pytest.mark.parametrize("H,hd", [(2, 64), (12, 128)])
def test_decode_values_at_the_end_of_the_range(store, H, hd):
    """bf16 values near the type's largest: the output is between them, also where the scores rise along the keys."""
    import torch
    lens = [600, 40, 1]
    cu = ref.starts(lens)
    k, v = _rows(3, torch.bfloat16, cu[-1], 1, hd)
    v = (v.sign() * 1.25 * 2.0 ** 127).to(torch.bfloat16)
    q = _rows(4, torch.bfloat16, 3, H, hd)[0]
    q[:, :, 0] = 3.0
    k[:, 0, 0] = torch.linspace(-12, 12, cu[-1], device="cuda").to(torch.bfloat16)
    _check_decode(_cache(k, v, lens, store), q, k, v, lens, store, 1.0)


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_values_at_the_end_of_the_range(hd):
    import torch
    import wave_engine_b200 as wb
    T = 700
    k, v = _rows(3, torch.bfloat16, T, 1, hd)
    v = (v.sign() * 1.25 * 2.0 ** 127).to(torch.bfloat16)
    q = _rows(4, torch.bfloat16, T, 2, hd)[0]
    q[:, :, 0] = 3.0
    k[:, 0, 0] = torch.linspace(-6, 6, T, device="cuda").to(torch.bfloat16)
    out, lse = wb.gqa_attention(q, k, v, [0, T], return_lse=True)
    ref.check(out, lse, *ref.attention(q, k, v, [0, T], [0, T], True, hd ** -0.5))


@pytest.mark.parametrize("store", ["native", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("H,Hkv,hd", [(8, 1, 64), (24, 2, 128), (2, 1, 64), (2, 2, 64), (3, 1, 42)])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_decode_queries_do_not_reach_each_other(store, dtype, H, Hkv, hd, bad):
    """A query that is not finite leaves every other head right, whose scores rise along the keys, and so do keys with
    infinities: products in no head's place are NaN there."""
    import torch
    dtype = getattr(torch, dtype)
    lens = [300, 5000, 1, 40]
    k, v = _rows(20, dtype, sum(lens), Hkv, hd)
    q = _rows(21, dtype, len(lens), H, hd)[0]
    k[:, :, 1] = torch.linspace(-4, 4, len(k), device="cuda")[:, None]  # scores that rise by 2^200 and more
    q[:, :, 1] = 200.0
    c = _cache(k, v, lens, store)
    clean, clean_lse = _check_decode(c, q, k, v, lens, store, hd ** -0.5)
    hit = torch.zeros(len(lens), H, dtype=torch.bool, device="cuda")
    q2 = q.clone()
    for i, h in ((0, 1), (1, H - 1), (2, 0), (3, 1)):
        q2[i, h, 0] = float(bad)
        hit[i, h] = True
    got, lse = c.decode(0, q2, return_lse=True)
    assert got[hit].isnan().all() or bad == "inf"
    got[hit], lse[hit] = clean[hit], clean_lse[hit]
    vv = _held(v, store)
    o, m, z = ref.attention(q, _held(k, store), vv, list(range(len(lens) + 1)), ref.starts(lens), True, hd ** -0.5)
    u_p, floor = (2.0 ** -16, 0.0) if store == "native" and dtype == torch.bfloat16 else (2.0 ** -11, ref.floor(max(lens), vv))
    ref.check(got, lse.T, o, m, z, u_p, floor)
    if store == "native":  # -infinity for the scores of the first half of the keys
        first = 0
        half = [n // 32 * 16 + 8 if n > 32 else 0 for n in lens]
        for n, x in zip(lens, half):
            k[first:first + x, :, 0] = -float("inf")
            first += n
        q[:, :, 0] = 1.0
        c = _cache(k, v, lens)
        out, lse = c.decode(0, q, return_lse=True)
        rest = [n - x for n, x in zip(lens, half)]
        keep = torch.isfinite(k[:, 0, 0])
        o, m, z = ref.attention(q, k[keep], v[keep], list(range(len(lens) + 1)), ref.starts(rest), True, hd ** -0.5)
        ref.check(out, lse.T, o, m, z, u_p, floor)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("H,Hkv,hd", [(2, 2, 64), (8, 1, 128), (3, 1, 42)])
def test_scores_of_minus_infinity(dtype, H, Hkv, hd):
    """A query whose visible scores are all -infinity has no weight anywhere: 0 and -inf from the prompt attention and
    from the decode; keys with such scores count for nothing beside others."""
    import torch
    import wave_engine_b200 as wb
    dtype = getattr(torch, dtype)
    n, T = 200, 420
    k, v = _rows(7, dtype, T, Hkv, hd)
    q = _rows(8, dtype, T, H, hd)[0]
    q[:, :, 0] = 1.0
    k[:, :, 0] = 0.0
    hidden = k.clone()
    hidden[:n, :, 0] = -float("inf")
    out, lse = wb.gqa_attention(q, hidden, v, [0, T], return_lse=True)
    assert not out[:n].any() and (lse[:, :n] == -float("inf")).all()
    o, m, z = ref.attention(q[n:], k[n:], v[n:], [0, T - n], [0, T - n], True, hd ** -0.5)
    ref.check(out[n:], lse[:, n:], o, m, z, floor=ref.floor(T, v, 5) if dtype == torch.float16 else 0.0)
    c = _cache(hidden, v, [T])
    for held in (1, n, T):
        c.lens[0, 0] = held
        out, lse = c.decode(0, q[-1:], return_lse=True)
        if held <= n:
            assert not out.any() and (lse == -float("inf")).all()
        else:
            ref.check(out, lse.T, o[-1:], m[-1:], (z[0][:, -1:], z[1][:, -1:]), 2.0 ** -11, ref.floor(T, v))


def _lowest(dtype, Hkv, hd, H, n, T, big):
    """Rows whose first n keys have, through dimension 0, the lowest scores that the type can make."""
    import torch
    k, v = _rows(9, dtype, T, Hkv, hd)
    q = _rows(10, dtype, T, H, hd)[0]
    q[:, :, 0] = big
    k[:, :, 0] = 0.0
    low = k.clone()
    low[:n, :, 0] = torch.finfo(dtype).min
    return q, k, low, v


# scores of 2^128 and 2^38 (bf16), 2^32 (fp16), 2^25 times the scale
LOWEST = [("bfloat16", 1.0), ("bfloat16", 2.0 ** -90), ("float16", 60000.0), ("bfloat16", 2.0 ** -103)]


@pytest.mark.parametrize("dtype,big", LOWEST)
@pytest.mark.parametrize("H,Hkv,hd", [(2, 2, 64), (8, 1, 128)])
def test_prompt_lowest_scores(dtype, big, H, Hkv, hd):
    """Keys whose scores are the lowest numbers there are (masked by a dimension of the type's lowest value) count for
    nothing beside others; queries that see nothing else still get a mean of values."""
    import torch
    import wave_engine_b200 as wb
    dtype = getattr(torch, dtype)
    n, T = 300, 700
    q, k, low, v = _lowest(dtype, Hkv, hd, H, n, T, big)
    out, lse = wb.gqa_attention(q, low, v, [0, T], return_lse=True)
    o, m, z = ref.attention(q[n:], k[n:], v[n:], [0, T - n], [0, T - n], True, hd ** -0.5)
    ref.check(out[n:], lse[:, n:], o, m, z, floor=ref.floor(T, v, 5) if dtype == torch.float16 else 0.0)
    assert torch.isfinite(out[:n]).all() and out[:n].abs().max() <= v.abs().max()
    want = ref.attention(q[:n], low[:n], v[:n], [0, n], [0, n], True, hd ** -0.5)[2][0]
    assert ((lse[:, :n].double() - want) / want).abs().max() < 1e-5
    # the highest scores: one key takes all, those before it nothing
    high = k.clone()
    high[n, :, 0] = torch.finfo(dtype).max
    out, lse = wb.gqa_attention(q, high, v, [0, T], return_lse=True)
    o = v[n].double().repeat_interleave(H // Hkv, 0).expand(T - n, H, hd)
    z = ref.attention(q[n:], high[n:n + 1], v[n:n + 1], [0, T - n], [0, 1], False, hd ** -0.5)[2]
    assert ((out[n:].double() - o).abs() <= 2.02 * ref.ROUNDOFF[dtype] * o.abs()).all()
    assert ((lse[:, n:].double() - z[0]) / z[0]).abs().max() < 1e-5
    assert torch.equal(out[:n], wb.gqa_attention(q, k, v, [0, T])[:n])


@pytest.mark.parametrize("store", ["native", "int8", "e4m3"])
@pytest.mark.parametrize("dtype,big", LOWEST)
@pytest.mark.parametrize("H,Hkv,hd", [(2, 2, 64), (24, 2, 128)])
def test_decode_lowest_scores(store, dtype, big, H, Hkv, hd):
    import torch
    if store != "native" and big < 1.0:
        return  # 8-bit keys: dimensions of a bf16 query far below its largest are 0
    dtype = getattr(torch, dtype)
    n, T = 300, 700
    q, k, low, v = _lowest(dtype, Hkv, hd, H, n, T, big)
    q = q[-1:]
    c = _cache(low, v, [T], store)
    out, lse = c.decode(0, q, return_lse=True)
    kk, vv = _held(k[n:], store), _held(v[n:], store)
    o, m, z = ref.attention(q, kk, vv, [0, 1], [0, T - n], True, hd ** -0.5)
    pair = store == "native" and dtype == torch.bfloat16
    ref.check(out, lse.T, o, m, z, 2.0 ** -16 if pair else 2.0 ** -11, 0.0 if pair else ref.floor(T, vv))
    for held in (1, 30, n):
        c.lens[0, 0] = held
        out, lse = c.decode(0, q, return_lse=True)
        assert torch.isfinite(out).all() and out.abs().max() <= 1.01 * v.abs().max()
        want = ref.attention(q, _held(low[:held], store), _held(v[:held], store), [0, 1], [0, held], True, hd ** -0.5)[2][0]
        assert ((lse.T.double() - want) / want).abs().max() < 1e-5
    if store == "native":
        c.lens[0, 0] = T
        high = k[n:n + 1].clone()
        high[:, :, 0] = torch.finfo(dtype).max
        c.write(0, high, v[n:n + 1], [0], [0, 1], [T - 1])
        o = v[n].double().repeat_interleave(H // Hkv, 0)[None]
        assert ((c.decode(0, q).double() - o).abs() <= 2.02 * ref.ROUNDOFF[dtype] * o.abs()).all()


@pytest.mark.parametrize("scale", [0.0, 1e-36, -1e-36])
def test_scales_near_zero(scale):
    """Scores of 1e32 and a scale that makes them nothing, or little: the mean of the values."""
    import torch
    import wave_engine_b200 as wb
    T, hd = 300, 64
    k, v = _rows(18, torch.bfloat16, T, 1, hd)
    q, _ = _rows(19, torch.bfloat16, T, 2, hd)
    out, lse = wb.gqa_attention(q * 1e16, k * 1e16, v, [0, T], scale=scale, return_lse=True)
    o, m, z = ref.attention(q, k, v, [0, T], [0, T], True, 0.0)
    ref.check(out, None, o, m, z)
    assert (lse.double() - z[0]).abs().max() < 1e-2


def test_first_call_inside_a_capture_on_the_own_stream():
    """Scratch that is made while the context's own stream is captured stays out of the graph."""
    import torch
    import wave_engine_b200 as wb
    from wave_engine_b200 import _lib
    ctx = wb.Context(0)
    q, _ = _rows(12, torch.bfloat16, 40, 4, 42)  # rows that are copied into scratch
    k, v = _rows(13, torch.bfloat16, 40, 2, 42)
    cu = _ints(0, 25, 40)
    want = wb.gqa_attention(q, k, v, cu)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    stream = torch.cuda.ExternalStream(_lib.lib().wb_context_own_stream(ctx.handle))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        wb.gqa_attention(q, k, v, cu, out=out, ctx=ctx)
    for _ in range(2):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    graph.reset()
    ctx.close()


def test_scratch_that_cannot_grow():
    """A call whose scratch does not fit is refused and costs nothing: the scratch there was serves the next call.  Growth
    that fits but not twice over is granted."""
    import torch
    import wave_engine_b200 as wb
    ctx = wb.Context(0)
    hd = 127  # rows that are copied into scratch: 256 bytes a key here, whatever the keys' own stride
    q, _ = _rows(14, torch.bfloat16, 3, 1, hd)
    one, _ = _rows(15, torch.bfloat16, 1, 1, hd)
    cu, ck = _ints(0, 3), _ints(0, 3)

    def call(rows):
        k = one.expand(rows, 1, hd)
        return wb.gqa_attention(q, k, one[0, 0].expand(rows, 1, hd), cu, ck, ctx=ctx)

    want = call(1000)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(3):
        with pytest.raises(wb.WaveB200Error):
            call(2 ** 31 - 1)  # two terabytes
        assert torch.equal(call(1000), want)
        torch.cuda.synchronize()
        assert torch.cuda.mem_get_info()[0] >= free - 2 ** 20
    part = free // 512  # keys whose copies (K and V) fill the memory
    assert torch.equal(call(int(0.35 * part)), want)
    assert torch.equal(call(int(0.42 * part)), want)
    ctx.close()


def _step(seed, lens, H=8, Hkv=2, hd=128, store="native"):
    """A decode and an append with queries and rows at fixed places, and what the decode gives."""
    import torch
    k, v = _rows(seed, torch.bfloat16, sum(lens), Hkv, hd)
    c = _cache(k, v, lens, store)
    q = _rows(seed + 1, torch.bfloat16, len(lens), H, hd)[0]
    odd = _rows(seed + 2, torch.bfloat16, 50, 2, 42)[0]  # rows that are copied into scratch
    out, prompt = torch.zeros_like(q), torch.zeros_like(odd)
    start, cu = _ints(*(n - 1 for n in lens)), _ints(0, 20, 50)
    last = torch.stack([k[n - 1] for n in ref.starts(lens)[1:]]), torch.stack([v[n - 1] for n in ref.starts(lens)[1:]])

    def step():
        import wave_engine_b200 as wb
        c.write(0, *last, None, None, start)
        c.decode(0, q, out=out)
        wb.gqa_attention(odd, odd, odd, cu, out=prompt)

    return step, out, prompt


def test_a_graph_outlives_its_thread():
    """The context of a thread that captured a graph ends with it; the graph keeps what its kernels use."""
    import gc
    import threading
    import torch
    import wave_engine_b200 as wb
    made = {}

    def capture():
        step, out, prompt = _step(30, [3000, 70, 1500])
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
            stream.synchronize()
            made["want"] = out.clone(), prompt.clone()
            made["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(made["graph"], stream=stream):
                step()
            stream.synchronize()
        made["out"], made["keep"] = (out, prompt), step

    thread = threading.Thread(target=capture)
    thread.start()
    thread.join()
    gc.collect()
    ctx = wb.Context(0)  # takes what memory the thread's context gave back
    junk = torch.full((64 << 20,), -1, dtype=torch.int32, device="cuda")
    q, _ = _rows(33, torch.bfloat16, 2000, 4, 42)
    wb.gqa_attention(q, q, q, [0, 2000], ctx=ctx)
    for _ in range(3):
        for x in made["out"]:
            x.zero_()
        made["graph"].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(made["out"], made["want"]))
    assert (junk == -1).all()
    ctx.close()


def test_graphs_of_one_stream_run_side_by_side():
    """Two graphs captured on one stream, replayed on two at the same time, beside calls."""
    import torch
    steps = [_step(40 + 10 * i, [5000 + 100 * i, 64, 900]) for i in range(3)]
    capture = torch.cuda.Stream()
    capture.wait_stream(torch.cuda.current_stream())
    graphs, want = [], []
    with torch.cuda.stream(capture):
        for step, out, prompt in steps:
            step()
            capture.synchronize()
            want.append((out.clone(), prompt.clone()))
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=capture):
                step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(50):
        for _, out, prompt in steps:
            out.zero_(), prompt.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for graph, stream in zip(graphs[:2], streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            with torch.cuda.stream(capture):
                steps[2][0]()
        torch.cuda.synchronize()
        for (_, out, prompt), (o, p) in zip(steps, want):
            assert torch.equal(out, o) and torch.equal(prompt, p)


def test_scratch_of_graphs_is_given_back():
    import time
    import torch
    import wave_engine_b200 as wb
    q, _ = _rows(50, torch.bfloat16, 1, 1, 127)
    rows = 4000000  # 2 GB of copies
    k, cu = q.expand(rows, 1, 127), _ints(0, 1)
    ctx = wb.Context(0)
    out = torch.empty_like(q)
    ck = _ints(0, 10)
    wb.gqa_attention(q, k[:10], k[:10], cu, ck, out=out, ctx=ctx)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        wb.gqa_attention(q, k, k, cu, ck, out=out, ctx=ctx)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, q) and torch.cuda.mem_get_info()[0] < free - 2 ** 30
    ctx.close()
    graph.replay()
    torch.cuda.synchronize()
    graph.reset()
    torch.cuda.empty_cache()
    for _ in range(100):
        wb.Context(0).close()  # frees what no graph holds any more
        if torch.cuda.mem_get_info()[0] >= free - 2 ** 28:
            break
        time.sleep(0.05)
    assert torch.cuda.mem_get_info()[0] >= free - 2 ** 28


@pytest.mark.parametrize("slots", [None, [0, 1, 2, 3], [2, 0, 3, 1]])
def test_starts_that_are_the_lengths(slots):
    """start = the cache's own lengths: all of them are read before one changes, in a graph too."""
    import torch
    import wave_engine_b200 as wb
    Hkv, hd, held, add = 4, 64, [100, 7, 300, 0], [200, 129, 1, 250]
    k, v = _rows(60, torch.bfloat16, sum(held), Hkv, hd)
    k2, v2 = _rows(61, torch.bfloat16, sum(add), Hkv, hd)
    at = [0, 1, 2, 3] if slots is None else slots
    cu = _ints(*ref.starts(add))
    c = wb.GqaCache(1, Hkv, hd, 4, 600, 20)
    for i in range(4):
        c.reserve(i, 600)
    index = None if slots is None else _ints(*slots)

    def call():
        c.write(0, k2, v2, index, cu, c.lens[0])

    def check():
        assert wb.default_context(0).take_device_error() == 0
        want = [0] * 4
        for i, s in enumerate(at):
            want[s] = held[i] + add[i]
        assert c.lens[0].tolist() == want
        gk, gv = c.read(0, index, cu, sum(add), _ints(*held))
        assert torch.equal(gk, k2) and torch.equal(gv, v2)

    for _ in range(20):
        c.write(0, k, v, [0, 1, 2, 3], ref.starts(held), [0, 0, 0, 0])
        call()
        check()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    c.write(0, k, v, [0, 1, 2, 3], ref.starts(held), [0, 0, 0, 0])
    graph.replay()
    check()


def test_gradients_are_not_lost_silently():
    """Forward only: tensors that want a gradient are refused where autograd records."""
    import torch
    import wave_engine_b200 as wb
    q, _ = _rows(16, torch.bfloat16, 5, 4, 64)
    k, v = _rows(17, torch.bfloat16, 5, 2, 64)
    c = _cache(k, v, [5])
    calls = [lambda q, k, v: wb.gqa_attention(q, k, v, [0, 5]), lambda q, k, v: c.write(0, k, v, [0], [0, 5], [0]),
             lambda q, k, v: c.decode(0, q[:1])]
    for i, call in enumerate(calls):
        for x in range(3):
            args = [t.clone().requires_grad_(y == x) for y, t in enumerate((q, k, v))]
            used = x == 0 if i == 2 else x > 0 if i == 1 else True
            if used:
                with pytest.raises(ValueError, match="gradient"):
                    call(*args)
            else:
                call(*args)
            with torch.no_grad():
                call(*args)
            with torch.inference_mode():
                call(*args)
    out = torch.zeros_like(q, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        wb.gqa_attention(q, k, v, [0, 5], out=out)
    with pytest.raises(ValueError, match="gradient"):
        c.decode(0, q[:1], out=out[:1])


def test_no_dimensions_are_refused():
    import torch
    import wave_engine_b200 as wb
    q, _ = _rows(62, torch.bfloat16, 3, 4, 64)
    k, v = _rows(63, torch.bfloat16, 3, 2, 64)
    c = _cache(k, v, [3])
    with pytest.raises(ValueError):
        wb.gqa_attention(q[:, :, :0], k[:, :, :0], v[:, :, :0], [0, 3])
    with pytest.raises(ValueError):
        c.decode(0, q[:1, :, :0])
    with pytest.raises(ValueError):
        c.write(0, k[:, :, :0], v[:, :, :0], [0], [0, 3], [0])
    with pytest.raises((ValueError, wb.WaveB200Error)):
        wb.gqa_attention(q[:, :0], k, v, [0, 3])


def test_decode_of_too_many_sequences_is_refused():
    import torch
    import wave_engine_b200 as wb
    n = 2 ** 24
    pages = torch.zeros(1, 1, 128, 16, dtype=torch.bfloat16, device="cuda")
    table, lens = (torch.zeros(*s, dtype=torch.int32, device="cuda") for s in ((n, 1), (n,)))
    q = torch.zeros(n, 1, 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(wb.WaveB200Error, match="sequences"):
        wb.gqa_decode(q, pages, pages, table, lens)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("H,Hkv,hd", [(2, 2, 64), (8, 1, 128), (3, 1, 42)])
def test_infinite_queries(dtype, H, Hkv, hd):
    """A query with an infinity: NaN where it sees a score of +infinity, 0 and -inf where all it sees is -infinity."""
    import torch
    import wave_engine_b200 as wb
    dtype = getattr(torch, dtype)
    n, T = 150, 400
    k, v = _rows(64, dtype, T, Hkv, hd)
    q = _rows(65, dtype, T, H, hd)[0]
    k[:, :, 0] = -1.0
    k[n, :, 0] = 1.0
    clean, clean_lse = wb.gqa_attention(q, k, v, [0, T], return_lse=True)
    hit = [0, 63, n - 1, n, n + 1, 256, T - 1]
    q[hit, H - 1, 0] = float("inf")
    out, lse = wb.gqa_attention(q, k, v, [0, T], return_lse=True)
    for t in hit:
        if t < n:
            assert not out[t, H - 1].any() and lse[H - 1, t] == -float("inf")
        else:
            assert out[t, H - 1].isnan().all() and lse[H - 1, t].isnan()
    other = torch.ones(T, H, dtype=torch.bool, device="cuda")
    other[hit, H - 1] = False
    assert torch.equal(out[other], clean[other]) and torch.equal(lse.T[other], clean_lse.T[other])
    c = _cache(k, v, [T])
    for held in (1, n, n + 1, T):
        c.lens[0, 0] = held
        out, lse = c.decode(0, q[-1:], return_lse=True)
        if held <= n:
            assert not out[0, H - 1].any() and lse[0, H - 1] == -float("inf")
        else:
            assert out[0, H - 1].isnan().all() and lse[0, H - 1].isnan()
        assert torch.isfinite(out[0, :H - 1]).all()


@pytest.mark.parametrize("sizes", [dict(prompts=(5,)), dict(prompts=(130, 7), chunk=0), dict(prompts=(3, 4), steps=0)])
def test_example_without_a_chunk(sizes):
    """examples/gqa_serve.py with one sequence, no continued chunk, no steps."""
    import torch
    from tests.test_gqa_example_gpu import _example
    got, whole, _ = _example().serve("native", **sizes)
    for u, w in zip(got, whole):
        assert u.shape == w.shape and (u.float() - w.float()).pow(2).mean(1).sqrt().max().item() <= 2 * 2.0 ** -6
    assert torch.cuda.current_stream() == torch.cuda.default_stream()
