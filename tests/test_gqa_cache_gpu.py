"""The paged key-value cache of the grouped-head attention: writing (16 bit,
int8, e4m3), reading back, one-token attention over it."""
from __future__ import annotations

import pytest

from tests import gqa_ref as ref

pytestmark = pytest.mark.gpu

STORES = ["native", "int8", "e4m3"]


def _kinds():
    import torch
    return {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _rows(seed, dtype, T, Hkv, hd):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    k = torch.randn(T, Hkv, hd, generator=g, device="cuda")
    k[..., 1::7] *= 5.0
    v = torch.randn(T, Hkv, hd, generator=g, device="cuda") * torch.rand(T, Hkv, 1, generator=g, device="cuda")
    return k.to(dtype), v.to(dtype)


def _stored(x, store):
    """What x reads back as."""
    return x if store == "native" else ref.values(*ref.quantise(x, _kinds()[store]), x.dtype)


def _same(a, b):
    import torch
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("Hkv,hd", [(2, 42), (3, 64), (1, 128), (4, 48), (2, 1), (1, 104)])
def test_write_read(store, dtype, Hkv, hd):
    """Packed prompts, appended rows, single tokens; pages out of order; other slots untouched."""
    import torch
    import wave_engine_b200 as wb
    dtype = getattr(torch, dtype)
    cache = wb.GqaCache(2, Hkv, hd, max_seqs=5, max_ctx=600, n_pages=16, dtype=dtype, store=store)
    for n in (100, 200, 300, 400):
        for seq in (4, 1, 2):
            cache.reserve(seq, n)
    lens = [130, 0, 257]
    slots = [4, 1, 2]
    cu = ref.starts(lens)
    k, v = _rows(1, dtype, cu[-1], Hkv, hd)
    cache.write(1, k, v, slots, cu)
    assert cache.lens[1].tolist() == [0, 0, 257, 0, 130] and not cache.lens[0].any()
    k2, v2 = _rows(2, dtype, 3, Hkv, hd)
    dev = torch.tensor(slots, dtype=torch.int32, device="cuda")
    cache.write(1, k2, v2, dev)  # one token each, appended
    assert cache.lens[1].tolist() == [0, 1, 258, 0, 131]
    # all of it back, and a window
    gk, gv = cache.read(1, slots, [0, 131, 132, 390])
    want = [torch.cat([x[0:130], y[0:1], y[1:2], x[130:387], y[2:3]]) for x, y in ((k, k2), (v, v2))]
    assert _same(gk, _stored(want[0], store)) and _same(gv, _stored(want[1], store))
    gk, gv = cache.read(1, dev, torch.tensor([0, 2, 2, 132], dtype=torch.int32, device="cuda"), 132,
                        torch.tensor([127, 0, 100], dtype=torch.int32, device="cuda"))
    for g, w in ((gk, want[0]), (gv, want[1])):
        assert _same(g, _stored(torch.cat([w[127:129], w[132 + 100:132 + 230]]), store))
    # rewriting from an earlier position shortens the slot
    cache.write(1, k[:5], v[:5], [2], [0, 5], [60])
    assert cache.lens[1, 2] == 65
    assert wb.default_context(0).take_device_error() == 0
    pad = cache.k_pages.view(torch.uint8) if store != "native" else cache.k_pages
    assert not pad[..., hd:].any()


@pytest.mark.parametrize("store", ["int8", "e4m3"])
def test_quantised_edges(store):
    """Zeros, the smallest subnormals, the largest values, infinities and NaN."""
    import torch
    import wave_engine_b200 as wb
    hd = 64
    for dtype in (torch.bfloat16, torch.float16):
        k, _ = _rows(3, dtype, 8, 1, hd)
        top = torch.finfo(dtype).max
        k[0] = 0
        k[1] = 0
        k[1, 0, 5] = torch.finfo(dtype).smallest_normal / 4
        k[2] = torch.finfo(dtype).tiny
        k[3, 0, 0], k[3, 0, 1] = top, -top
        k[4, 0, 9] = float("inf")
        k[5, 0, 0] = float("nan")
        k[6, 0, 63], k[6, 0, 62] = -float("inf"), float("nan")
        cache = wb.GqaCache(1, 1, hd, 1, 128, 1, dtype=dtype, store=store)
        cache.reserve(0, 8)
        cache.write(0, k, k.flip(2), [0], [0, 8])
        gk, gv = cache.read(0, [0], [0, 8])
        want = _stored(k[[0, 1, 2, 3, 7]], store)
        assert torch.equal(gk[[0, 1, 2, 3, 7]], want) and torch.equal(gv[[0, 1, 2, 3, 7]], want.flip(2))
        assert gk[4:7].isnan().all() and gv[4:7].isnan().all()


@pytest.mark.parametrize("store", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_quantised_ties(store, dtype):
    """Bit for bit the division's rounding, on many rows of every size, quotients midway between two stored values among them."""
    import torch
    import wave_engine_b200 as wb
    dtype = getattr(torch, dtype)
    n, Hkv, hd = 4096, 4, 128
    k, v = _rows(21, dtype, n, Hkv, hd)
    size = torch.exp2(torch.randint(-20, 12, (n, Hkv, 1), device="cuda").float())
    k, v = (k.float() * size).to(dtype), (v.float() / size).to(dtype)
    if dtype == torch.bfloat16:
        k[:64] *= 2.0 ** -110   # scales below the range of the remainder
        v[:64] *= 2.0 ** 100
    for kind, top in ((torch.int8, 127), (torch.float8_e4m3fn, 448)):
        q, s = ref.quantise(k, kind)
        if kind == _kinds()[store]:
            y = (k.float() / s[..., None]).abs()
            ties = (y - y.floor() == 0.5) if store == "int8" else ((y.view(torch.int32) & 0xFFFFF) == 0x80000)
            assert ties.sum() > 100
    cache = wb.GqaCache(1, Hkv, hd, 1, n, n // 128, dtype=dtype, store=store)
    cache.reserve(0, n)
    cache.write(0, k, v, [0], [0, n])
    gk, gv = cache.read(0, [0], [0, n])
    assert _same(gk, _stored(k, store)) and _same(gv, _stored(v, store))
    table = cache.table[0, :n // 128].long()
    held = cache.k_pages[0].view(torch.uint8)[table].view(_kinds()[store]).float().permute(0, 2, 1, 3).reshape(n, Hkv, hd)
    q, s = ref.quantise(k, _kinds()[store])
    finite = torch.isfinite(s)
    assert torch.equal(held[finite], q.float()[finite]) and finite.float().mean() > 0.9
    assert torch.equal(cache.k_scale[0][table].permute(0, 2, 1).reshape(n, Hkv), s)


def test_outside_the_pages():
    import torch
    import wave_engine_b200 as wb
    ctx = wb.Context(0)
    cache = wb.GqaCache(1, 2, 64, 2, 256, 3, ctx=ctx)
    cache.reserve(0, 128)
    k, v = _rows(0, torch.bfloat16, 200, 2, 64)
    with pytest.raises(wb.WaveB200Error):
        cache.write(0, k, v, [0], [0, 200], [100])       # past the table
    with pytest.raises(wb.WaveB200Error):
        cache.write(0, k[:2], v[:2], [1, 1])             # the same slot twice
    with pytest.raises(wb.WaveB200Error):
        cache.write(0, k[:1], v[:1], [2])
    i = lambda *c: torch.tensor(c, dtype=torch.int32, device="cuda")  # noqa: E731
    cache.write(0, k, v, i(0), i(0, 200))                # page 1 is not mapped
    assert ctx.take_device_error() & 0x8
    assert cache.lens[0, 0] == 0
    gk, _ = cache.read(0, i(0), i(0, 128), 128)
    assert torch.equal(gk, k[:128])                      # what has a page is written
    for args in ((i(5), i(0, 3)), (i(-1), i(0, 3))):
        cache.write(0, k[:3], v[:3], *args)
        assert ctx.take_device_error() & 0x8
    cache.write(0, k[:3], v[:3], i(0), i(0, 3), i(-7))
    assert ctx.take_device_error() & 0x8
    cache.write(0, k[:3], v[:3], i(0), i(0, 3), i(2 ** 31 - 2))
    assert ctx.take_device_error() & 0x8
    gk, _ = cache.read(0, i(0), i(0, 4), 4, i(126))
    assert ctx.take_device_error() & 0x8
    assert torch.equal(gk[:2], k[126:128]) and not gk[2:].any()
    ctx.close()


def test_pool():
    import torch
    import wave_engine_b200 as wb
    cache = wb.GqaCache(1, 1, 32, 3, 512, 5)
    cache.reserve(0, 300)
    cache.reserve(0, 200)
    assert cache.free_pages() == 2
    with pytest.raises(RuntimeError):
        cache.reserve(1, 400)
    with pytest.raises(ValueError):
        cache.reserve(1, 513)
    cache.release(0)
    assert cache.free_pages() == 5 and (cache.table == -1).all() and not cache.lens.any()
    with pytest.raises(ValueError):
        wb.GqaCache(1, 1, 129, 1, 1, 1)
    with pytest.raises(ValueError):
        wb.GqaCache(1, 1, 64, 1, 1, 1, dtype=torch.float32)


# ---- one-token attention -------------------------------------------------------------------------

def _filled(store, dtype, Hkv, hd, lens, seed=0, junk=True):
    """A cache whose slots 0.. hold lens positions, pages dealt out in turns, and their 64-bit values."""
    import torch
    import wave_engine_b200 as wb
    pages = sum(-(-n // 128) for n in lens) + 1
    cache = wb.GqaCache(1, Hkv, hd, max(1, len(lens)), max(max(lens), 1), pages, dtype=dtype, store=store)
    if junk:  # what lies past a length is not read: NaN everywhere first
        for p in (cache.k_pages, cache.v_pages):
            if store == "native":
                p.fill_(float("nan"))
            else:
                p.view(torch.uint8).fill_(0x7F)
        if store != "native":
            cache.k_scale.fill_(float("nan"))
            cache.v_scale.fill_(float("nan"))
    at = 1
    while at <= max(lens) + 127:
        for i, n in enumerate(lens):
            cache.reserve(i, min(n, at))
        at += 128
    cu = ref.starts(lens)
    k, v = _rows(seed, dtype, cu[-1], Hkv, hd)
    cache.write(0, k, v, list(range(len(lens))), cu)
    if store == "native":
        return cache, k.double(), v.double(), cu
    kk, vv = (a.double() * s.double()[..., None] for a, s in
              ((x[0].float(), x[1]) for x in (ref.quantise(t, _kinds()[store]) for t in (k, v))))
    return cache, kk, vv, cu


def _decode(store, dtype, H, Hkv, hd, lens, seed=0, scale=None):
    import torch
    import wave_engine_b200 as wb
    dtype = getattr(torch, dtype)
    cache, k, v, cu = _filled(store, dtype, Hkv, hd, lens, seed)
    q = torch.randn(len(lens), H, hd, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)
    out, lse = cache.decode(0, q, return_lse=True, scale=scale)
    o, m, z = ref.attention(q, k, v, list(range(len(lens) + 1)), cu, True, hd ** -0.5 if scale is None else scale)
    pair = store == "native" and dtype == torch.bfloat16
    ref.check(out, lse.T, o, m, z, 2.0 ** -16 if pair else 2.0 ** -11, 0.0 if pair else ref.floor(max(lens), v))
    again = cache.decode(0, q, scale=scale)
    assert torch.equal(again, out)
    assert wb.default_context(0).take_device_error() == 0
    return cache, q, out


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("H,Hkv,hd", [(4, 2, 42), (8, 8, 48), (12, 4, 64), (4, 1, 80), (10, 2, 104), (32, 8, 128),
                                      (17, 1, 128), (40, 1, 64), (3, 3, 1), (128, 2, 128), (2, 2, 16)])
def test_decode_heads(store, dtype, H, Hkv, hd):
    _decode(store, dtype, H, Hkv, hd, [300, 1, 129, 0, 64])


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("lens", [[0], [1], [15], [16], [17], [63], [64], [65], [127], [128], [129], [5000], [20001],
                                  [0, 0, 0], [3000, 1, 0, 700, 128, 2000], [9] * 200, list(range(1, 400, 7))])
def test_decode_lengths(store, lens):
    _decode(store, "bfloat16", 8, 2, 128, lens, seed=len(lens))
    _decode(store, "float16", 3, 1, 64, lens, seed=len(lens))


def test_decode_large_scores():
    for store in STORES:
        _decode(store, "bfloat16", 4, 1, 128, [3000, 50], scale=3.0)
        _decode(store, "float16", 4, 2, 64, [3000, 50], scale=-2.0)


@pytest.mark.parametrize("store", ["int8", "e4m3"])
def test_decode_value_sizes(store):
    """Values of very different sizes: a heavy key with tiny values beside light keys with large ones, and rows of zeros."""
    import torch
    import wave_engine_b200 as wb
    hd, n = 64, 600
    k, v = _rows(9, torch.bfloat16, n, 1, hd)
    k *= 0.05
    k[0] = 3.0
    v[0] *= 1e-6
    v[5:40] = 0
    v[300] *= 1e4
    q = torch.full((1, 2, hd), 1.0, device="cuda", dtype=torch.bfloat16)
    q[0, 1] = -1.0
    cache = wb.GqaCache(1, 1, hd, 1, n, 5, store=store)
    cache.reserve(0, n)
    cache.write(0, k, v, [0], [0, n])
    out, lse = cache.decode(0, q, return_lse=True, scale=1.0)
    kk, vv = (x[0].double() * x[1].double()[..., None] for x in (ref.quantise(t, _kinds()[store]) for t in (k, v)))
    o, m, z = ref.attention(q, kk, vv, [0, 1], [0, n], True, 1.0)
    ref.check(out, lse.T, o, m, z, 2.0 ** -11, ref.floor(n, vv))


def test_decode_slots_strides_and_bounds():
    import torch
    import wave_engine_b200 as wb
    cache, q, out = _decode("native", "bfloat16", 8, 2, 64, [300, 5, 129, 0])
    rows = torch.randn(3, 20, 64, device="cuda").to(torch.bfloat16)
    mine = rows[:, 3:11]
    mine.copy_(q[[2, 0, 1]])
    got = cache.decode(0, mine, slots=[2, 0, 1])
    assert torch.equal(got, out[[2, 0, 1]])
    got = cache.decode(0, mine, slots=torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(got, out[[2, 0, 1]])
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(cache.decode(0, odd), out)
    with pytest.raises(wb.WaveB200Error):
        cache.decode(0, q, slots=[0, 1, 2, 4])
    with pytest.raises(wb.WaveB200Error):
        cache.decode(0, q, slots=[0, 1, 2, 2])
    with pytest.raises(wb.WaveB200Error):
        cache.decode(0, q[:, :7])
    with pytest.raises(ValueError):
        cache.decode(0, q[:, :, :32])
    with pytest.raises(ValueError):
        cache.decode(0, q.float())
    # lengths and pages that do not fit, on the device
    ctx = wb.default_context(0)
    for n in (513, -1, 2 ** 31 - 1):
        cache.lens[0, 1] = n
        got = cache.decode(0, q)
        assert ctx.take_device_error() & 0x8
        assert torch.equal(got[[0, 2, 3]], out[[0, 2, 3]]) and torch.isfinite(got).all()
    cache.lens[0, 1] = 5
    cache.table[2, 1] = 10 ** 6
    got = cache.decode(0, q)
    assert ctx.take_device_error() & 0x8
    assert torch.equal(got[[0, 1, 3]], out[[0, 1, 3]])
    cache.lens[0, 2] = 128  # the last position was on the unmapped page
    assert torch.allclose(got[2].float(), cache.decode(0, q)[2].float(), atol=2e-2)
    got = cache.decode(0, q, slots=torch.tensor([0, 77, 2, -1], dtype=torch.int32, device="cuda"))
    assert ctx.take_device_error() & 0x8
    assert torch.equal(got[0], out[0]) and not got[[1, 3]].any()


@pytest.mark.parametrize("store", STORES)
def test_decode_sees_infinities(store):
    """A NaN in a visible key or value reaches its head; other heads and sequences stay as they were."""
    import torch
    import wave_engine_b200 as wb
    cache, q, out = _decode(store, "bfloat16", 4, 2, 64, [300, 260])
    k, v = _rows(0, torch.bfloat16, 1, 2, 64)
    k[0, 1, 3] = float("nan")
    cache.write(0, k, v, [0], [0, 1], [200])
    cache.lens[0, 0] = 300
    got = cache.decode(0, q)
    assert got[0, 2:].isnan().all() and torch.equal(got[1], out[1]) and torch.isfinite(got[0, :2]).all()
    assert wb.default_context(0).take_device_error() == 0


def test_decode_graph_and_step():
    """Write, then attend, captured once and replayed as the sequences grow; against the prompt attention."""
    import torch
    import wave_engine_b200 as wb
    H, Hkv, hd, T = 8, 2, 64, 150
    q = torch.randn(2 * T, H, hd, device="cuda").to(torch.bfloat16)
    k, v = _rows(4, torch.bfloat16, 2 * T, Hkv, hd)
    full = wb.gqa_attention(q, k, v, [0, T, 2 * T])
    cache = wb.GqaCache(1, Hkv, hd, 2, T, 4)
    for i in range(2):
        cache.reserve(i, T)
    at = lambda x, t: x.view(2, T, *x.shape[1:])[:, t]  # noqa: E731
    n = 120
    cache.write(0, torch.cat([k[:n], k[T:T + n]]), torch.cat([v[:n], v[T:T + n]]), [0, 1], [0, n, 2 * n])
    qs, ks, vs = (torch.zeros_like(at(x, 0)) for x in (q, k, v))
    out = torch.zeros_like(qs)
    slots = torch.tensor([0, 1], dtype=torch.int32, device="cuda")

    def step():
        cache.write(0, ks, vs, slots)
        cache.decode(0, qs, slots, out=out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t in range(n, T):
        qs.copy_(at(q, t)), ks.copy_(at(k, t)), vs.copy_(at(v, t))
        graph.replay()
        # both are the same sums rounded once to bf16 at the end, with
        # probabilities rounded to bf16 before the sum: see gqa_ref
        a, b = out.double(), at(full, t).double()
        assert ((a - b).abs() <= 2 ** -7 * (1 + b.abs())).all()
    assert cache.lens[0].tolist() == [T, T]


@pytest.mark.parametrize("n", [256, 257, 700])
@pytest.mark.parametrize("store", STORES)
def test_many_sequences(n, store):
    """More sequences than a block holds the lengths of, a third of them empty."""
    _decode(store, "bfloat16", 4, 2, 64, [(i * 37) % 150 if i % 3 else 0 for i in range(n)])


def test_host_index_arrays_are_refused_during_a_capture():
    """A graph would read them after they are gone; the capture itself goes on."""
    import torch
    import wave_engine_b200 as wb
    T, Hkv, hd = 5, 2, 64
    k, v = _rows(3, torch.bfloat16, T, Hkv, hd)
    q = torch.randn(T, 4, hd, device="cuda").to(torch.bfloat16)
    cu = torch.tensor([0, 2, T], dtype=torch.int32, device="cuda")
    cache = wb.GqaCache(1, Hkv, hd, 2, 128, 2)
    cache.reserve(0, 8)
    cache.reserve(1, 8)
    calls = [lambda c: wb.gqa_attention(q, k, v, c), lambda c: cache.write(0, k, v, cu=c),
             lambda c: cache.read(0, cu=c, total=T)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for call in calls:
            call(cu)
        want = wb.gqa_attention(q, k, v, cu)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = wb.gqa_attention(q, k, v, cu)
            for call in calls:
                with pytest.raises(wb.WaveB200Error, match="captured"):
                    call([0, 2, T])
            with pytest.raises(wb.WaveB200Error, match="captured"):
                cache.decode(0, q[:2], slots=[1, 0])
        graph.replay()
        stream.synchronize()
    assert torch.equal(out, want)
