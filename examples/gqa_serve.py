"""A small grouped-head decoder served from a paged cache: prompts of every
length in one packed pass, a second chunk that continues some of them, then
one token of every sequence per step, replayed from a CUDA graph.

    python examples/gqa_serve.py [--store native|int8|e4m3] [--steps 16]

Random weights; the blocks are x + proj(attention(norm(x))), their linear
parts torch's.  At the end the same rows are computed once more without a
cache, one packed pass over the whole sequences, and the largest difference
is printed."""
import argparse
import os
import sys
import time

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import wave_engine_b200 as wb  # noqa: E402


class Decoder:
    def __init__(self, n_layers, n_head, n_kv_head, head_dim, dtype, seed=0):
        g = torch.Generator("cuda").manual_seed(seed)
        normal = lambda *s: (torch.randn(s, generator=g, device="cuda") * s[-1] ** -0.5).to(dtype)  # noqa: E731
        self.H, self.Hkv, self.hd, self.E = n_head, n_kv_head, head_dim, n_head * head_dim
        self.qkv = [normal((n_head + 2 * n_kv_head) * head_dim, self.E) for _ in range(n_layers)]
        self.proj = [normal(self.E, self.E) for _ in range(n_layers)]

    def forward(self, x, attend):
        """x [tokens][n_embd]; attend(layer, q, k, v) -> [tokens][n_head][head_dim].
        q, k and v are slices of the fused projection's rows."""
        for layer, (w, p) in enumerate(zip(self.qkv, self.proj)):
            rows = F.linear(F.layer_norm(x, (self.E,)), w).view(-1, self.H + 2 * self.Hkv, self.hd)
            q, k, v = rows.split([self.H, self.Hkv, self.Hkv], 1)
            x = x + F.linear(attend(layer, q, k, v).reshape(-1, self.E), p)
        return x


def _starts(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def serve(store="e4m3", prompts=(5, 300, 1, 129), chunk=70, steps=16, n_layers=2, n_head=12, n_kv_head=4, head_dim=64,
          dtype=torch.bfloat16, seed=0):
    """Returns (rows by sequence from the cache, the same without, ms per decode step)."""
    model = Decoder(n_layers, n_head, n_kv_head, head_dim, dtype, seed)
    n = len(prompts)
    more = [chunk if i % 2 else 0 for i in range(n)]  # every second sequence gets a chunk
    total = [p + m + steps for p, m in zip(prompts, more)]
    g = torch.Generator("cuda").manual_seed(seed + 1)
    x = [torch.randn(t, model.E, generator=g, device="cuda").to(dtype) for t in total]
    cache = wb.GqaCache(n_layers, n_kv_head, head_dim, max_seqs=n, max_ctx=max(total),
                        n_pages=sum(-(-t // 128) for t in total), dtype=dtype, store=store)
    for i, t in enumerate(total):
        cache.reserve(i, t)

    # the prompts: written to the cache, attended from the rows at hand
    cu = _starts(prompts)

    def prompt(layer, q, k, v):
        cache.write(layer, k, v, cu=cu)
        return wb.gqa_attention(q, k, v, cu)

    y = model.forward(torch.cat([a[:p] for a, p in zip(x, prompts)]), prompt)
    done = [[part] for part in y.split(list(prompts))]

    # a chunk that continues cached positions: written, and its queries see
    # what the cache holds
    slots = [i for i in range(n) if more[i]]
    cu_q = _starts([more[i] for i in slots])
    held = [prompts[i] + more[i] for i in slots]
    cu_k = _starts(held)

    def continued(layer, q, k, v):
        cache.write(layer, k, v, slots=slots, cu=cu_q)
        keys, values = cache.read(layer, slots=slots, cu=cu_k, total=sum(held))
        return wb.gqa_attention(q, keys, values, cu_q, cu_k)

    if slots:
        y = model.forward(torch.cat([x[i][prompts[i]:prompts[i] + more[i]] for i in slots]), continued)
        for i, part in zip(slots, y.split([more[i] for i in slots])):
            done[i].append(part)

    # one token each per step: the whole step is one CUDA graph (lengths and
    # the table stay on the device)
    def token(layer, q, k, v):
        cache.write(layer, k, v)
        return cache.decode(layer, q)

    row = torch.zeros(n, model.E, dtype=dtype, device="cuda")
    stream = torch.cuda.Stream()
    lens = cache.lens.clone()
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        model.forward(row, token)  # workspaces
        cache.lens.copy_(lens)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = model.forward(row, token)
        start = time.perf_counter()
        for s in range(steps):
            row.copy_(torch.stack([a[t - steps + s] for a, t in zip(x, total)]))
            graph.replay()
            for i in range(n):
                done[i].append(out[i:i + 1].clone())
        stream.synchronize()
        ms = (time.perf_counter() - start) * 1e3 / max(1, steps)
    torch.cuda.default_stream().wait_stream(stream)

    cu_all = _starts(total)
    whole = model.forward(torch.cat(x), lambda layer, q, k, v: wb.gqa_attention(q, k, v, cu_all))
    return [torch.cat(d) for d in done], list(whole.split(total)), ms


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--store", default="e4m3", choices=["native", "int8", "e4m3"])
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args()
    got, whole, ms = serve(a.store, steps=a.steps, n_layers=a.layers)
    worst = max((u.float() - w.float()).abs().max().item() for u, w in zip(got, whole))
    size = max(w.float().abs().max().item() for w in whole)
    print(f"{len(got)} sequences of {', '.join(str(len(u)) for u in got)} rows, cache {a.store}: "
          f"largest difference {worst:.4f} of {size:.2f}; {ms:.3f} ms per decode step")


if __name__ == "__main__":
    main()
