"""Attention over a window, from training to serving, on one GPU: ``python -m
spcomm3d_amd.attention_example``.

1. Fits keys, values and queries of a few packed sequences to targets by gradient descent, one
   :meth:`Context.attend` and one :meth:`Context.attend_grad` a step.
2. Takes a prompt into a paged 8-bit cache (:meth:`Cache.append`, which rotates it by position),
   then one token a step: an append and a :meth:`Cache.attend`, recorded once and replayed.  The
   device's own lengths and page table say where a step stands, so nothing is recorded again.
3. Compares each served token with attention over the whole sequence in 16 bits.

All numbers are synthetic, drawn from a seed.
"""
from __future__ import annotations

import numpy as np

from . import device


def _heads(ctx, x, heads, dim, keep, dtype="f32"):
    """A panel of the rows of ``x`` and its heads."""
    p = ctx.panel(x.shape[0], x.shape[1], dtype)
    p.upload(device.to_bf16(x) if dtype == "bf16" else np.ascontiguousarray(x, dtype=np.float32))
    keep.append(p)
    return p.heads(heads, dim)


def fit(ctx, steps=60, rows=(90, 41, 130), heads=4, kv_heads=2, dim=32, window=48, sinks=2, rate=0.4, seed=0):
    """Losses of ``steps`` steps of gradient descent on |o - target|^2 / 2 per element."""
    rng = np.random.default_rng(seed)
    n, keep = sum(rows), []
    x = {name: rng.normal(size=(n, count * dim)).astype(np.float32)
         for name, count in (("q", heads), ("k", kv_heads), ("v", kv_heads))}
    target = 0.3 * rng.normal(size=(n, heads * dim)).astype(np.float32)
    h = {name: _heads(ctx, x[name], heads if name == "q" else kv_heads, dim, keep) for name in x}
    g = {name: _heads(ctx, np.zeros_like(x[name]), heads if name == "q" else kv_heads, dim, keep) for name in x}
    o, d_o = (_heads(ctx, np.zeros_like(target), heads, dim, keep) for _ in range(2))
    lse = ctx.vals(n * heads, np.float32)
    band = ctx.band(rows, window=window, sinks=sinks)
    losses = []
    for _ in range(steps):
        ctx.attend(band, h["q"], h["k"], h["v"], o, lse=lse)
        off = o.panel.download() - target
        losses.append(float(np.mean(off * off)) / 2)
        d_o.panel.upload(off)
        ctx.attend_grad(band, h["q"], h["k"], h["v"], o, lse, d_o, g["q"], g["k"], g["v"])
        for name in x:
            x[name] -= rate * g[name].panel.download()
            h[name].panel.upload(x[name])
    for handle in (*keep, lse, band):
        handle.close()
    return losses


def rotations(positions, turned):
    """Cosines, then sines, of every position's angles."""
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(turned // 2) / (turned // 2))
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


def serve(ctx, prompt=100, tokens=40, heads=8, kv_heads=2, dim=64, page=32, window=64, sinks=4, seed=1):
    """Largest difference of any served element from attention over the whole sequence with 16-bit
    keys and values, over the root mean square of the outputs."""
    rng = np.random.default_rng(seed)
    n, keep = prompt + tokens, []
    q, k, v = (rng.normal(size=(n, c * dim)).astype(np.float32) for c in (heads, kv_heads, kv_heads))
    pages = -(-n // page)
    table = rng.permutation(pages).astype(np.uint32)
    cache = ctx.cache("f8", pages, page, kv_heads, dim)
    turn = ctx.panel_from(rotations(n, dim))

    def words(values):  # 32-bit words on the device
        w = ctx.vals(max(len(values), 4), np.float32)
        w.upload(np.resize(np.asarray(values, dtype=np.uint32), w.n).view(np.float32))
        keep.append(w)
        return w

    table_dev, lens = words(table), words([prompt])
    keep.append(turn)
    # the prompt, one chunk
    first = device.CacheSeqs(1, table_dev.device_ptr(), pages, lens.device_ptr(), words([0, prompt]).device_ptr(),
                             rows=prompt, max_rows=prompt, max_len=n)
    parts = [_heads(ctx, x[:prompt], c, dim, keep, "bf16") for x, c in ((k, kv_heads), (v, kv_heads), (q, heads))]
    turned = _heads(ctx, np.zeros_like(q[:prompt]), heads, dim, keep, "bf16")
    cache.append(first, parts[0], parts[1], rotations=turn, q=parts[2], q_out=turned)
    # then token by token, recorded
    one = device.CacheSeqs(1, table_dev.device_ptr(), pages, lens.device_ptr(), words([0, 1]).device_ptr(), rows=1,
                           max_rows=1, max_len=n)
    k1, v1, q1 = (_heads(ctx, x[:1], c, dim, keep, "bf16") for x, c in ((k, kv_heads), (v, kv_heads), (q, heads)))
    turned1, o1 = (_heads(ctx, np.zeros_like(q[:1]), heads, dim, keep, "bf16") for _ in range(2))

    def step():
        cache.append(one, k1, v1, rotations=turn, q=q1, q_out=turned1)
        cache.attend(one, turned1, o1, window=window, sinks=sinks)

    lens.upload(np.full(4, prompt + 1, np.uint32).view(np.float32))
    step()  # makes the workspace that a recording may not
    ctx.capture_begin()
    step()
    graph = ctx.capture_end()
    served = []
    for t in range(prompt, n):
        lens.upload(np.full(4, t + 1, np.uint32).view(np.float32))
        for h, x in ((k1, k), (v1, v), (q1, q)):
            h.panel.upload(device.to_bf16(x[t:t + 1]))
        graph.launch()
        served.append(device.from_bf16(o1.panel.download())[0])
    graph.close()
    # the whole sequence at once, rotated by an append to a 16-bit cache of the same rows
    whole = ctx.cache("bf16", pages, page, kv_heads, dim)
    lens.upload(np.full(4, n, np.uint32).view(np.float32))
    every = device.CacheSeqs(1, table_dev.device_ptr(), pages, lens.device_ptr(), words([0, n]).device_ptr(), rows=n,
                             max_rows=n, max_len=n)
    kn, vn, qn = (_heads(ctx, x, c, dim, keep, "bf16") for x, c in ((k, kv_heads), (v, kv_heads), (q, heads)))
    turned_n, o_n = (_heads(ctx, np.zeros_like(q), heads, dim, keep, "bf16") for _ in range(2))
    whole.append(every, kn, vn, rotations=turn, q=qn, q_out=turned_n)
    whole.attend(every, turned_n, o_n, window=window, sinks=sinks)
    want = device.from_bf16(o_n.panel.download())[prompt:]
    for handle in (*keep, cache, whole):
        handle.close()
    return float(np.abs(np.array(served) - want).max() / np.sqrt(np.mean(want ** 2)))


def main():
    with device.Context(0) as ctx:
        losses = fit(ctx)
        print(f"fit: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {len(losses)} steps")
        print(f"serve: 8-bit cache token by token, largest difference from 16 bits at once "
              f"{100 * serve(ctx):.1f} % of the outputs' size")


if __name__ == "__main__":
    main()
