"""The cases on which the attention operators' speed is followed.

A case is one pass of one operator, as a user's program calls it:

``attend``  attention of packed sequences over the band of the last ``window`` keys (0: all of
            them) and the first ``sinks`` ones: what a prefill computes
``train``   the same and its gradients: what a training step computes
``append``  new keys and values go to a paged cache, the position rotation applied to them and to
            the queries on the way
``read``    attention of the newest tokens of every sequence over that cache, held in 16 bits or
            in 8 with a scale for each page and head

With ``own`` false, ``run`` computes them in their plain form: elementary torch operations in
32 bits, rounded once at the end.
"""
import math

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
          "f8": torch.float8_e4m3fn}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2, "f8": 1}
MOST_SCORES = 9e9  # scores that the plain form of a drawn case holds at once, at most
MOST_CACHE = 1.0e9  # cached numbers of a drawn case, at most
F8_MOST = 448.0


def listed():
    return [
        # the smallest calls: one short prompt, launches and host time are all there is
        {"name": "attend_short_bf16_d64", "kind": "attend", "dtype": "bf16", "seqs": 1, "shortest": 48,
         "longest": 48, "prefix": 0, "heads": 4, "kv_heads": 4, "dim": 64, "window": 0, "sinks": 0},
        # a batch of prompts of odd lengths behind a common prefix, shared heads, a window
        {"name": "attend_ragged_f16_w512", "kind": "attend", "dtype": "f16", "seqs": 9, "shortest": 37,
         "longest": 2501, "prefix": 200, "heads": 16, "kv_heads": 4, "dim": 128, "window": 512,
         "sinks": 4},
        # one long document
        {"name": "attend_16k_bf16_w4096", "kind": "attend", "dtype": "bf16", "seqs": 1,
         "shortest": 16384, "longest": 16384, "prefix": 0, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 4096, "sinks": 4},
        # training in single precision, small
        {"name": "train_small_f32_w128", "kind": "train", "dtype": "f32", "seqs": 2, "shortest": 411,
         "longest": 600, "prefix": 0, "heads": 4, "kv_heads": 2, "dim": 64, "window": 128, "sinks": 2},
        # packed documents without a window, a head size that is no power of two
        {"name": "train_packed_bf16_d96", "kind": "train", "dtype": "bf16", "seqs": 5, "shortest": 301,
         "longest": 2700, "prefix": 0, "heads": 12, "kv_heads": 4, "dim": 96, "window": 0, "sinks": 0},
        # a training step over a long context
        {"name": "train_8k_bf16_w1024", "kind": "train", "dtype": "bf16", "seqs": 1, "shortest": 8192,
         "longest": 8192, "prefix": 0, "heads": 32, "kv_heads": 8, "dim": 128, "window": 1024,
         "sinks": 4},
        # a token of every sequence of a serving batch goes to an 8-bit cache
        {"name": "append_64_f8", "kind": "append", "dtype": "bf16", "cache": "f8", "page": 64,
         "seqs": 64, "shortest": 200, "longest": 4000, "new": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "turned": 128},
        # prompts in chunks go to a 16-bit cache, half of each head is rotated
        {"name": "append_chunks_bf16", "kind": "append", "dtype": "bf16", "cache": "bf16", "page": 32,
         "seqs": 8, "shortest": 1800, "longest": 5000, "new": 1777, "heads": 32, "kv_heads": 8,
         "dim": 128, "turned": 64},
        # the smallest read: one sequence, one token
        {"name": "read_one_bf16_d64", "kind": "read", "dtype": "bf16", "cache": "bf16", "page": 16,
         "seqs": 1, "shortest": 700, "longest": 700, "new": 1, "heads": 8, "kv_heads": 2, "dim": 64,
         "window": 0, "sinks": 0},
        # a serving batch over an 8-bit cache
        {"name": "read_64_f8", "kind": "read", "dtype": "bf16", "cache": "f8", "page": 64, "seqs": 64,
         "shortest": 200, "longest": 4000, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0, "sinks": 0},
        # few long sequences over an 8-bit cache
        {"name": "read_100k_f8", "kind": "read", "dtype": "bf16", "cache": "f8", "page": 64, "seqs": 4,
         "shortest": 90001, "longest": 110000, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0, "sinks": 0},
        # drafted tokens of long conversations, of which a window and the first tokens stay visible
        {"name": "read_drafts_f16_w1000", "kind": "read", "dtype": "f16", "cache": "f16", "page": 32,
         "seqs": 16, "shortest": 900, "longest": 20000, "new": 5, "heads": 16, "kv_heads": 4,
         "dim": 128, "window": 1000, "sinks": 4},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["attend", "train", "append", "read", "read"])
        kv = rng.choice([1, 2, 4, 8])
        case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16"]),
                "seqs": _log_int(rng, 1, 64), "kv_heads": kv, "heads": kv * rng.choice([1, 2, 3, 4, 8]),
                "dim": rng.choice([64, 64, 80, 96, 128, 128])}
        if kind in ("attend", "train"):
            if kind == "train" and rng.random() < 0.25:
                case["dtype"] = "f32"
            case["longest"] = _log_int(rng, 17, 8000)
            case["shortest"] = _log_int(rng, max(1, case["longest"] // 12), case["longest"])
            case["prefix"] = rng.choice([0, 0, _log_int(rng, 1, 500)])
        else:
            case["cache"] = rng.choice(["f8", "f8", case["dtype"]])
            case["page"] = rng.choice([16, 32, 64, 128])
            case["longest"] = _log_int(rng, 40, 100000)
            case["shortest"] = _log_int(rng, max(8, case["longest"] // 20), case["longest"])
            if kind == "read":
                case["new"] = rng.choice([1, 1, 1, 2, 4, 7])
            else:
                case["new"] = min(case["shortest"], rng.choice([1, 1, 1, _log_int(rng, 2, 2000)]))
                case["turned"] = rng.choice([case["dim"], case["dim"] // 2])
        if kind != "append":
            case["window"] = rng.choice([0, _log_int(rng, 16, max(17, case["longest"]))])
            case["sinks"] = rng.choice([0, 1, 4, 33]) if case["window"] else 0
        if case["heads"] > 64:
            continue
        lens = _lens(case)
        if kind in ("attend", "train"):
            if case["seqs"] * case["heads"] * max(lens) * (max(lens) + case["prefix"]) <= MOST_SCORES / (
                    2 if kind == "train" else 1) / (2 if case["dtype"] == "f32" else 1):
                return case
        elif (case["seqs"] * case["longest"] * kv * case["dim"] * 2 <= MOST_CACHE
              and case["seqs"] * case["new"] * case["heads"] * case["dim"] <= 2e8
              and (kind == "append" or case["seqs"] * case["new"] * case["heads"] * case["longest"] <= 1e9)):
            return case


# ---- what a case amounts to -------------------------------------------------------------------
def _lens(case):
    """Lengths of the sequences, the same ones for every seed (which gets them in its own order):
    spaced evenly over their logarithm."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    if n == 1:
        return [hi]
    return [int(round(lo * (hi / lo) ** (b / (n - 1)))) for b in range(n)]


def _pairs(rows, cols, window, sinks):
    """Visible (row, column) pairs of one sequence, and the columns that some row sees."""
    p = np.arange(cols - rows, cols, dtype=np.int64)
    p = p[p >= 0]
    if not window:
        return int((p + 1).sum()), int(cols if p.size else 0)
    first = np.maximum(p - window + 1, 0)
    lone = np.minimum(first, sinks)  # first columns left of the window
    seen = cols - int(first[0]) + min(int(first[0]), sinks) if p.size else 0
    return int((p - first + 1 + lone).sum()), seen


def work(case):
    w, d, hq, hkv = _SIZE[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    lens = _lens(case)
    if case["kind"] in ("attend", "train"):
        pairs = sum(_pairs(n, n + case["prefix"], case["window"], case["sinks"])[0] for n in lens)
        tq, tk = sum(lens), sum(lens) + case["prefix"] * len(lens)
        once = w * d * (2 * tq * hq + 2 * tk * hkv) + 4 * tq * hq  # q, o, k, v, lse
        if case["kind"] == "attend":
            return {"bytes": once, "flops": 4 * d * hq * pairs}
        grad = w * d * (4 * tq * hq + 4 * tk * hkv) + 4 * tq * hq  # q, o, do, dq, k, v, dk, dv, lse
        return {"bytes": once + grad, "flops": 14 * d * hq * pairs}
    c, rows = _SIZE[case["cache"]], case["seqs"] * case["new"]
    if case["kind"] == "append":
        pages = sum((n - 1) // case["page"] - (n - case["new"]) // case["page"] + 1 for n in lens)
        kv = rows * hkv * d * 2 * (w + c)
        scales = 16 * pages * hkv if case["cache"] == "f8" else 0
        return {"bytes": kv + 2 * rows * hq * d * w + 4 * rows * case["turned"] + scales,
                "flops": 3 * rows * (hq + hkv) * case["turned"]}
    got = [_pairs(case["new"], n, case["window"], case["sinks"]) for n in lens]
    seen = sum(s for _, s in got)
    scales = 8 * hkv * seen // case["page"] if case["cache"] == "f8" else 0
    return {"bytes": 2 * seen * hkv * d * c + scales + 2 * rows * hq * d * w,
            "flops": 4 * d * hq * sum(p for p, _ in got)}


# ---- inputs -----------------------------------------------------------------------------------
def _normal(gen, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(_TORCH[dtype])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lens):
    return [0] + [int(x) for x in np.cumsum(lens)]


def _prepare_packed(case, gen, s):
    """Queries, keys and values side by side in one panel, as one projection writes them; behind a
    prefix the queries have a panel of their own."""
    d, hq, hkv, prefix = case["dim"], case["heads"], case["kv_heads"], case["prefix"]
    rows = [_lens(case)[i] for i in torch.randperm(case["seqs"], generator=gen, device="cuda").tolist()]
    cols = [n + prefix for n in rows]
    tq, tk, nq, nk = sum(rows), sum(cols), hq * d, hkv * d
    names = [""] if case["kind"] == "attend" else ["", "d_"]
    for pre in names:
        if prefix:
            s[pre + "qs"] = _normal(gen, (tq, nq), case["dtype"])
            s[pre + "kvs"] = _normal(gen, (tk, 2 * nk), case["dtype"])
            s[pre + "q"], kv = s[pre + "qs"], s[pre + "kvs"]
        else:
            s[pre + "qkvs"] = _normal(gen, (tq, nq + 2 * nk), case["dtype"])
            s[pre + "q"], kv = s[pre + "qkvs"][:, :nq], s[pre + "qkvs"][:, nq:]
        s[pre + "k"], s[pre + "v"] = kv[:, :nk], kv[:, nk:]
    s["o"] = torch.zeros(tq, nq, dtype=_TORCH[case["dtype"]], device="cuda")
    s["lse"] = torch.zeros(tq, hq, device="cuda")
    if case["kind"] == "train":
        s["d_o"] = _normal(gen, (tq, nq), case["dtype"])
    s["rows"], s["cols"] = rows, cols
    if not own:  # where the padded form finds its rows
        for name, lens in (("rows", rows), ("cols", cols)):
            at = torch.arange(max(lens), device="cuda")[None]
            n, first = _ints(lens)[:, None], _ints(_starts(lens)[:-1])[:, None]
            s["is_" + name], s["at_" + name] = at < n, (first + torch.minimum(at, n - 1)).long()
            s["back_" + name] = s["is_" + name].view(-1).nonzero().view(-1)
        return
    from spcomm3d_amd import device

    ctx = s["ctx"] = _context()
    s["band"] = ctx.band(rows, cols, window=case["window"], sinks=case["sinks"])
    h = s["h"] = {}
    for pre in names:
        if prefix:
            q, kv, at = _panel(ctx, s[pre + "qs"]), _panel(ctx, s[pre + "kvs"]), 0
        else:
            q = kv = _panel(ctx, s[pre + "qkvs"])
            at = nq
        h[pre + "q"] = q.heads(hq, d)
        h[pre + "k"], h[pre + "v"] = kv.heads(hkv, d, at), kv.heads(hkv, d, at + nk)
    h["o"] = _panel(ctx, s["o"]).heads(hq, d)
    h["lse"] = device.Vals(ctx, tq * hq, np.float32, dev=s["lse"].data_ptr())
    if case["kind"] == "train":
        h["d_o"] = _panel(ctx, s["d_o"]).heads(hq, d)


def _rotations(case, gen):
    """cos and sin side by side for every position."""
    half = case["turned"] // 2
    rate = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = torch.arange(case["longest"], device="cuda", dtype=torch.float64)[:, None] * rate
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _prepare_cache(case, gen, s):
    """A cache under way: pages dealt to the sequences at random, what they hold, the new rows."""
    d, hq, hkv, page, n = case["dim"], case["heads"], case["kv_heads"], case["page"], case["seqs"]
    lens = [_lens(case)[i] for i in torch.randperm(n, generator=gen, device="cuda").tolist()]
    most = -(-case["longest"] // page)
    held = [-(-x // page) for x in lens]
    pages = sum(held) + 3
    rows = n * case["new"]
    dealt = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    at = torch.arange(most, device="cuda")[None]
    own_at = _ints(_starts(held)[:-1])[:, None] + torch.minimum(at, _ints(held)[:, None] - 1)
    s["table"] = dealt[own_at.long()].contiguous()
    s["lens"], s["starts"] = _ints(lens), _ints([b * case["new"] for b in range(n + 1)])
    for name, shape in (("k", (pages, hkv, page, d)), ("v", (pages, hkv, d, page))):
        if case["cache"] == "f8":  # pages and heads of different sizes
            up = torch.randint(-9, -5, (pages, hkv), generator=gen, device="cuda").float().exp2()
            s[name + "_scale"] = up
            s["cache_" + name] = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
            step = max(1, (1 << 28) // (hkv * page * d))
            for p in range(0, pages, step):
                part = torch.randn((min(step, pages - p),) + shape[1:], generator=gen, device="cuda")
                s["cache_" + name][p:p + step] = part.mul_(100.0).clamp_(-F8_MOST, F8_MOST).to(torch.float8_e4m3fn)
        else:
            s["cache_" + name] = _normal(gen, shape, case["cache"])
    nq, nk = hq * d, hkv * d
    if case["kind"] == "append":
        s["qkvs"] = _normal(gen, (rows, nq + 2 * nk), case["dtype"])
        s["q"], s["k"], s["v"] = s["qkvs"][:, :nq], s["qkvs"][:, nq:nq + nk], s["qkvs"][:, nq + nk:]
        s["turned_q"] = torch.zeros(rows, nq, dtype=_TORCH[case["dtype"]], device="cuda")
        s["rotations"] = _rotations(case, gen)
    else:
        s["q"] = _normal(gen, (rows, nq), case["dtype"])
        s["o"] = torch.zeros(rows, nq, dtype=_TORCH[case["dtype"]], device="cuda")
    if not own:
        return
    from spcomm3d_amd import device

    ctx = s["ctx"] = _context()
    f8 = case["cache"] == "f8"
    s["cache"] = ctx.cache(case["cache"], pages, page, hkv, d, k=s["cache_k"].data_ptr(),
                           v=s["cache_v"].data_ptr(), k_scale=s["k_scale"].data_ptr() if f8 else None,
                           v_scale=s["v_scale"].data_ptr() if f8 else None)
    s["seqs"] = device.CacheSeqs(n, s["table"].data_ptr(), most, s["lens"].data_ptr(),
                                 s["starts"].data_ptr(), rows=rows, max_rows=case["new"],
                                 max_len=case["longest"])
    h = s["h"] = {}
    if case["kind"] == "append":
        qkv = _panel(ctx, s["qkvs"])
        h["q"], h["k"], h["v"] = qkv.heads(hq, d), qkv.heads(hkv, d, nq), qkv.heads(hkv, d, nq + nk)
        h["turned_q"] = _panel(ctx, s["turned_q"]).heads(hq, d)
        h["rotations"] = _panel(ctx, s["rotations"])
    else:
        h["q"], h["o"] = _panel(ctx, s["q"]).heads(hq, d), _panel(ctx, s["o"]).heads(hq, d)


_ctx = None


def _context():
    """The context of the process: one per rank, kept for its life."""
    global _ctx
    if _ctx is None:
        from spcomm3d_amd import device

        _ctx = device.Context(0)
    return _ctx


def _panel(ctx, t):
    name = {v: k for k, v in _TORCH.items()}[t.dtype]
    return ctx.panel(t.shape[0], t.shape[1], name, dev=t.data_ptr())


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    if case["kind"] in ("attend", "train"):
        _prepare_packed(case, gen, s)
    else:
        _prepare_cache(case, gen, s)
    torch.cuda.synchronize()
    return s


# ---- the plain forms ----------------------------------------------------------------------------
def _weights(scores, visible):
    """Softmax over the visible columns, in place of the scores, and the logarithm of its sum; rows
    that see nothing weigh nothing."""
    scores.masked_fill_(~visible, -math.inf)
    most = scores.amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, torch.zeros_like(most), most)
    scores.sub_(most).exp_()
    total = scores.sum(-1, keepdim=True)
    scores.div_(torch.where(total == 0, torch.ones_like(total), total))
    return scores, (most + total.log()).squeeze(-1)


def _visible(pos, cols, case):
    """Whether the row at position pos sees the column."""
    seen = cols <= pos
    if case["window"]:
        seen = seen & ((pos - cols < case["window"]) | (cols < case["sinks"]))
    return seen


def _plain_packed(s):
    case = s["case"]
    d, hkv, g = case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    b, nr, nc = case["seqs"], s["at_rows"].shape[1], s["at_cols"].shape[1]

    def by_row(t):  # [sequence, shared head, head of it * row, dim]
        t = t.float()[s["at_rows"]].view(b, nr, hkv, g, d)
        return t.permute(0, 2, 3, 1, 4).reshape(b, hkv, g * nr, d)

    def by_col(t):
        return t.float()[s["at_cols"]].view(b, nc, hkv, d).permute(0, 2, 1, 3).contiguous()

    def rows_of(t):  # and back
        t = t.view(b, hkv, g, nr, -1).permute(0, 3, 1, 2, 4).reshape(b * nr, -1)
        return t[s["back_rows"]]

    def cols_of(t):
        return t.permute(0, 2, 1, 3).reshape(b * nc, hkv * d)[s["back_cols"]]

    q, k, v = by_row(s["q"]), by_col(s["k"]), by_col(s["v"])
    n_rows, n_cols = s["is_rows"].sum(1), s["is_cols"].sum(1)
    pos = (n_cols - n_rows)[:, None, None] + torch.arange(nr, device="cuda")[None, :, None]
    visible = _visible(pos, torch.arange(nc, device="cuda")[None, None, :], case)
    visible = (visible & s["is_rows"][:, :, None] & s["is_cols"][:, None, :])[:, None, None]
    scale = 1.0 / math.sqrt(d)
    scores = torch.matmul(q * scale, k.transpose(2, 3).contiguous())
    p, lse = _weights(scores.view(b, hkv, g, nr, nc), visible)
    p = p.view(b, hkv, g * nr, nc)
    o = torch.matmul(p, v)
    out = {"o": rows_of(o).to(s["o"].dtype), "lse": rows_of(lse.reshape(b, hkv, g * nr, 1))}
    if case["kind"] == "attend":
        return out
    d_o = by_row(s["d_o"]) * s["is_rows"][:, None, None, :, None].expand(b, 1, g, nr, 1).reshape(b, 1, g * nr, 1)
    dp = torch.matmul(d_o, v.transpose(2, 3).contiguous())
    dv = torch.matmul(p.transpose(2, 3), d_o)
    ds = dp.sub_((d_o * o).sum(-1, keepdim=True)).mul_(p)
    dq, dk = torch.matmul(ds, k) * scale, torch.matmul(ds.transpose(2, 3), q) * scale
    out.update(dq=rows_of(dq).to(s["o"].dtype), dk=cols_of(dk).to(s["o"].dtype),
               dv=cols_of(dv).to(s["o"].dtype))
    return out


def _turn(x, cos, sin):
    """The rotation of the first columns of each head: pairs (j, j + half)."""
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _scale_for(most):
    """The smallest power of two 2^e, -40 <= e <= 40, with most <= 448 * 2^e."""
    m, e = torch.frexp(most)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(most == 0, torch.full_like(e, -40), e.clamp(-40, 40))
    return torch.ldexp(torch.ones_like(most), e)


def _f8_codes(x):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_append(s):
    case = s["case"]
    b, new, page, d, hkv = case["seqs"], case["new"], case["page"], case["dim"], case["kv_heads"]
    first = s["lens"] - new  # position of the first new row
    pos = (first[:, None] + torch.arange(new, device="cuda")).reshape(-1)
    half = case["turned"] // 2
    cos, sin = s["rotations"][pos][:, None, :half], s["rotations"][pos][:, None, half:]
    q = _turn(s["q"].float().view(b * new, -1, d), cos, sin)
    k = _turn(s["k"].float().view(b * new, hkv, d), cos, sin)
    s["turned_q"].copy_(q.view(b * new, -1))
    # the pages that get rows; sequences that fill fewer than others name their last one again
    count = (new + page - 2) // page + 1
    at = first[:, None] // page + torch.arange(count, device="cuda")
    at = torch.minimum(at, (s["lens"][:, None] - 1) // page)
    pages = torch.gather(s["table"].long(), 1, at.long())
    slot = at[:, :, None] * page + torch.arange(page, device="cuda")  # positions of a page's slots
    fresh = (slot >= first[:, None, None]) & (slot < s["lens"][:, None, None])
    row = torch.arange(b, device="cuda")[:, None, None] * new + (slot - first[:, None, None]).clamp(0, new - 1)
    older = slot < first[:, None, None]
    out = {"q": s["turned_q"]}
    for name, rows in (("k", k), ("v", s["v"].float().view(b * new, hkv, d))):
        held = s["cache_" + name]
        x = rows[row].permute(0, 1, 3, 2, 4)  # [sequence, page, head, slot, dim]
        held = held.view(torch.uint8) if case["cache"] == "f8" else held
        was = held[pages]
        was = was if name == "k" else was.transpose(3, 4)
        f, old = fresh[:, :, None, :, None], older[:, :, None, :, None]
        if case["cache"] == "f8":
            scales = s[name + "_scale"]
            before = scales[pages]
            need = _scale_for(torch.where(f, x.abs(), torch.zeros_like(x)).amax((3, 4)))
            begun = older.any(2)[:, :, None]
            scale = torch.where(begun, torch.maximum(need, before), need)
            ratio = torch.where(begun, before / scale, torch.ones_like(scale))
            kept = _f8_codes(was.contiguous().view(torch.float8_e4m3fn).float() * ratio[..., None, None])
            x = torch.where(f, _f8_codes(x / scale[..., None, None]), torch.where(old, kept, was))
            scales[pages] = scale
            out[name + "_scale"] = scales
        else:
            x = torch.where(f, x.to(held.dtype), was)
        held[pages] = x if name == "k" else x.transpose(3, 4)
        out["cache_" + name] = s["cache_" + name]
    return out


def _pages(held, at):
    """The pages of a cache that are named."""
    if held.dtype == torch.float8_e4m3fn:
        return held.view(torch.uint8)[at].view(held.dtype)
    return held[at]


def _plain_read(s):
    case = s["case"]
    b, new, d, hkv = case["seqs"], case["new"], case["dim"], case["kv_heads"]
    g, pages = case["heads"] // hkv, s["table"].long()
    k, v = _pages(s["cache_k"], pages).float(), _pages(s["cache_v"], pages).float()
    if case["cache"] == "f8":
        k, v = k * s["k_scale"][pages][..., None, None], v * s["v_scale"][pages][..., None, None]
    k = k.transpose(1, 2).reshape(b, hkv, -1, d)
    v = v.permute(0, 2, 1, 4, 3).reshape(b, hkv, -1, d)
    q = s["q"].float().view(b, new, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * new, d)
    pos = s["lens"][:, None, None] - new + torch.arange(new, device="cuda")[None, :, None]
    visible = _visible(pos, torch.arange(k.shape[2], device="cuda")[None, None, :], case)
    scores = torch.matmul(q * (1.0 / math.sqrt(d)), k.transpose(2, 3).contiguous())
    p, _ = _weights(scores.view(b, hkv, g, new, -1), visible[:, None, None])
    o = torch.matmul(p.view(b, hkv, g * new, -1), v)
    o = o.view(b, hkv, g, new, d).permute(0, 3, 1, 2, 4).reshape(b * new, -1)
    return {"o": o.to(s["o"].dtype)}


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"append": _plain_append, "read": _plain_read}.get(kind, _plain_packed)(s)
    ctx, case, h = s["ctx"], s["case"], s["h"]
    if kind == "append":
        s["cache"].append(s["seqs"], h["k"], h["v"], rotations=h["rotations"], q=h["q"], q_out=h["turned_q"])
        out = {"q": s["turned_q"], "cache_k": s["cache_k"], "cache_v": s["cache_v"]}
        if case["cache"] == "f8":
            out.update(k_scale=s["k_scale"], v_scale=s["v_scale"])
        return out
    if kind == "read":
        s["cache"].attend(s["seqs"], h["q"], h["o"], window=case["window"], sinks=case["sinks"])
        return {"o": s["o"]}
    ctx.attend(s["band"], h["q"], h["k"], h["v"], h["o"], lse=h["lse"])
    out = {"o": s["o"], "lse": s["lse"]}
    if kind == "train":
        ctx.attend_grad(s["band"], h["q"], h["k"], h["v"], h["o"], h["lse"], h["d_o"], h["d_q"], h["d_k"], h["d_v"])
        out.update(dq=s["d_q"], dk=s["d_k"], dv=s["d_v"])
    return out


# ---- the definition, in 64 bits -------------------------------------------------------------------
def _attention64(q, k, v, first, case, d_o=None):
    """One head of one sequence: the row i sits at position first + i of the columns."""
    pos = first + torch.arange(q.shape[0], device=q.device)
    c = torch.arange(k.shape[0], device=q.device)
    gap = pos[:, None] - c[None, :]
    hidden = gap < 0
    if case["window"]:
        hidden |= (gap >= case["window"]) & (c >= case["sinks"])[None, :]
    x = (q @ k.T) / math.sqrt(case["dim"])
    x[hidden] = -math.inf
    lse = torch.logsumexp(x, 1)
    p = torch.exp(x - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None])
    o = p @ v
    if d_o is None:
        return o, lse
    x = p * (d_o @ v.T - (d_o * o).sum(1)[:, None]) / math.sqrt(case["dim"])
    return o, lse, x @ k, x.T @ q, p.T @ d_o


def exact(case, seed):
    s = prepare(case, seed)
    d, hq, hkv = case["dim"], case["heads"], case["kv_heads"]
    g = hq // hkv
    if case["kind"] in ("attend", "train"):
        names = ["q", "k", "v"] + (["d_o"] if case["kind"] == "train" else [])
        x = {n: s[n].double().view(s[n].shape[0], -1, d) for n in names}
        out = {"o": torch.zeros_like(x["q"]), "lse": torch.zeros(x["q"].shape[:2], dtype=torch.float64, device="cuda")}
        if "d_o" in x:
            out.update(dq=torch.zeros_like(x["q"]), dk=torch.zeros_like(x["k"]), dv=torch.zeros_like(x["v"]))
        r0 = c0 = 0
        for n, m in zip(s["rows"], s["cols"]):
            r, c = slice(r0, r0 + n), slice(c0, c0 + m)
            for h in range(hq):
                d_o = x["d_o"][r, h] if "d_o" in x else None
                got = _attention64(x["q"][r, h], x["k"][c, h // g], x["v"][c, h // g], m - n, case, d_o)
                out["o"][r, h], out["lse"][r, h] = got[:2]
                if d_o is not None:
                    out["dq"][r, h] = got[2]
                    out["dk"][c, h // g] += got[3]
                    out["dv"][c, h // g] += got[4]
            r0, c0 = r0 + n, c0 + m
        return {n: t if n == "lse" else t.view(t.shape[0], -1) for n, t in out.items()}
    page, new, lens = case["page"], case["new"], s["lens"].tolist()
    table = s["table"].long()
    if case["kind"] == "read":
        q = s["q"].double().view(-1, hq, d)
        o = torch.zeros_like(q)
        for b, n in enumerate(lens):
            at = table[b, :-(-n // page)]
            k, v = _pages(s["cache_k"], at).float().double(), _pages(s["cache_v"], at).float().double()
            if case["cache"] == "f8":
                k *= s["k_scale"][at].double()[:, :, None, None]
                v *= s["v_scale"][at].double()[:, :, None, None]
            for h in range(hq):
                o[b * new:(b + 1) * new, h] = _attention64(
                    q[b * new:(b + 1) * new, h], k[:, h // g].reshape(-1, d)[:n],
                    v[:, h // g].transpose(1, 2).reshape(-1, d)[:n], n - new, case)[0]
        return {"o": o.view(o.shape[0], -1)}
    half = case["turned"] // 2
    x = {n: s[n].double().view(case["seqs"], new, -1, d) for n in ("q", "k", "v")}
    pos = torch.stack([torch.arange(n - new, n, device="cuda") for n in lens])
    cos, sin = s["rotations"].double()[pos].unsqueeze(2).chunk(2, -1)
    for n in ("q", "k"):
        left, right = x[n][..., :half].clone(), x[n][..., half:2 * half].clone()
        x[n][..., :half], x[n][..., half:2 * half] = left * cos - right * sin, right * cos + left * sin
    out = {"q": x["q"].reshape(case["seqs"] * new, -1)}
    for n in ("k", "v"):
        held, scales = s["cache_" + n].float().double(), s[n + "_scale"].double() if case["cache"] == "f8" else None
        for b, end in enumerate(lens):
            for p in range((end - new) // page, (end - 1) // page + 1):
                lo, hi = max(p * page, end - new), min((p + 1) * page, end)
                at = table[b, p]
                tile = held[at] if n == "k" else held[at].transpose(1, 2)  # [head, slot, dim]
                rows = x[n][b, lo - end + new:hi - end + new].transpose(0, 1)
                if scales is not None:
                    e = torch.ceil(torch.log2(rows.abs().amax((1, 2)) / F8_MOST)).clamp(-40, 40)
                    grown = torch.maximum(2.0 ** e, scales[at]) if lo > p * page else 2.0 ** e
                    if lo > p * page:
                        back = tile[:, :lo - p * page] * (scales[at] / grown)[:, None, None]
                        tile[:, :lo - p * page] = back.float().to(torch.float8_e4m3fn).double()
                    scales[at] = grown
                    rows = (rows / grown[:, None, None]).float().to(torch.float8_e4m3fn).double()
                tile[:, lo - p * page:hi - p * page] = rows
        out["cache_" + n] = held
        if scales is not None:
            out[n + "_scale"] = scales
    return out
