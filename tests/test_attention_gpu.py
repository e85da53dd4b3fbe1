"""Attention over a band on the GPU against 64 bits: forward, gradients, refusals, recording."""
import ctypes

import numpy as np
import pytest

from spcomm3d_amd import _capi as capi
from spcomm3d_amd import device
from tests import _attention as ref

pytestmark = pytest.mark.gpu


class Setup:
    """Operands of one call, side by side or apart, in panels with more rows and columns than needed."""

    def __init__(self, ctx, dtype, rows, cols, heads, kv_heads, dim, window, sinks, seed=0, packed=False,
                 scale=None):
        self.ctx, self.dtype, self.rows, self.cols = ctx, dtype, rows, cols
        self.heads, self.kv_heads, self.dim, self.window, self.sinks = heads, kv_heads, dim, window, sinks
        self.scale = dim ** -0.5 if scale is None else scale
        rng = np.random.default_rng(seed)
        self.T, self.S = sum(rows), sum(cols)
        nq, nk = heads * dim, kv_heads * dim
        self.val, self.h, self.panels = {}, {}, {}
        spare = 2

        def panel(name, n, width):
            bits = ref.to_bits(rng.normal(size=(n + spare, width)), dtype)
            p = ctx.panel(n + spare, width, dtype)
            p.upload(bits)
            self.panels[name] = p
            return p, ref.from_bits(bits, dtype)

        if packed:
            p, x = panel("qkv", self.T, nq + 2 * nk + 8)
            for name, col, count in (("q", 8, heads), ("k", 8 + nq, kv_heads), ("v", 8 + nq + nk, kv_heads)):
                self.h[name] = p.heads(count, dim, col)
                self.val[name] = x[:self.T, col:col + count * dim].reshape(-1, count, dim)
        else:
            for name, n, count, col in (("q", self.T, heads, 0), ("k", self.S, kv_heads, 16),
                                        ("v", self.S, kv_heads, 0)):
                p, x = panel(name, n, count * dim + col)
                self.h[name] = p.heads(count, dim, col)
                self.val[name] = x[:n, col:].reshape(n, count, dim)
        p, x = panel("d_o", self.T, nq)
        self.h["d_o"], self.val["d_o"] = p.heads(heads, dim), x[:self.T].reshape(-1, heads, dim)
        for name, n, count in (("o", self.T, heads), ("dq", self.T, heads), ("dk", self.S, kv_heads),
                               ("dv", self.S, kv_heads)):
            p = ctx.panel(n + spare, count * dim + 8, dtype)
            p.upload(ref.to_bits(np.full((n + spare, count * dim + 8), np.nan), dtype))
            self.panels[name] = p
            self.h[name] = p.heads(count, dim, 8)
        self.lse = ctx.vals(self.T * heads + 3, np.float32)
        self.lse.fill(float("nan"))
        self.band = ctx.band(rows, cols, window=window, sinks=sinks)

    def attend(self):
        h = self.h
        self.ctx.attend(self.band, h["q"], h["k"], h["v"], h["o"], lse=self.lse, scale=self.scale)

    def grad(self):
        h = self.h
        self.ctx.attend_grad(self.band, h["q"], h["k"], h["v"], h["o"], self.lse, h["d_o"], h["dq"], h["dk"],
                             h["dv"], scale=self.scale)

    def got(self, name):
        """The result, after checking that nothing around it was written."""
        x = ref.from_bits(self.panels[name].download(), self.dtype)
        n, h = x.shape[0] - 2, self.h[name]
        assert np.isnan(x[n:]).all() and np.isnan(x[:, :8]).all()
        return x[:n, 8:].reshape(n, h.nheads, h.dim)

    def got_lse(self):
        x = self.lse.download()
        assert np.isnan(x[self.T * self.heads:]).all()
        return x[:self.T * self.heads].reshape(self.T, self.heads).astype(np.float64)

    def want(self, grad=True):
        return ref.band(self.val["q"], self.val["k"], self.val["v"], self.rows, self.cols, self.window, self.sinks,
                        self.scale, self.dtype, self.val["d_o"] if grad else None, self.got("o") if grad else None)

    def close(self):
        self.band.close()
        self.lse.close()
        for p in self.panels.values():
            p.close()

    def check(self):
        self.attend()
        self.grad()
        want = self.want()
        for name in ("o", "dq", "dk", "dv"):
            assert ref.worst(self.got(name), want[name]) <= 1, name
        assert ref.worst(self.got_lse(), want["lse"]) <= 1


# rows, columns, window, sinks
SHAPES = {
    "one": ([1], [1], 0, 0),
    "one_of_many": ([1], [131], 0, 0),
    "tile": ([64], [64], 0, 0),
    "tile_and_one": ([65], [65], 0, 0),
    "ragged": ([3, 70, 1, 129], [3, 70, 1, 129], 0, 0),
    "prefix": ([17, 5], [80, 140], 0, 0),
    "unseen_rows": ([90, 4], [33, 2], 0, 0),       # more rows than columns: the first see nothing
    "nothing": ([0, 5, 7, 0], [4, 0, 7, 0], 0, 0),  # no rows, no columns, neither
    "window_one": ([100], [100], 1, 0),
    "window": ([200, 33], [200, 40], 50, 0),
    "window_sinks": ([300], [300], 64, 4),
    "sinks_past_a_tile": ([260, 10], [290, 10], 40, 70),
    "window_far": ([5], [700], 100, 3),
    "sinks_of_a_later_row": ([40], [40], 8, 30),
    "long": ([515], [515], 0, 0),
}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,dim,heads,kv_heads", [("f32", 64, 2, 1), ("bf16", 128, 4, 2), ("f16", 96, 3, 3)])
def test_band_against_64_bits(ctx, shape, dtype, dim, heads, kv_heads):
    rows, cols, window, sinks = SHAPES[shape]
    s = Setup(ctx, dtype, rows, cols, heads, kv_heads, dim, window, sinks, seed=len(shape))
    s.check()
    s.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [8, 24, 64, 72, 80, 96, 104, 128])
def test_head_sizes_side_by_side(ctx, dtype, dim):
    s = Setup(ctx, dtype, [37, 90], [37, 90], 8, 8, dim, 60, 2, seed=dim, packed=True)
    s.check()
    s.close()


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (16, 8), (24, 8), (12, 4), (5, 5)])
def test_shared_heads_sum_their_gradients(ctx, heads, kv_heads):
    s = Setup(ctx, "bf16", [150, 20], [150, 20], heads, kv_heads, 64, 0, 0, seed=heads)
    s.check()
    s.close()


def test_many_tiles_take_the_large_ones(ctx):
    """Enough rows and heads for tiles of 128 rows, and columns in pieces that are joined."""
    s = Setup(ctx, "bf16", [1100, 700], [1100, 700], 40, 8, 64, 200, 4, seed=5)
    s.check()
    s.close()


def test_a_large_scale_and_scores_far_apart(ctx):
    s = Setup(ctx, "f32", [130], [130], 2, 2, 32, 0, 0, seed=8, scale=9.0)
    s.check()
    s.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(ctx, dtype):
    """inf and NaN in v (and NaN in k) at columns that some rows of the same tile do not see."""
    rows, window, sinks = 150, 40, 2
    s = Setup(ctx, dtype, [rows], [rows], 2, 1, 64, window, sinks, seed=3)
    v = s.panels["v"].download()
    v[100, 3], v[100, 5], v[20, 7], v[1, 9] = (ref.to_bits(np.array([[x]]), dtype)[0, 0]
                                               for x in (np.inf, np.nan, -np.inf, np.nan))
    s.panels["v"].upload(v)
    k = s.panels["k"].download()
    k[120, 16:] = ref.to_bits(np.full((1, 1), np.nan), dtype)[0, 0]
    s.panels["k"].upload(k)
    s.attend()
    got = s.got("o")
    s.val["v"] = ref.from_bits(v, dtype)[:rows].reshape(rows, 1, 64)
    clean = s.val["v"].copy()
    clean[~np.isfinite(clean)] = 0
    kept = s.val["v"]
    s.val["v"] = clean
    want, bound = s.want(grad=False)["o"]
    see = ref.visible(rows, rows, window, sinks)
    sees_k = see[:, 120]
    for c, d in ((100, 3), (100, 5), (20, 7), (1, 9)):
        want[see[:, c], :, d] = kept[c, 0, d]
    assert np.isnan(got[sees_k]).all()
    assert ref.worst(got[~sees_k], (want[~sees_k], bound[~sees_k])) <= 1
    s.close()


def test_scores_of_the_lowest_value_weigh_nothing(ctx):
    """A column whose scores are the type's lowest value is seen and gets no weight."""
    s = Setup(ctx, "f32", [40], [40], 1, 1, 32, 0, 0, seed=4)
    q, k = s.panels["q"].download(), s.panels["k"].download()
    q[:, 0], k[:, 16] = 1.0, 0.0
    k[5, 16] = np.finfo(np.float32).min
    s.panels["q"].upload(q)
    s.panels["k"].upload(k)
    s.val["q"], s.val["k"] = q[:40].reshape(40, 1, 32).astype(np.float64), k[:40, 16:].reshape(40, 1, 32).astype(np.float64)
    s.attend()
    got = s.got("o")
    P, _ = ref.softmax(s.scale * (s.val["q"][:, 0] @ s.val["k"][:, 0].T), ref.visible(40, 40, 0, 0))
    assert P[20, 5] == 0 and np.allclose(got[:, 0], P @ s.val["v"][:, 0], rtol=0, atol=2e-5)
    s.close()


def test_gradients_against_differences(ctx):
    """The derivative of sum(w o) along random directions, by differences of the 64-bit form."""
    rows, cols, H, G, D, window, sinks = [19, 30], [25, 30], 4, 2, 16, 12, 3
    s = Setup(ctx, "f32", rows, cols, H, G, D, window, sinks, seed=21)
    s.attend()
    s.grad()
    rng = np.random.default_rng(5)

    def loss(x):
        o = ref.band(x["q"], x["k"], x["v"], rows, cols, window, sinks, s.scale, "f32")["o"][0]
        return float((o * s.val["d_o"]).sum())

    for name in ("q", "k", "v"):
        g = s.got("d" + name)
        for _ in range(4):
            step = rng.normal(size=g.shape)
            at = {n: s.val[n].copy() for n in ("q", "k", "v")}
            h = 1e-5
            at[name] = s.val[name] + h * step
            up = loss(at)
            at[name] = s.val[name] - h * step
            diff = (up - loss(at)) / (2 * h)
            # differences: h^2 of third derivatives; the 32-bit gradient: 1e-5 of its magnitudes
            assert abs(diff - float((g * step).sum())) <= 1e-6 + 1e-5 * float(np.abs(g * step).sum())
    s.close()


def test_softmax_between_the_two_products(ctx):
    """The same numbers as the library's SDDMM and SpMM over the pattern, with a softmax between."""
    n, D, window, sinks = 300, 32, 64, 4
    s = Setup(ctx, "f32", [n], [n], 1, 1, D, window, sinks, seed=6)
    s.attend()
    see = ref.visible(n, n, window, sinks)
    ii, jj = (x.astype(np.uint32) for x in np.nonzero(see))
    q, k, v = (np.ascontiguousarray(s.val[x][:, 0], dtype=np.float32) for x in ("q", "k", "v"))
    plan = ctx.plan(n, n, ii, jj, np.full(ii.size, s.scale, np.float32))
    A, B, V, Y, C = ctx.panel_from(q), ctx.panel_from(k), ctx.panel_from(v), ctx.panel(n, D, "f32"), ctx.vals(ii.size, "f32")
    ctx.sddmm(plan, A, B, C)
    scores = np.full((n, n), -np.inf)
    scores[ii, jj] = C.download()
    P, _ = ref.softmax(scores, see)
    plan.set_values(P[ii, jj].astype(np.float32))
    Y.fill(0.0)
    ctx.spmm(plan, V, Y)
    assert np.allclose(s.got("o")[:, 0], Y.download(), rtol=0, atol=2e-5)
    for h in (plan, A, B, V, Y, C):
        h.close()
    s.close()


def test_runs_give_the_same_bits(ctx):
    s = Setup(ctx, "bf16", [900], [900], 8, 2, 128, 100, 4, seed=13)
    s.attend()
    s.grad()
    first = [s.panels[n].download() for n in ("o", "dq", "dk", "dv")]
    for _ in range(3):
        s.attend()
        s.grad()
        for a, n in zip(first, ("o", "dq", "dk", "dv")):
            assert np.array_equal(a, s.panels[n].download())
    s.close()


def test_recorded_step_replays(ctx):
    s = Setup(ctx, "bf16", [260, 31], [260, 31], 4, 2, 64, 90, 4, seed=17)
    ctx.capture_begin()
    s.attend()
    with pytest.raises(capi.Spc3dError):  # its workspace is not there yet
        s.grad()
    ctx.capture_end().close()
    s.attend()
    s.grad()
    ctx.capture_begin()
    s.attend()
    s.grad()
    graph = ctx.capture_end()
    rng = np.random.default_rng(2)
    for _ in range(3):
        for name in ("q", "k", "v", "d_o"):
            bits = ref.to_bits(rng.normal(size=(s.panels[name].m, s.panels[name].n)), "bf16")
            s.panels[name].upload(bits)
            h, n = s.h[name], s.panels[name].m - 2
            s.val[name] = ref.from_bits(bits, "bf16")[:n, h.col:].reshape(n, h.nheads, h.dim)
        graph.launch()
        ctx.sync()
        replay = {n: s.got(n) for n in ("o", "dq", "dk", "dv")}
        want = s.want()
        s.attend()
        s.grad()
        for n, x in replay.items():
            assert np.array_equal(x, s.got(n)) and ref.worst(x, want[n]) <= 1
    graph.close()
    s.close()


def test_refusals(ctx):
    s = Setup(ctx, "bf16", [20], [20], 4, 2, 64, 0, 0)
    h, lib, ok = s.h, ctx._lib, s.scale

    def attend(q=h["q"], k=h["k"], v=h["v"], o=h["o"], scale=ok, lse=None, band=None):
        return lib.spc3d_attend(ctx._h, (band or s.band)._h, q._ref if q else None, k._ref, v._ref, scale, o._ref,
                                lse._h if lse else None)

    P = s.panels
    f32 = ctx.panel(22, 256, "f32")
    f8 = ctx.panel(22, 256, "e4m3")
    odd = ctx.panel(22, 260, "bf16")
    short = ctx.panel(19, 256, "bf16")
    small = ctx.vals(79, np.float32)
    wide = ctx.vals(80, np.float64)
    for want, kw in (
            (capi.ERR_INVALID_ARG, dict(q=None)),
            (capi.ERR_INVALID_ARG, dict(scale=0.0)),
            (capi.ERR_INVALID_ARG, dict(scale=-1.0)),
            (capi.ERR_INVALID_ARG, dict(scale=float("inf"))),
            (capi.ERR_INVALID_ARG, dict(scale=float("nan"))),
            (capi.ERR_SIZE_MISMATCH, dict(o=f32.heads(4, 64))),           # another type
            (capi.ERR_INVALID_ARG, dict(q=f8.heads(4, 64))),              # no such operand
            (capi.ERR_INVALID_ARG, dict(o=odd.heads(4, 64))),             # rows of no whole vectors
            (capi.ERR_INVALID_ARG, dict(k=P["k"].heads(2, 64, 4))),       # nor its first column
            (capi.ERR_SIZE_MISMATCH, dict(k=P["k"].heads(2, 64, 24))),    # ends behind the panel
            (capi.ERR_SIZE_MISMATCH, dict(o=short.heads(4, 64))),         # fewer rows than the band's
            (capi.ERR_INVALID_ARG, dict(q=P["q"].heads(4, 60))),          # no multiple of 8
            (capi.ERR_INVALID_ARG, dict(q=P["q"].heads(1, 136))),         # too wide
            (capi.ERR_INVALID_ARG, dict(q=P["q"].heads(0, 64))),
            (capi.ERR_SIZE_MISMATCH, dict(q=P["q"].heads(8, 32))),        # not as wide as k's
            (capi.ERR_SIZE_MISMATCH, dict(q=P["q"].heads(3, 64), o=P["o"].heads(3, 64, 8))),  # no multiple of k's
            (capi.ERR_SIZE_MISMATCH, dict(v=P["v"].heads(1, 64))),
            (capi.ERR_SIZE_MISMATCH, dict(o=P["o"].heads(3, 64, 8))),
            (capi.ERR_INVALID_ARG, dict(o=h["q"])),                       # overlaps an input
            (capi.ERR_SIZE_MISMATCH, dict(lse=small)),
            (capi.ERR_SIZE_MISMATCH, dict(lse=wide))):
        assert attend(**kw) == want, kw
        assert lib.spc3d_last_error()
    bad = device.Heads(P["q"], 4, 64)
    bad._arg.reserved = 1
    assert attend(q=bad) == capi.ERR_INVALID_ARG
    other = device.Context(0)
    band = other.band([20])
    assert attend(band=band) == capi.ERR_INVALID_ARG
    band.close()
    other.close()
    grad = lambda **kw: lib.spc3d_attend_grad(  # noqa: E731
        ctx._h, s.band._h, *(({**h, **kw})[n]._ref for n in "qkv"), ok, h["o"]._ref, s.lse._h,
        *(({**h, **kw})[n]._ref for n in ("d_o", "dq", "dk", "dv")))
    assert grad(dq=h["q"]) == capi.ERR_INVALID_ARG
    assert grad(dk=P["dv"].heads(2, 64, 8)) == capi.ERR_INVALID_ARG      # two gradients in one place
    assert grad(dk=P["dq"].heads(4, 64, 8)) == capi.ERR_SIZE_MISMATCH
    assert lib.spc3d_attend_grad(ctx._h, s.band._h, h["q"]._ref, h["k"]._ref, h["v"]._ref, ok, h["o"]._ref, None,
                                 h["d_o"]._ref, h["dq"]._ref, h["dk"]._ref, h["dv"]._ref) == capi.ERR_INVALID_ARG
    with pytest.raises(capi.Spc3dError):
        ctx.band([1 << 31], [5])
    # an SDDMM does not take such panels, nor a value vector their types
    plan = ctx.plan(2, 2, [0], [1], np.ones(1, np.float32))
    C = ctx.vals(1, "f32")
    assert lib.spc3d_sddmm(ctx._h, plan._h, P["q"]._h, P["q"]._h, C._h) == capi.ERR_SIZE_MISMATCH
    hv = ctypes.c_void_p()
    assert lib.spc3d_vals_create(ctx._h, capi.BF16, 4, ctypes.byref(hv)) == capi.ERR_INVALID_ARG
    for x in (plan, C, f32, f8, odd, short, small, wide):
        x.close()
    s.close()


@pytest.mark.parametrize("dtype,one", [("bf16", 0x3F80), ("f16", np.float16(1.0)), ("e4m3", 0x38)])
def test_panels_of_the_short_types(ctx, dtype, one):
    p, q = ctx.panel(5, 7, dtype), ctx.panel(5, 7, dtype)
    p.fill(1.0)
    assert (p.download() == one).all()
    x = np.arange(35).reshape(5, 7).astype(p.dtype)
    p.upload(x)
    q.copy_from(p)
    assert np.array_equal(q.download(), x)
    p.close()
    q.close()
