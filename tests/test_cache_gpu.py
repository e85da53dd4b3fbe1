"""The paged cache on the GPU: what an append leaves in it, bit for bit, and attention over it
against 64 bits."""
import numpy as np
import pytest

from spcomm3d_amd import _capi as capi
from spcomm3d_amd import device
from tests import _attention as ref

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF


class Bytes:
    """Device memory for any array."""

    def __init__(self, ctx, host):
        host = np.ascontiguousarray(host)
        self.host_dtype, self.shape = host.dtype, host.shape
        self.n = (host.nbytes + 3) // 4
        self.vals = ctx.vals(max(self.n, 4), np.float32)
        self.upload(host)

    def upload(self, host):
        raw = np.zeros(self.vals.n * 4, np.uint8)
        host = np.ascontiguousarray(host)
        raw[:host.nbytes] = host.reshape(-1).view(np.uint8)
        self.vals.upload(raw.view(np.float32))

    def download(self):
        raw = self.vals.download().view(np.uint8)
        return raw[:int(np.prod(self.shape)) * self.host_dtype.itemsize].view(self.host_dtype).reshape(self.shape)

    @property
    def ptr(self):
        return self.vals.device_ptr()

    def close(self):
        self.vals.close()


class World:
    """A cache, its sequences and panels for one call at a time; the host cache goes along."""

    def __init__(self, ctx, dtype, cache, page, heads, kv_heads, dim, nseq, max_len, seed=0):
        self.ctx, self.dtype, self.page = ctx, dtype, page
        self.heads, self.kv_heads, self.dim, self.max_len = heads, kv_heads, dim, max_len
        self.rng = np.random.default_rng(seed)
        self.stride = -(-max_len // page) + 1
        pages = nseq * (self.stride - 1) + 3
        self.host = ref.HostCache(cache, pages, page, kv_heads, dim)
        self.mem = {n: Bytes(ctx, getattr(self.host, n)) for n in ("k", "v", "k_scale", "v_scale")}
        f8 = cache == "f8"
        self.cache = ctx.cache(cache, pages, page, kv_heads, dim, k=self.mem["k"].ptr, v=self.mem["v"].ptr,
                               k_scale=self.mem["k_scale"].ptr if f8 else None,
                               v_scale=self.mem["v_scale"].ptr if f8 else None)
        self.order = self.rng.permutation(pages)[:nseq * (self.stride - 1)].reshape(nseq, -1).astype(np.uint32)
        self.lens = np.zeros(nseq, np.int64)
        self.dev = {}
        self.panels = []

    def seqs(self, new, max_rows=None, table=None):
        """The device arrays for sequences that have just grown by new[b] rows."""
        for x in self.dev.values():
            x.close()
        if table is None:
            table = np.full((len(self.lens), self.stride), NONE, np.uint32)
            for b, n in enumerate(self.lens):
                held = -(-int(n) // self.page)
                table[b, :held] = self.order[b, :held]
        self.table = table
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        self.dev = {"table": Bytes(self.ctx, table), "lens": Bytes(self.ctx, self.lens.astype(np.uint32)),
                    "starts": Bytes(self.ctx, starts)}
        return device.CacheSeqs(len(self.lens), self.dev["table"].ptr, table.shape[1], self.dev["lens"].ptr,
                                self.dev["starts"].ptr, rows=int(starts[-1]),
                                max_rows=max_rows or max(int(max(new)), 1), max_len=self.max_len)

    def heads_panel(self, rows, count, x=None, col=8):
        """Heads of a panel, and its values in float32; nothing given: not-a-number."""
        width = col + count * self.dim
        if x is None:
            x = self.rng.normal(size=(rows + 1, width))
        bits = ref.to_bits(x, self.dtype)
        p = self.ctx.panel(rows + 1, width, self.dtype)
        p.upload(bits)
        self.panels.append(p)
        return p.heads(count, self.dim, col), ref.from_bits(bits, self.dtype)[:rows, col:].reshape(rows, count, self.dim)

    def empty_panel(self, rows, count):
        return self.heads_panel(rows, count, np.full((rows + 1, 8 + count * self.dim), np.nan))[0]

    def got(self, heads, rows):
        x = ref.from_bits(heads.panel.download(), self.dtype)
        assert np.isnan(x[rows:]).all() and np.isnan(x[:, :8]).all()  # nothing around it is written
        return x[:rows, 8:].reshape(rows, heads.nheads, self.dim)

    def append(self, new, rotations=None, sizes=1.0, with_q=True, check=True):
        """Grow by new[b] rows through the library and on the host; compares every bit."""
        self.lens += np.array(new)
        seqs = self.seqs(new)
        rows = int(np.sum(new))
        k, kx = self.heads_panel(rows, self.kv_heads, self.rng.normal(size=(rows + 1, 8 + self.kv_heads * self.dim)) * sizes)
        v, vx = self.heads_panel(rows, self.kv_heads, self.rng.normal(size=(rows + 1, 8 + self.kv_heads * self.dim)) * sizes)
        q, qx = self.heads_panel(rows, self.heads)
        out = self.empty_panel(rows, self.heads)
        rot = None
        pos = np.concatenate([np.arange(n - m, n) for n, m in zip(self.lens, new)]) if rows else []
        kr, qr = kx.astype(np.float32), qx.astype(np.float32)
        if rotations is not None:
            rot = self.ctx.panel_from(rotations)
            self.panels.append(rot)
            kr, qr = ref.rotate(kr, rotations, pos), ref.rotate(qr, rotations, pos)
        self.cache.append(seqs, k, v, rotations=rot, q=q if with_q else None, q_out=out if with_q else None)
        r = 0
        for b, m in enumerate(new):
            self.host.append(self.order[b], int(self.lens[b]) - m, kr[r:r + m], vx[r:r + m].astype(np.float32))
            r += m
        if check:
            self.check_cache()
        if with_q:
            want = ref.from_bits(ref.to_bits(qr, self.dtype), self.dtype)
            assert np.array_equal(self.got(out, rows), want)

    def check_cache(self):
        for n in ("k", "v"):
            got, want = self.mem[n].download(), getattr(self.host, n)
            if self.host.dtype == "f8":
                got, want = ref.F8[got], ref.F8[want]
            assert np.array_equal(got, want, equal_nan=want.dtype.kind == "f"), n
        if self.host.dtype == "f8":
            for n in ("k_scale", "v_scale"):
                assert np.array_equal(self.mem[n].download(), getattr(self.host, n), equal_nan=True), n

    def put_host(self):
        for n in self.mem:
            self.mem[n].upload(getattr(self.host, n))

    def read(self, new, window=0, sinks=0, table=None, q=None, tol=1.0):
        seqs = self.seqs(new, table=table)
        rows = int(np.sum(new))
        q, qx = self.heads_panel(rows, self.heads) if q is None else q
        o = self.empty_panel(rows, self.heads)
        lse = self.ctx.vals(rows * self.heads + 1, np.float32)
        lse.fill(float("nan"))
        self.panels.append(lse)
        self.cache.attend(seqs, q, o, window=window, sinks=sinks, lse=lse)
        k, v = zip(*(self.host.values(self.table[b], int(n)) for b, n in enumerate(self.lens)))
        want = ref.band(qx, np.concatenate(k), np.concatenate(v), list(new), [int(n) for n in self.lens], window, sinks,
                        self.dim ** -0.5, self.dtype)
        got = self.got(o, rows)
        assert ref.worst(got, want["o"]) <= tol
        assert ref.worst(lse.download()[:-1].reshape(rows, self.heads).astype(np.float64), want["lse"]) <= tol
        assert np.isnan(lse.download()[-1])
        return got

    def fill(self, lens, sizes=1.0):
        """Sequences of these lengths, put on the device as the host cache has them."""
        for b, n in enumerate(lens):
            shape = (int(n), self.kv_heads, self.dim)
            self.host.append(self.order[b], 0, (self.rng.normal(size=shape) * sizes).astype(np.float32),
                             (self.rng.normal(size=shape) * sizes).astype(np.float32))
        self.lens = np.array(lens, dtype=np.int64)
        self.put_host()

    def close(self):
        self.cache.close()
        for x in list(self.mem.values()) + list(self.dev.values()) + self.panels:
            x.close()


def rotations(positions, n):
    a = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(n // 2) / (n // 2))
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


CACHES = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8"), ("f16", "f8")]


@pytest.mark.parametrize("dtype,cache", CACHES)
@pytest.mark.parametrize("page,dim,turned", [(16, 64, 64), (32, 128, 64), (64, 80, 16), (128, 16, None), (64, 128, 128)])
def test_append_bit_for_bit(ctx, dtype, cache, page, dim, turned):
    """Chunks, single tokens, sequences that get nothing; sizes that make scales grow."""
    w = World(ctx, dtype, cache, page, 6, 3, dim, 4, 300, seed=page + dim)
    rot = None if turned is None else rotations(300, turned)
    for new, sizes in (([5, 0, 33, 1], 1.0), ([1, 1, 1, 1], 0.1), ([1, 0, 1, 1], 40.0), ([130, 3, 0, 17], 2.0),
                       ([1, 1, 1, 1], 3000.0), ([1, 0, 0, 70], 0.01)):
        w.append(new, rot, sizes)
    w.read([1, 1, 1, 1])
    w.close()


@pytest.mark.parametrize("cache", ["bf16", "f8"])
def test_append_without_queries_and_in_one_sequence(ctx, cache):
    w = World(ctx, "bf16", cache, 16, 2, 1, 32, 1, 40, seed=2)
    w.append([1], with_q=False)
    w.append([39], rotations(40, 32), with_q=False)
    w.close()


def test_append_of_values_that_are_not_finite(ctx):
    """They do not count for the scale; infinities become the largest, NaN stays."""
    w = World(ctx, "bf16", "f8", 16, 2, 1, 32, 1, 16, seed=2)
    x = w.rng.normal(size=(1, 40))
    x[0, 8 + 3], x[0, 8 + 4], x[0, 8 + 5] = np.inf, np.nan, -np.inf
    w.lens += 1
    seqs = w.seqs([1])
    k, kx = w.heads_panel(1, 1, np.concatenate([x, x]))
    w.cache.append(seqs, k, k)
    w.host.append(w.order[0], 0, kx.astype(np.float32), kx.astype(np.float32))
    w.check_cache()
    assert ref.F8[w.host.k[w.order[0, 0], 0, 0, 3]] == 448.0
    w.close()


@pytest.mark.parametrize("size", [0.0, 1e-30, 1e-12, 1e20, 3e38])
def test_append_of_very_small_and_large_values(ctx, size):
    w = World(ctx, "bf16", "f8", 16, 1, 1, 16, 1, 32, seed=4)
    w.append([3], sizes=size)
    w.append([2], sizes=1.0)
    w.append([1], sizes=size)
    w.close()


def test_append_leaves_pages_it_does_not_have_and_rows_past_the_bounds(ctx):
    w = World(ctx, "bf16", "f8", 16, 2, 1, 32, 2, 64, seed=6)
    w.lens += np.array([20, 5])
    table = np.array([[w.order[0, 0], w.host.pages + 7, NONE], [w.order[1, 0], NONE, NONE]], np.uint32)
    seqs = w.seqs([20, 5], table=table)
    k, kx = w.heads_panel(25, 1)
    w.cache.append(seqs, k, k)
    x = kx.astype(np.float32)
    w.host.append(table[0], 0, x[:20], x[:20])
    w.host.append(table[1], 0, x[20:], x[20:])
    w.check_cache()
    w.close()


@pytest.mark.parametrize("dtype,cache", CACHES)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_read_lengths_about_pages_and_steps(ctx, dtype, cache, page):
    """One row a sequence; sequences of no token, one, about a page and about a step of 64."""
    lens = [0, 1, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 200]
    w = World(ctx, dtype, cache, page, 8, 2, 64, len(lens), 200, seed=page)
    w.fill(lens)
    w.read([1] * len(lens))
    w.close()


@pytest.mark.parametrize("dtype,cache", CACHES)
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 96, 112, 128])
def test_read_head_sizes_and_several_rows(ctx, dtype, cache, dim):
    w = World(ctx, dtype, cache, 32, 6, 2, dim, 5, 170, seed=dim)
    w.fill([3, 40, 170, 5, 100])
    w.read([3, 0, 7, 5, 1])
    w.close()


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (40, 0), (64, 4), (100, 70), (500, 3), (30, 1000)])
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f8")])
def test_read_a_window_and_the_first_tokens(ctx, dtype, cache, window, sinks):
    """Pages that nobody sees are not there."""
    lens, new = [900, 333, 64, 20], [1, 5, 2, 3]
    w = World(ctx, dtype, cache, 16, 4, 2, 64, 4, 900, seed=window)
    w.fill(lens)
    table = np.full((4, w.stride), NONE, np.uint32)
    for b, n in enumerate(lens):
        see = ref.visible(new[b], n, window, sinks).any(0)
        for p in range(-(-n // 16)):
            if see[p * 16:p * 16 + 16].any():
                table[b, p] = w.order[b, p]
    w.read(new, window, sinks, table=table)
    w.close()


@pytest.mark.parametrize("heads,kv_heads,rows", [(1, 1, 1), (16, 1, 1), (24, 3, 2), (5, 5, 4), (40, 2, 3), (8, 8, 40)])
def test_read_heads_that_share(ctx, heads, kv_heads, rows):
    w = World(ctx, "bf16", "f8", 64, heads, kv_heads, 64, 2, 300, seed=heads)
    w.fill([300, 130])
    w.read([rows, rows])
    w.close()


@pytest.mark.parametrize("dtype,cache", CACHES)
def test_read_long_sequences_shared_by_workgroups(ctx, dtype, cache):
    w = World(ctx, dtype, cache, 64, 4, 1, 128, 2, 9000, seed=9)
    w.fill([9000, 4100], sizes=0.5)
    first = w.read([1, 2])
    assert first.shape == (3, 4, 128)
    w.close()


def test_read_pages_of_very_different_scales(ctx):
    """The weights of half stay exact where a page's values are 2^20 times another's."""
    for dtype in ("f16", "bf16"):
        w = World(ctx, dtype, "f8", 16, 2, 1, 32, 3, 96, seed=3)
        w.fill([96, 70, 33])
        for b in range(3):
            for p in range(6):
                w.host.v_scale[w.order[b, p]] *= np.float32(2.0 ** (-20 if (b + p) % 2 else 0))
        w.put_host()
        w.read([1, 1, 2])
        w.close()


def test_read_rows_without_a_token_and_lengths_past_the_table(ctx):
    """A length below the rows: the first rows have no position and see nothing."""
    w = World(ctx, "bf16", "bf16", 16, 2, 1, 32, 2, 50, seed=1)
    w.fill([50, 2])
    got = w.read([1, 4])
    assert not got[1:3].any()
    # a length past max_len is taken for max_len
    seqs = w.seqs([1, 1])
    q, qx = w.heads_panel(2, 2)
    o, o2 = w.empty_panel(2, 2), w.empty_panel(2, 2)
    w.cache.attend(seqs, q, o)
    w.dev["lens"].upload(np.array([4000000000, 2], np.uint32))
    w.cache.attend(seqs, q, o2)
    assert np.array_equal(w.got(o, 2), w.got(o2, 2))
    w.close()


def test_read_values_that_are_not_finite_reach_only_the_rows_that_see_them(ctx):
    w = World(ctx, "bf16", "f8", 16, 2, 1, 32, 1, 40, seed=5)
    w.fill([40])
    at = w.order[0, 38 // 16]
    w.host.v[at, 0, 7, 38 % 16] = 0x7F
    w.put_host()
    seqs = w.seqs([4])
    q, qx = w.heads_panel(4, 2)
    o = w.empty_panel(4, 2)
    w.cache.attend(seqs, q, o)
    got = w.got(o, 4)
    k, v = w.host.values(w.order[0], 40)
    v[38, 0, 7] = 0
    want, bound = ref.band(qx, k, v, [4], [40], 0, 0, 32 ** -0.5, "bf16")["o"]
    want[2:, :, 7] = np.nan  # positions 38 and 39
    assert ref.worst(got, (want, bound)) <= 1
    w.close()


def test_step_recorded_and_replayed(ctx):
    """An append and a read in one graph that goes by the device's lengths and tables."""
    w = World(ctx, "bf16", "f8", 16, 4, 2, 64, 3, 1200, seed=8)
    w.fill([1000, 10, 47])
    rot = ctx.panel_from(rotations(1200, 64))
    seqs = w.seqs([1, 1, 1])
    q, _ = w.heads_panel(3, 4)
    k, _ = w.heads_panel(3, 2)
    v, _ = w.heads_panel(3, 2)
    turned, o, o2 = w.empty_panel(3, 4), w.empty_panel(3, 4), w.empty_panel(3, 4)
    w.cache.attend(seqs, q, o)  # makes the workspace
    ctx.capture_begin()
    w.cache.append(seqs, k, v, rotations=rot, q=q, q_out=turned)
    w.cache.attend(seqs, turned, o)
    graph = ctx.capture_end()
    for step in range(4):
        w.lens += 1
        table = np.full((3, w.stride), NONE, np.uint32)
        for b, n in enumerate(w.lens):
            table[b, :-(-int(n) // 16)] = w.order[b, :-(-int(n) // 16)]
        w.dev["table"].upload(table)
        w.dev["lens"].upload(w.lens.astype(np.uint32))
        xs = []
        for h in (q, k, v):
            bits = ref.to_bits(w.rng.normal(size=(h.panel.m, h.panel.n)), "bf16")
            h.panel.upload(bits)
            xs.append(ref.from_bits(bits, "bf16")[:3, 8:].reshape(3, h.nheads, 64).astype(np.float32))
        graph.launch()
        ctx.sync()
        pos = w.lens - 1
        kr = ref.rotate(xs[1], rotations(1200, 64), pos)
        for b in range(3):
            w.host.append(w.order[b], int(pos[b]), kr[b:b + 1], xs[2][b:b + 1])
        w.check_cache()
        kk, vv = zip(*(w.host.values(w.order[b], int(n)) for b, n in enumerate(w.lens)))
        qx = ref.from_bits(ref.to_bits(ref.rotate(xs[0], rotations(1200, 64), pos), "bf16"), "bf16")
        want = ref.band(qx, np.concatenate(kk), np.concatenate(vv), [1] * 3, [int(n) for n in w.lens], 0, 0, 0.125, "bf16")
        assert ref.worst(w.got(o, 3), want["o"]) <= 1
        w.cache.attend(seqs, turned, o2)
        assert np.array_equal(w.got(o, 3), w.got(o2, 3))
    graph.close()
    rot.close()
    w.close()


def test_owned_cache(ctx):
    c = ctx.cache("f8", 4, 32, 2, 64)
    assert all(c.device_ptrs())
    c.close()
    c = ctx.cache("bf16", 4, 32, 2, 64)
    assert c.device_ptrs()[0] and c.device_ptrs()[1] and c.device_ptrs()[2:] == (0, 0)
    c.close()


def test_refusals(ctx):
    for args in (("f32", 4, 16, 1, 64), ("bf16", 4, 24, 1, 64), ("bf16", 4, 16, 0, 64), ("bf16", 4, 16, 1, 136),
                 ("bf16", 4, 16, 1, 12), ("f8", 4, 16, 1, 24)):
        with pytest.raises(capi.Spc3dError) as e:
            ctx.cache(*args)
        assert e.value.status == capi.ERR_INVALID_ARG
    w = World(ctx, "bf16", "f8", 16, 4, 2, 64, 2, 40)
    w.fill([30, 40])
    lib, seqs = ctx._lib, w.seqs([1, 1])
    with pytest.raises(capi.Spc3dError):  # keys and values in one place
        ctx.cache("bf16", 2, 16, 2, 64, k=w.mem["k"].ptr, v=w.mem["k"].ptr)
    with pytest.raises(capi.Spc3dError):  # scales in 16 bits
        ctx.cache("bf16", 2, 16, 2, 64, k=w.mem["k"].ptr, v=w.mem["v"].ptr, k_scale=w.mem["k_scale"].ptr)
    with pytest.raises(capi.Spc3dError):  # none in 8 bits
        ctx.cache("f8", 2, 16, 2, 64, k=w.mem["k"].ptr, v=w.mem["v"].ptr)
    q, k, o = w.heads_panel(2, 4)[0], w.heads_panel(2, 2)[0], w.empty_panel(2, 4)
    f32 = ctx.panel(3, 256, "f32")
    half = ctx.panel(3, 264, "f16").heads(4, 64, 8)
    short = ctx.panel(1, 264, "bf16").heads(4, 64, 8)
    rot = ctx.panel(40, 64, "f32")
    few = ctx.panel(39, 64, "f32")
    wide = ctx.panel(40, 80, "f32")
    odd = ctx.panel(40, 24, "f32")

    def read(seqs=seqs, q=q, o=o, scale=0.1, lse=None):
        return lib.spc3d_cache_attend(ctx._h, w.cache._h, seqs._ref if seqs else None, q._ref, scale, 0, 0, o._ref,
                                      lse._h if lse else None)

    def append(k=k, v=k, rot=rot, q=q, q_out=o):
        return lib.spc3d_cache_append(ctx._h, w.cache._h, seqs._ref, k._ref, v._ref, rot._h,
                                      q._ref if q else None, q_out._ref if q_out else None)

    bad, mis = capi.ERR_INVALID_ARG, capi.ERR_SIZE_MISMATCH
    word = w.seqs([1, 1])
    seqs = word
    word._arg.reserved = 1
    assert read(seqs=word) == bad
    word._arg.reserved = 0
    word._arg.max_len = 1 << 31
    assert read(seqs=word) == capi.ERR_TOO_LARGE
    word._arg.max_len = 40
    lens, word._arg.lens = word._arg.lens, None
    assert read(seqs=word) == bad
    word._arg.lens = lens + 2
    assert read(seqs=word) == bad
    word._arg.lens = lens
    small = ctx.vals(7, np.float32)
    for want, kw in ((bad, dict(seqs=None)), (bad, dict(scale=0.0)), (bad, dict(q=f32.heads(4, 64))), (mis, dict(o=half)),
                     (mis, dict(q=short)), (mis, dict(q=w.heads_panel(2, 3)[0], o=w.heads_panel(2, 3)[0])),
                     (mis, dict(o=k)), (bad, dict(o=q)), (mis, dict(lse=small)),
                     (mis, dict(q=q.panel.heads(8, 32, 8)))):
        kw.setdefault("seqs", seqs)
        assert read(**kw) == want, kw
    for want, kw in ((mis, dict(k=q)), (mis, dict(v=half)), (mis, dict(rot=few)), (mis, dict(rot=wide)), (bad, dict(rot=odd)),
                     (bad, dict(q=None)), (bad, dict(q_out=None)), (bad, dict(q_out=q)), (mis, dict(q_out=k))):
        assert append(**kw) == want, kw
    # an operand that is the cache itself
    inside = ctx.panel(3, 264, "bf16", dev=w.mem["k"].ptr)
    assert read(o=inside.heads(4, 64, 8)) == bad
    assert append(k=inside.heads(2, 64, 8)) == bad
    for x in (f32, half.panel, short.panel, rot, few, wide, odd, small, inside):
        x.close()
    w.close()


def test_example_from_training_to_serving(ctx):
    """The example's own two parts.  An 8-bit value is off by 1/16 of itself at most and half the
    largest scale's spacing; keys move scores by as much of their size, so that a few tenths of an
    output's size is the most that a token may be off."""
    from spcomm3d_amd import attention_example as example

    losses = example.fit(ctx, steps=30)
    assert losses[-1] < 0.8 * losses[0] and all(b < a for a, b in zip(losses, losses[1:]))
    assert example.serve(ctx) < 0.3
