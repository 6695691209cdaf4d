"""Low-rank adapters beside a shared linear, against the formula in 64 bits."""
import numpy as np
import pytest

import g4serve as gs
import g4w8a8 as g4
from servecases import View, dev

pytestmark = pytest.mark.gpu

DT = {"f32": np.float32, "f16": np.float16, "i8": np.int8}


def values(r, kind, shape):
    x = r.standard_normal(shape)
    return np.clip(np.rint(30 * x), -128, 127).astype(np.int8) if kind == "i8" else x.astype(DT[kind])


class Case:
    """Random operands. ids: the adapter of each row."""

    def __init__(self, ids, adapters=4, k=256, n=64, rank=16, x="f16", base="f32", out="f32", ranks=None, scales=True, seed=0,
                 out_scale=0.0):
        r = np.random.default_rng(seed)
        self.ids, self.k, self.n, self.kinds = np.array(ids, np.int32), k, n, (x, base, out)
        t = len(ids)
        self.a = (r.standard_normal((adapters, rank, k)) / np.sqrt(k)).astype(np.float16)
        self.b = (0.3 * r.standard_normal((adapters, n, rank))).astype(np.float16)
        self.ranks = None if ranks is None else np.array(ranks, np.int32)
        if ranks is not None:  # what lies behind an adapter's rank is not used, whatever it holds
            for i, m in enumerate(ranks):
                self.a[i, max(0, m):] = np.nan
                self.b[i, :, max(0, m):] = np.inf
        self.scales = r.uniform(0.5, 2, adapters).astype(np.float32) if scales else None
        self.x = values(r, x, (t, k))
        self.base = None if base is None else values(r, base, (t, n))
        self.x_scale, self.base_scale = np.float32(0.04), np.float32(0.03)
        self.out_scale = np.float32(out_scale)

    def want(self):
        """(out, bound) before the output's type: sums of n products in f32 are n + 2 roundings off of the sum of
        magnitudes (in any order), H's error goes through B, H's two f16 values are 2^-23 off (two roundings more) or,
        by the smaller one's last place under the row's largest, 2^-38 of that, and each step of the epilogue adds
        one."""
        u = 2.0 ** -24
        x = self.x.astype(np.float64) * (float(self.x_scale) if self.kinds[0] == "i8" else 1.0)
        y = np.zeros((len(self.ids), self.n))
        if self.base is not None:
            y = self.base.astype(np.float64) * (float(self.base_scale) if self.kinds[1] == "i8" else 1.0)
        bound = np.abs(y) * 2 * u
        for i in range(len(self.a)):
            rows = np.nonzero(self.ids == i)[0]
            m = self.a.shape[1] if self.ranks is None else min(max(int(self.ranks[i]), 0), self.a.shape[1])
            a, b = self.a[i, :m].astype(np.float64), self.b[i, :, :m].astype(np.float64)
            s = 1.0 if self.scales is None else float(self.scales[i])
            h = x[rows] @ a.T
            h_off = (self.k + 2) * u * (np.abs(x[rows]) @ np.abs(a).T)
            d = s * (h @ b.T)
            h_off = h_off + (m + 4) * u * np.abs(h) + 2.0 ** -38 * np.abs(h).max(1, keepdims=True, initial=0)
            bound[rows] += s * (h_off @ np.abs(b).T) + 4 * u * (np.abs(d) + np.abs(y[rows]))
            y[rows] += d
        return y, bound

    def upload(self):
        t = len(self.ids)
        opt = lambda v: None if v is None else dev(v)
        self.adapters = gs.Adapters(dev(self.a), dev(self.b), opt(self.scales), opt(self.ranks))
        self.groups = g4.DeviceBuffer(gs.adapter_groups_bytes(t, len(self.a)))
        self.d_ids, self.d_x, self.d_base = dev(self.ids), dev(self.x), opt(self.base)
        self.ws = g4.DeviceBuffer(gs.adapter_workspace_bytes(self.adapters, t))
        self.out = dev(np.full((t, self.n), 77, DT[self.kinds[2]]))
        gs.adapter_groups(self.d_ids, self.groups, len(self.a))
        return self

    def call(self, out=None, stream=None, x=None, base=None):
        gs.adapter_linear(self.adapters, self.groups, self.d_x if x is None else x, self.d_base if base is None else base,
                          self.out if out is None else out, self.ws, x_scale=float(self.x_scale),
                          base_scale=float(self.base_scale), out_scale=float(self.out_scale), stream=stream)

    def check(self, got=None):
        g4.synchronize()
        got = self.out.download() if got is None else got
        y, bound = self.want()
        for i, a in enumerate(self.ids):
            if a == -2:
                assert (got[i] == 77).all()
        there = self.ids != -2
        got, y, bound = got[there], y[there], bound[there]
        kind, s = self.kinds[2], float(self.out_scale)
        if s:  # within half a step of the grid, at its ends past them
            v = got.astype(np.float64) * (s if kind == "i8" else 1.0)
            q = np.rint(v / s)
            assert (np.abs(v / s - q) <= (2.0 ** -11 if kind == "f16" else 2.0 ** -22) * np.abs(q)).all()
            lo, hi = np.where(q == -128, -np.inf, (q - 0.5) * s), np.where(q == 127, np.inf, (q + 0.5) * s)
            slack = bound + np.abs(y) * 2.0 ** -22
            assert ((y >= lo - slack) & (y <= hi + slack)).all()
            return
        if kind == "f16":
            bound = bound + np.maximum(np.abs(y) * 2.0 ** -11, 2.0 ** -25) * 1.01
        assert (np.abs(got - y) <= bound + np.abs(y) * 2.0 ** -24).all(), np.abs(got - y).max()


def ids_of(r, t, adapters, runs=False):
    if runs:
        return np.sort(r.integers(-1, adapters, t))
    return r.integers(-1, adapters, t)


@pytest.mark.parametrize("out", ["f32", "f16", "i8"])
@pytest.mark.parametrize("base", ["f32", "f16", "i8", None])
@pytest.mark.parametrize("x", ["f32", "f16", "i8"])
def test_types(gpu, x, base, out):
    ids = ids_of(np.random.default_rng(1), 37, 4)
    for n, scale in ((64, 0.03), (50, 0.03), (64, 0.0)):
        if out == "i8" and not scale:
            continue
        c = Case(ids, x=x, base=base, out=out, n=n, out_scale=scale).upload()
        c.call()
        c.check()


@pytest.mark.parametrize("k", [8, 24, 128, 136, 1536, 6144])
@pytest.mark.parametrize("x", ["f32", "f16", "i8"])
def test_inner_sizes(gpu, k, x):
    c = Case(ids_of(np.random.default_rng(2), 19, 4), k=k, x=x, rank=24).upload()
    c.call()
    c.check()


@pytest.mark.parametrize("rank", [16, 32, 64, 128])
@pytest.mark.parametrize("x", ["f32", "f16", "i8"])
def test_chunks_of_k(gpu, x, rank):
    """K about whole chunks of 256, and about as many as a block holds at once; long rows of zeros too."""
    for k in (248, 256, 264, 768, 1288, 2040, 2048, 2056, 2304, 2568):
        c = Case(ids_of(np.random.default_rng(k), 21, 3), adapters=3, k=k, n=40, x=x, rank=rank)
        c.x[5] = 0
        c.x[6, :-1] = 0
        c.upload()
        c.call()
        c.check()


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 96, 104, 128])
def test_ranks(gpu, rank):
    """The pool's rank, and adapters of less, of none and of a rank out of range."""
    for x in ("f16", "f32"):
        ids = ids_of(np.random.default_rng(rank), 70, 6)
        c = Case(ids, adapters=6, rank=rank, x=x, ranks=[rank, 1, rank - 3, 0, -5, rank]).upload()
        c.call()
        c.check()


def test_rank_past_the_pool_is_the_pools(gpu):
    c = Case([0, 1, 1], adapters=2, rank=16)
    c.ranks = np.array([16, 2 ** 31 - 1], np.int32)
    c.upload()
    c.call()
    c.check()


@pytest.mark.parametrize("n", [1, 3, 15, 16, 17, 255, 256, 257, 504, 511, 512, 513, 1032, 2048, 6145])
def test_outer_sizes(gpu, n):
    c = Case(ids_of(np.random.default_rng(3), 21, 4), n=n, x="i8").upload()
    c.call()
    c.check()


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 100, 1000, 2500])
@pytest.mark.parametrize("runs", [True, False])
@pytest.mark.parametrize("adapters", [1, 5, 40])
def test_batches(gpu, tokens, runs, adapters):
    ids = ids_of(np.random.default_rng(tokens), tokens, adapters, runs)
    c = Case(ids, adapters=adapters, k=192, n=80, x="f16").upload()
    c.call()
    c.check()


@pytest.mark.parametrize("rank", [8, 32, 40, 128])
@pytest.mark.parametrize("x", ["f32", "f16", "i8"])
def test_long_batches(gpu, x, rank):
    """Enough rows and sizes for H to go through memory: pairs of tiles of one adapter and of two, none, odd sizes."""
    r = np.random.default_rng(rank)
    for t, k, n, base, out in ((700, 6144, 1500, "f32", "f16"), (1300, 4104, 2056, "f16", "f32")):
        ids = np.concatenate([[2] * 41, np.sort(r.integers(-2, 5, t - 60)), [0] * 19])
        c = Case(ids, adapters=5, k=k, n=n, rank=rank, x=x, base=base, out=out, ranks=[rank, 3, rank, 0, rank - 5]).upload()
        assert c.ws.nbytes > t * rank * 4  # there is an H
        c.call()
        c.check()


def test_ids(gpu):
    """No adapter (-1, and ids out of range), no row (-2); none at all, all of one."""
    for ids in ([-1, -2, 0, 99, 3, -7, -2, 2 ** 31 - 1], [-1] * 5, [-2] * 5, [3] * 40, list(range(4)) * 9):
        c = Case(ids, adapters=4).upload()
        c.call()
        c.check()


def test_many_adapters(gpu):
    r = np.random.default_rng(5)
    c = Case(r.integers(-2, 3000, 700), adapters=3000, k=16, n=24, rank=8).upload()
    c.call()
    c.check()


def test_without_scales_and_in_place(gpu):
    r = np.random.default_rng(6)
    for kind in ("f32", "f16", "i8"):
        c = Case(ids_of(r, 33, 4), base=kind, out=kind, scales=False, out_scale=0.03 if kind == "i8" else 0.0).upload()
        c.d_base = c.out = dev(c.base)
        c.call()
        c.check()


def test_strides(gpu):
    """x, base and out as parts of wider rows, aligned and not, and adapters apart."""
    r = np.random.default_rng(7)
    for k, n, xs, bs, os_ in ((256, 64, 264, 68, 72), (256, 64, 512, 65, 67), (64, 30, 72, 100, 31)):
        for x, base, out in (("f16", "f32", "f32"), ("i8", "i8", "f16"), ("f32", "f16", "f32")):
            c = Case(ids_of(r, 20, 3), adapters=3, k=k, n=n, x=x, base=base, out=out).upload()
            views = []
            for host, width, stride in ((c.x, k, xs), (c.base, n, bs), (np.full((20, n), 77, DT[out]), n, os_)):
                wide = np.full((20, stride), 5, host.dtype)
                wide[:, :width] = host
                views.append(View(dev(wide), 0, (20, width), (stride, 1), host.dtype))
            a, b = (np.full((3, y[0].size + 24), np.nan, np.float16) for y in (c.a, c.b))
            for i in range(3):
                a[i, :c.a[i].size], b[i, :c.b[i].size] = c.a[i].ravel(), c.b[i].ravel()
            va = View(dev(a), 0, c.a.shape, (a.shape[1], k, 1), np.float16)
            vb = View(dev(b), 0, c.b.shape, (b.shape[1], c.b.shape[2], 1), np.float16)
            c.adapters = gs.Adapters(va, vb, dev(c.scales))
            c.call(out=views[2], x=views[0], base=views[1])
            g4.synchronize()
            wide = views[2].base.download()
            assert (wide[:, n:] == 5).all()
            c.check(wide[:, :n])


def test_far_rows(gpu):
    """Rows past 2^31 elements: x, base and out a row apart, and two adapters."""
    far = (1 << 31) + 64
    c = Case([1, 0], adapters=2, k=256, n=64, rank=16, x="i8", base="i8", out="i8", out_scale=0.03).upload()
    views = []
    for host in (c.x, c.base, np.full((2, 64), 77, np.int8)):
        room = g4.DeviceBuffer.empty((far + host.shape[1],), np.int8)
        for i in range(2):
            row = np.ascontiguousarray(host[i])
            g4._check(g4.lib().g4_memcpy_h2d(room.ptr + i * far, row.ctypes.data, row.nbytes, None))
        views.append(View(room, 0, host.shape, (far, 1), np.int8))
    pools = []
    for host in (c.a, c.b):
        room = g4.DeviceBuffer.empty((far + host[0].size,), np.float16)
        for i in range(2):
            one = np.ascontiguousarray(host[i])
            g4._check(g4.lib().g4_memcpy_h2d(room.ptr + 2 * i * far, one.ctypes.data, one.nbytes, None))
        pools.append(View(room, 0, host.shape, (far, host.shape[2], 1), np.float16))
    c.adapters = gs.Adapters(*pools, dev(c.scales))
    c.call(out=views[2], x=views[0], base=views[1])
    g4.synchronize()
    got = np.zeros((2, 64), np.int8)
    for i in range(2):
        g4._check(g4.lib().g4_memcpy_d2h(got[i].ctypes.data, views[2].ptr + i * far, 64, None))
    g4.synchronize()
    c.check(got)


def test_a_bad_row_stays_alone(gpu):
    """NaN and infinities in one row's x reach that row only."""
    c = Case([0, 0, 1, 0, -1, 0], x="f16")
    c.x[1] = np.nan
    c.x[3, 5] = np.inf
    c.x[4] = np.nan  # without an adapter: x is not read
    c.upload()
    c.call()
    g4.synchronize()
    got = c.out.download()
    assert np.isnan(got[1]).all() and not np.isfinite(got[3]).any()
    c.ids[[1, 3]], good = -2, got.copy()
    good[[1, 3]] = 77
    c.x[[1, 3, 4]] = 0
    c.check(good)


@pytest.mark.parametrize("rank", [8, 72])
def test_infinities_are_those_of_the_formula(gpu, rank):
    """An infinite x, and sums that pass f32: outputs of their sign, NaN where the formula has one."""
    c = Case([0, 0, 1, 1, 2], adapters=3, rank=rank, ranks=[1, 2, rank], x="f32", out="f32", k=64, n=40)
    c.b[0, ::7, 0] = 0
    c.x[0, 3], c.x[2, 5] = np.inf, -np.inf
    c.x[1] = np.float32(3e38) * np.sign(c.a[0, 0]).astype(np.float32)
    c.x[4, 9] = np.nan
    c.upload()
    c.call()
    g4.synchronize()
    got = c.out.download()
    with np.errstate(all="ignore"):
        for i, a in enumerate(c.ids):
            m = c.ranks[a]
            h = np.array([np.float32((c.x[i].astype(np.float64) * c.a[a, r]).sum()) for r in range(m)], np.float64)
            want = (c.base[i] + float(c.scales[a]) * (h * c.b[a, :, :m].astype(np.float64)).sum(1)).astype(np.float32)
            there = ~np.isfinite(want)
            assert np.array_equal(np.isnan(want), np.isnan(got[i])) and np.array_equal(want[there], got[i][there], equal_nan=True), i


@pytest.mark.parametrize("t,k,n", [(41, 512, 64), (1000, 6144, 1024)])
def test_a_row_does_not_depend_on_its_batch(gpu, t, k, n):
    """The same row in another place, among other adapters, of as many tokens: the same bits."""
    r = np.random.default_rng(8)
    c = Case([2] + [0] * (t - 1), k=k, n=n).upload()
    c.call()
    g4.synchronize()
    one = c.out.download()[0]
    d = Case(list(r.integers(0, 4, t - 11)) + [2] + [1] * 10, k=k, n=n)
    d.a, d.b, d.scales = c.a, c.b, c.scales
    d.x[t - 11], d.base[t - 11] = c.x[0], c.base[0]
    d.upload()
    for _ in range(3):
        gs.adapter_groups(d.d_ids, d.groups, 4)
        d.call()
        g4.synchronize()
        assert np.array_equal(d.out.download()[t - 11], one)


def test_replays(gpu):
    """Grouping and two linears captured, each with a workspace of its own, over changing ids."""
    r = np.random.default_rng(9)
    c, d = Case(ids_of(r, 50, 4)).upload(), Case(ids_of(r, 50, 4), n=130, x="i8", seed=1).upload()
    stream = g4.Stream()

    def both(s=None):
        gs.adapter_groups(c.d_ids, c.groups, 4, stream=s)
        c.call(stream=s)
        gs.adapter_linear(d.adapters, c.groups, d.d_x, d.d_base, d.out, d.ws, x_scale=float(d.x_scale), stream=s)

    both()
    g4.synchronize()
    graph = g4.Graph(stream, lambda: both(stream.handle))
    for i in range(4):
        c.ids = d.ids = ids_of(np.random.default_rng(i), 50, 4).astype(np.int32)
        c.d_ids.upload(c.ids)
        c.out.fill(0)
        g4.synchronize()
        graph.launch()
        stream.synchronize()
        c.check()
        d.check()
        both()
        c.check()
    graph.close()
