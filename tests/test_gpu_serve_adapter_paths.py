"""Low-rank adapters on each way that a call can be run. One launch leaves its workspace as it was; two hand the first
product over in it, so a filled workspace shows which way a call of a type and size takes."""
import numpy as np
import pytest

import g4serve as gs
import g4w8a8 as g4
from test_gpu_serve_adapters import Case

pytestmark = pytest.mark.gpu


def ways(c):
    """How many launches the call took: 1 or 2."""
    c.ws.fill(0xA5)
    c.call()
    g4.synchronize()
    return 2 if (c.ws.download() != 0xA5).any() else 1


def mixed_ids(r, t, adapters):
    """Runs of one adapter (pairs of its tiles), of unlike ones, of none, and rows that are left."""
    ids = np.sort(r.integers(-2, adapters, t))
    ids[: t // 3] = r.integers(0, adapters)
    return ids


@pytest.mark.parametrize("rank", [8, 16])
@pytest.mark.parametrize("x", ["f16", "i8"])
@pytest.mark.parametrize("t,k,n", [
    (40, 6400, 64),    # a few chunks of K a range, all at once
    (75, 20480, 40),   # ranges of more chunks than the ring has places, for one tile and for two
    (2100, 256, 6200),  # one chunk in one range
    (2048, 1536, 6144),  # prompts on a projection up
    (1300, 4104, 3000),  # K that ends inside a chunk
])
def test_low_ranks_in_two_launches(gpu, x, rank, t, k, n):
    r = np.random.default_rng(t + rank)
    c = Case(mixed_ids(r, t, 5), adapters=5, k=k, n=n, rank=rank, x=x, ranks=[rank, 3, rank, 0, rank - 5]).upload()
    assert ways(c) == 2
    c.check()


@pytest.mark.parametrize("x,rank,k", [("f16", 16, 6144), ("f16", 64, 1536), ("i8", 16, 4096), ("f32", 8, 1024)])
def test_small_calls_in_one_launch(gpu, x, rank, k):
    c = Case(mixed_ids(np.random.default_rng(k), 40, 3), adapters=3, k=k, n=300, rank=rank, x=x).upload()
    assert ways(c) == 1
    c.check()


@pytest.mark.parametrize("x", ["f16", "f32"])
@pytest.mark.parametrize("rank", [16, 64])
@pytest.mark.parametrize("t,k,n,launches", [(41, 512, 64, 1), (60, 8192, 96, 2), (1000, 6400, 2100, 2)])
def test_a_row_does_not_depend_on_its_batch(gpu, t, k, n, launches, rank, x):
    """The same row in another place, among other adapters, of as many tokens: the same bits, on either way."""
    if x == "f32" and rank == 64:
        launches = 2  # (whose one launch stops at rank 32)
    r = np.random.default_rng(8)
    kw = dict(k=k, n=n, rank=rank, x=x)
    c = Case([2] + [0] * (t - 1), **kw).upload()
    assert ways(c) == launches
    one = c.out.download()[0]
    d = Case(list(r.integers(0, 4, t - 11)) + [2] + [1] * 10, **kw)
    d.a, d.b, d.scales = c.a, c.b, c.scales
    d.x[t - 11], d.base[t - 11] = c.x[0], c.base[0]
    d.upload()
    for _ in range(3):
        gs.adapter_groups(d.d_ids, d.groups, 4)
        assert ways(d) == launches
        assert np.array_equal(d.out.download()[t - 11], one)


@pytest.mark.parametrize("rank,k", [(16, 64), (16, 8192), (64, 64)])
@pytest.mark.parametrize("x_log,b_log,s_log", [(126, -20, 17), (120, -24, 25), (-90, 10, -40), (-100, 14, -36), (0, 0, 0),
                                               (60, 12, -100)])
def test_scales_of_any_size(gpu, rank, k, x_log, b_log, s_log):
    """A first product next to f32's ends and a scale that takes the outputs back: as near as any other. Each row's x has
    one element, so that the sums are as large as their largest product."""
    c = Case([0, 1, 0, 2, 3, 1], k=k, rank=rank, x="f32", base=None, n=70)
    r = np.random.default_rng(k)
    c.x[:] = 0
    at = r.integers(0, k, 6)
    c.x[np.arange(6), at] = np.ldexp(r.uniform(0.5, 1, 6), x_log).astype(np.float32)
    c.a = r.uniform(0.5, 1, c.a.shape).astype(np.float16)
    c.b = np.ldexp(r.uniform(0.5, 1, c.b.shape) * r.choice([-1, 1], c.b.shape), b_log).astype(np.float16)
    c.scales = np.ldexp(r.uniform(0.5, 1, 4), s_log).astype(np.float32)
    c.upload()
    c.call()
    g4.synchronize()
    y, bound = c.want()
    assert np.abs(y).max() < 3e38 and np.abs(y).max() > 2.0 ** -125
    # outputs that come out small between larger terms lose the places that f32 has no numbers for
    assert (np.abs(c.out.download() - y) <= bound + np.abs(y) * 2.0 ** -24 + 2.0 ** -149).all()
