"""Sampling with temperature, top-k, top-p and min-p, against its definition in 64 bits."""
import numpy as np
import pytest

import g4serve as gs
import g4w8a8 as g4
from servecases import View, dev

pytestmark = pytest.mark.gpu

LAST = np.float32(1 - 2.0 ** -24)


def weights(x, cap, t):
    """(log weights relative to the largest, sum of weights) of a row in 64 bits; a NaN has no weight."""
    y = x.astype(np.float64)
    y = np.where(np.isnan(y), -np.inf, cap * np.tanh(y / cap) if cap else y)
    y = np.where(x == -np.inf, -np.inf, y)
    top = y.max()
    if top == np.inf:
        z = np.where(y == top, 0.0, -np.inf)
    else:
        with np.errstate(invalid="ignore"):
            z = np.where(y == -np.inf, -np.inf, (y - top) / t)
    return z, np.exp(z).sum()


def sample(x, cap, t, k, p, m, u, slip=(0.0, 0.0)):
    """(token, log probability) of one row. slip: how far top-p's target and the draw's are moved, in parts."""
    if not (x > -np.inf).any():
        return -1, 0.0
    greedy = not t > 0
    z, total = weights(x, cap, 1.0 if greedy else float(np.float32(t)))
    order = np.lexsort((np.arange(len(x)), -np.where(np.isnan(x), -np.inf, x + 0.0)))
    if greedy:
        return int(order[0]), z[order[0]] - np.log(total)
    order = order[x[order] > -np.inf]
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        w = np.exp(z[order])
        before = np.concatenate([[0], np.cumsum(w)[:-1]])
        keep = before < max(float(np.float32(p)), 0) * w.sum() * (1 + slip[0])
        keep[0] = True
        order = order[keep]
    if m > 0:
        order = order[z[order] >= np.log(min(float(np.float32(m)), 1.0))]
    order = np.sort(order)
    run = np.cumsum(np.exp(z[order]))
    u = min(max(float(u), 0.0), float(LAST)) if u == u else 0.0
    at = int((run <= u * run[-1] * (1 + slip[1])).sum())
    return int(order[min(at, len(order) - 1)]), None


def check(logits, rows, params, u, got, cap, index=None):
    """Every row's token is what the definition gives; where a target lies next to a running sum, either neighbour.
    Weights are off by 1.2e-12 (2^z), 1e-13 of a logit over the temperature (the softcap) and half a step each, together
    by `slip` of the sum; the log probability by that and its rounding to f32."""
    tokens, lps = got
    vocab = logits.shape[1]
    shift = min(51, 62 - int(np.ceil(np.log2(vocab))) if vocab > 1 else 51)
    off = 0
    for i in range(rows):
        r = i if index is None else index[i]
        t, k, p, m = (params[n][i] if params[n] is not None else d
                      for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
        if not 0 <= r < len(logits):
            assert tokens[i] == -1 and lps[i] == 0, i
            continue
        x = logits[r]
        slip = vocab * 2.0 ** -(shift + 1) + 2e-12 + (1e-12 / float(t) if cap and t > 0 else 0)
        steps = [(a * slip, b * slip) for a in (0, -1, 1) for b in (0, -1, 1)]
        want = sample(x, cap, t, k, p, m, u[i])[0]
        if tokens[i] != want:
            assert tokens[i] in [sample(x, cap, t, k, p, m, u[i], s)[0] for s in steps], \
                (i, t, k, p, m, u[i], tokens[i], want)
            off += 1
        if want < 0:
            assert lps[i] == 0
            continue
        z, total = weights(x, cap, float(np.float32(t)) if t > 0 else 1.0)
        lp = z[tokens[i]] - np.log(total)
        assert abs(lps[i] - lp) <= abs(lp) * 2.0 ** -24 * 1.01 + 2 * slip + 2.0 ** -50, (i, lps[i], lp)
    return off


def run(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, cap=0.0, index=None, stream=None, d_logits=None):
    rows, vocab = len(u), logits.shape[1]
    opt = lambda x, dt: None if x is None else dev(np.asarray(x, dt))
    tokens, lps = dev(np.full(rows, -7, np.int32)), dev(np.full(rows, 9, np.float32))
    gs.sample_tokens(dev(logits) if d_logits is None else d_logits, dev(np.asarray(u, np.float32)), tokens, lps,
                     g4.DeviceBuffer(gs.sample_workspace_bytes(rows, vocab)), row_index=opt(index, np.int32),
                     temperature=opt(temperature, np.float32), top_k=opt(top_k, np.int32), top_p=opt(top_p, np.float32),
                     min_p=opt(min_p, np.float32), cap=cap, stream=stream)
    g4.synchronize()
    return tokens.download(), lps.download()


def both(logits, u, cap=0.0, index=None, **params):
    p = {n: params.get(n) for n in ("temperature", "top_k", "top_p", "min_p")}
    got = run(logits, u, cap=cap, index=index, **p)
    return check(logits, len(u), p, u, got, cap, index)


def mixed(r, rows, vocab):
    """Filters of every kind over the rows."""
    pick = lambda *v: r.choice(v, rows)
    return {"temperature": pick(0.0, 0.3, 0.8, 1.0, 2.5).astype(np.float32), "top_k": pick(0, 1, 2, 40, 700, vocab).astype(np.int32),
            "top_p": pick(1.0, 0.02, 0.5, 0.95, 0.999).astype(np.float32), "min_p": pick(0.0, 0.0, 0.02, 0.3).astype(np.float32)}


def numbers(r, rows):
    u = r.random(rows).astype(np.float32)
    u[:3] = [0.0, LAST, 0.5][:len(u[:3])]
    return u


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 1024, 1025, 4096, 4097, 32003, 262144])
def test_mixed_filters(gpu, vocab, cap):
    r = np.random.default_rng(vocab)
    rows = 40
    logits = (3 * r.standard_normal((rows, vocab))).astype(np.float32)
    logits[::2, r.integers(0, vocab, 20)] += 15
    both(logits, numbers(r, rows), cap=cap, **mixed(r, rows, vocab))


@pytest.mark.parametrize("only", ["temperature", "top_k", "top_p", "min_p", None])
def test_one_filter_given(gpu, only):
    r = np.random.default_rng(5)
    logits = (4 * r.standard_normal((24, 5000))).astype(np.float32)
    both(logits, numbers(r, 24), **({only: mixed(r, 24, 5000)[only]} if only else {}))


@pytest.mark.parametrize("rows", [1, 3, 300])
def test_rows(gpu, rows):
    r = np.random.default_rng(rows)
    logits = (4 * r.standard_normal((rows, 3001))).astype(np.float32)
    both(logits, numbers(r, rows), cap=20.0, **mixed(r, rows, 3001))


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("vocab", [131072, 200003, 262144])
@pytest.mark.parametrize("rows", [1, 4])
def test_few_wide_rows(gpu, rows, vocab, cap):
    """A unit shared by four waves, in blocks of sixteen; every kind of filter, peaked and flat rows, far logits, masks."""
    r = np.random.default_rng(rows + vocab)
    for i in range(6):
        logits = ((0.5, 4.0)[i % 2] * r.standard_normal((rows, vocab))).astype(np.float32)
        logits[:, r.integers(0, vocab, 30)] += 14
        logits[:, r.integers(0, vocab, 5000)] = (-np.inf, np.nan, -3.4e38)[i % 3]
        both(logits, r.random(rows).astype(np.float32), cap=cap, **mixed(r, rows, vocab))
    both(logits, [LAST] * rows, cap=cap)
    both(logits, [0.5] * rows, cap=cap, min_p=[0.01] * rows, temperature=[2.0] * rows)


@pytest.mark.parametrize("vocab", [3000, 262144])
def test_ties(gpu, vocab):
    """Logits on a coarse grid (a quantised head), all alike, or all alike but one: cuts go by the lower id, and more
    tokens share a bin than a list holds."""
    r = np.random.default_rng(1)
    grid = np.round(2 * r.standard_normal((10, vocab))).astype(np.float32)
    grid[8:] = 0.25
    grid[9, vocab // 2] = 12.0
    grid[7] = np.where(r.random(vocab) < 0.5, 0.0, -0.0)
    for k, p in ((5, 1.0), (1500, 1.0), (0, 0.3), (vocab - 1, 0.9), (2900, 0.999)):
        both(grid, numbers(r, 10), top_k=[k] * 10, top_p=[p] * 10, temperature=[0.9] * 10)


def test_crowded_bins(gpu):
    """One far token stretches the bins, so that nearly the whole row shares one: the row is read again."""
    r = np.random.default_rng(2)
    vocab = 50000
    logits = (0.01 * r.standard_normal((12, vocab))).astype(np.float32)
    logits[:, 77] = 25.0
    logits[6:, 78] = -3e4
    for t, k, p in ((4.0, 20000, 1.0), (4.0, 0, 0.6), (4.0, 30000, 0.7), (50.0, 49999, 0.9999)):
        both(logits, numbers(r, 12), temperature=[t] * 12, top_k=[k] * 12, top_p=[p] * 12, min_p=[0.0, 1e-4] * 6)


def odd_rows():
    """Rows of 5000 logits with masks, infinities and NaN."""
    r = np.random.default_rng(3)
    vocab = 5000
    x = (3 * r.standard_normal((12, vocab))).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2] = -np.inf
    x[2, 4999] = -3.4e38
    x[3, ::2] = -np.inf
    x[3, 1::4] = np.nan
    x[4, [7, 900, 4998]] = np.inf
    x[5, 8] = 3.4e38
    x[6] = -3.4028235e38  # a mask of the type's lowest value over everything
    x[7, 100:] = -3.4028235e38
    x[8, 17] = np.inf
    x[8, 18:] = np.nan
    x[9] = 0.0
    return x


@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_masked_and_infinite_logits(gpu, cap):
    x = odd_rows()
    for params in ({}, dict(top_k=[3] * 12), dict(top_p=[0.7] * 12), dict(top_k=[700] * 12, top_p=[0.5] * 12, min_p=[0.1] * 12),
                   dict(temperature=[0.0] * 12)):
        for u in (0.0, 0.4, LAST):
            both(x, np.full(12, u, np.float32), cap=cap, **params)


@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_masked_and_infinite_logits_of_many_rows(gpu, cap):
    """Enough requests for the parameters and the cuts to be found by kernels of their own, many of them on one row of
    logits."""
    r = np.random.default_rng(15)
    n = 1200
    index = r.integers(-1, 13, n).astype(np.int32)
    both(odd_rows(), numbers(r, n), cap=cap, index=index, **mixed(r, n, 5000))
    both(odd_rows(), numbers(r, n), cap=cap, index=index, top_p=r.choice([0.1, 0.9, 1.0], n), temperature=r.choice([0.01, 1, np.inf], n))


def test_ends_of_the_arguments(gpu):
    """Temperatures, filters and numbers at and past the ends of their ranges."""
    r = np.random.default_rng(4)
    nan, inf = np.nan, np.inf
    t = [nan, -1.0, 0.0, inf, 1e30, 1e-6, 1e-38, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 0.5]
    k = [0, 0, 0, 9, 0, 0, 3, -5, 2 ** 31 - 1, -2 ** 31, 1, 1999, 2000, 0, 0, 10]
    p = [1, 1, 1, 0.5, 0.3, 0.9, 0.9, nan, 2.0, 0.0, -1.0, 1.0, LAST, 1e-30, 1.0, -inf]
    m = [0, 0, 0, 0, 1.0, 0, 0, nan, -1, 0, 0, 2.0, 1e-30, 1.0, inf, 0]
    u = np.array([0.3, 0.3, 0.3, 0.9, 0.9, 0.9, 0.9, nan, -1, 2, inf, 0.2, 1.0, 0.9, 0.9, -inf], np.float32)
    logits = (2 * r.standard_normal((16, 2000))).astype(np.float32)
    both(logits, u, temperature=np.array(t, np.float32), top_k=k, top_p=np.array(p, np.float32), min_p=np.array(m, np.float32))


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("t", [np.inf, 3.4e38, 1e-45])
def test_temperatures_at_the_ends_with_masked_tokens(gpu, t, cap):
    """Every filter, rows with -infinity and NaN among the logits, and units that end inside a vocabulary."""
    r = np.random.default_rng(14)
    logits = (4 * r.standard_normal((6, 2500))).astype(np.float32)
    logits[1::2, r.integers(0, 2500, 900)] = -np.inf
    logits[2, ::3] = np.nan
    for params in ({}, {"min_p": [0.5] * 6}, {"min_p": [1.0] * 6}, {"top_k": [40] * 6}, {"top_p": [0.7] * 6}, {"top_k": [900] * 6, "top_p": [0.3] * 6}):
        both(logits, [0.0, 0.2, 0.5, 0.7, 0.9, LAST], cap=cap, temperature=[t] * 6, **params)


def test_largest_vocabulary(gpu):
    r = np.random.default_rng(12)
    vocab = 1 << 22
    logits = np.round(3 * r.standard_normal((3, vocab)), 2).astype(np.float32)
    both(logits, [0.3, 0.7, 0.99], temperature=[1.0, 2.0, 0.5], top_k=[0, 3000000, 5000], top_p=[0.9, 0.99, 1.0], cap=30.0)


def test_many_rows(gpu):
    """Enough blocks for the cuts to be found by a kernel of their own."""
    r = np.random.default_rng(13)
    rows, vocab = 200, 70001
    logits = (3 * r.standard_normal((rows, vocab))).astype(np.float32)
    logits[::2, r.integers(0, vocab, 20)] += 15
    logits[5] = np.nan
    logits[9] = -np.inf
    logits[20:24] = np.round(logits[20:24])
    for cap in (0.0, 30.0):
        both(logits, numbers(r, rows), cap=cap, **mixed(r, rows, vocab))


def test_row_index_and_strides(gpu):
    """Several requests of one row, rows that no request has, an index outside; rows apart, aligned and not."""
    r = np.random.default_rng(6)
    index = [2, 2, 0, -1, 4, 2, 5, 2 ** 31 - 1]
    for vocab, stride in ((1000, 1000), (1001, 1001), (1000, 1024), (997, 1003), (999, 1004)):
        base = dev((3 * r.standard_normal(5 * stride)).astype(np.float32))
        host = base.download()
        logits = np.stack([host[i * stride:i * stride + vocab] for i in range(5)])
        u, params = numbers(r, len(index)), mixed(r, len(index), vocab)
        view = View(base, 0, (5, vocab), (stride, 1), np.float32)
        got = run(logits, u, index=index, d_logits=view, **params)
        check(logits, len(index), params, u, got, 0.0, index)


def test_far_rows(gpu):
    """Rows past 2^31 elements."""
    vocab, n = 1 << 18, (1 << 13) + 2
    r = np.random.default_rng(8)
    x = (3 * r.standard_normal((1, vocab))).astype(np.float32)
    base = g4.DeviceBuffer.empty((n, vocab), np.float32)
    last = View(base, (n - 1) * vocab, (1, vocab), (vocab, 1), np.float32)
    g4._check(g4.lib().g4_memcpy_h2d(last.ptr, np.ascontiguousarray(x).ctypes.data, x.nbytes, None))
    got = run(base, [0.6], index=[n - 1], top_p=[0.9], d_logits=base)
    check(x, 1, dict(temperature=None, top_k=None, top_p=[0.9], min_p=None), [0.6], got, 0.0)


def test_runs_and_replays_are_alike(gpu):
    r = np.random.default_rng(9)
    rows, vocab = 16, 20000
    logits = np.round(8 * r.standard_normal((rows, vocab))).astype(np.float32) / 4
    params = mixed(r, rows, vocab)
    u = numbers(r, rows)
    d = [dev(a) for a in (logits, u)]
    f = {n: dev(a) for n, a in params.items()}
    stream, ws = g4.Stream(), [g4.DeviceBuffer(gs.sample_workspace_bytes(rows, vocab)) for _ in range(2)]
    outs = [[dev(np.zeros(rows, np.int32)), dev(np.zeros(rows, np.float32))] for _ in range(2)]
    call = lambda i, s=None: gs.sample_tokens(*d, *outs[i], ws[i], cap=30.0, stream=s, **f)
    call(0)
    g4.synchronize()
    first = [a.download() for a in outs[0]]
    check(logits, rows, params, u, first, 30.0)
    graph = g4.Graph(stream, lambda: call(1, stream.handle))
    for _ in range(4):
        for a in outs[1]:
            a.fill(0)
        ws[1].fill(0xA5)
        g4.synchronize()
        graph.launch()
        call(0)
        stream.synchronize()
        g4.synchronize()
        for i in range(2):
            for a, w in zip(outs[i], first):
                assert np.array_equal(a.download().view(np.uint8), w.view(np.uint8))
    graph.close()
