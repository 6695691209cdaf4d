"""The serving operators at the ends of what their arguments may be."""
import numpy as np
import pytest

import g4serve as gs
import test_gpu_serve_verify as verifycase
from servecases import Batch, attention, dev, to_kind

pytestmark = pytest.mark.gpu


def run(b, q, window=0, scale=0.1, out=np.float32):
    o = dev(np.full(q.shape, -3, out))
    gs.attention_chunk(b.pages, b.chunk, dev(q), o, b.workspace(q.shape[1], window), scale=scale, window=window)
    return o.download()


def queries(b, heads):
    return b.rng.standard_normal((b.tokens, heads, b.dim)).astype(np.float16)


@pytest.mark.parametrize("kind", ["i8", "f16"])
@pytest.mark.parametrize("window", [30, 31, 1 << 30, (1 << 31) - 40, (1 << 31) - 1])
def test_windows_of_any_size_and_rows_without_positions(gpu, kind, window):
    """A window that hides nothing is none, also where rows stand at negative positions: sequences with more
    rows than positions, alone in their tile and beside rows that have some."""
    b = Batch([(8, 0), (5, 2), (40, 3), (6, 30), (1, 1)], 1, 128, 16, kind, seed=6).upload()
    q = queries(b, 4)
    got = run(b, q, window)
    want, bound = attention(b, q, float(np.float32(0.1)), window)
    assert (np.abs(got - want) <= to_kind(want, bound, np.float32)).all()
    assert (got[:11] == 0).all()
    assert np.array_equal(got.view(np.uint32), run(b, q, 0).view(np.uint32))


def on_a_grid(c, step, most):
    """The case's logits on multiples of `step`, under `most` in magnitude: two that differ do so by far more than the
    smallest temperatures, ties are exact."""
    snap = lambda x: (np.clip(np.rint(x / step), -most // step, most // step) * step).astype(np.float32)
    return (snap(c[0]), snap(c[1]), *c[2:])


@pytest.mark.parametrize("t", [1e-3, 1e-6, 1e-9, 1e-12, 1e-13, 1e-16, 1e-30, 1e-40])
@pytest.mark.parametrize("cap,most", [(30.0, 12), (30.0, 60), (2.0, 0.75), (2.0, 5), (0.0, 60)])
def test_small_temperatures(gpu, cap, most, t):
    """All weight on the row's maximum, shared evenly where several logits have it, below half the cap and past it."""
    for seed in (1, 2):
        c = on_a_grid(verifycase.case([4, 1, 0, 7, 2], 3001, seed, spread=most / 3), most / 64, most)
        verifycase.check(c, 7, cap, t)


@pytest.mark.parametrize("shift", [0.0, 2000.0])
@pytest.mark.parametrize("cap", [1e-30, 1e-3, 100.0, 1e4, 1e9, 1e16, 1e30, 3e38])
def test_caps_of_every_size(gpu, cap, shift):
    """A cap far above the logits changes nothing, one far below them leaves them nearly alike."""
    c = verifycase.case([4, 1, 0, 7, 2], 9001, 3)
    c = (*(x + np.float32(shift) for x in c[:2]), *c[2:])
    got = verifycase.check(c, 7, cap, 0.9)
    if cap >= 1e16:
        plain = verifycase.check(c, 7, 0.0, 0.9)
        assert np.array_equal(got[0], plain[0]) and np.array_equal(got[1], plain[1])


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("t", [0.0, 0.9])
@pytest.mark.parametrize("cap", [0.0, 2.0, 30.0])
def test_masked_tokens_have_no_weight(gpu, cap, t, drafter):
    """-infinity is out of the draw whatever the cap, as NaN is; a drafted one is refused, a row of them is empty."""
    logits, dl, drafts, start, u, un = verifycase.case([4, 1, 0, 7, 2], 3001, 4, spread=0.3)
    logits[:, 7::2] = dl[:, 7::2] = np.nan
    logits[5, :2000] = np.nan
    drafts[0], drafts[5] = 8, 9  # sequence 3 drafted a token that is out
    dl[4] = np.nan
    logits[7] = np.nan  # sequence 2
    with np.errstate(invalid="ignore"):
        want = verifycase.verify(logits, dl if drafter else None, drafts, start, u, un, 7, cap, t)
    assert t == 0 or want[3] > 2.0 ** -32
    masked = lambda x: np.where(np.isnan(x), np.float32(-np.inf), x)
    got = verifycase.run(masked(logits), masked(dl) if drafter else None, drafts, start, u, un, 7, cap, t)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    assert (np.abs(got[2] - want[2]) <= np.abs(want[2]) * 2.0 ** -24 * 1.01 + 2.0 ** -36).all()
    assert got[1][3] == 0 and got[0][2, 0] == -1


def softcap_argmax(g4, logits, cap):
    rows, vocab = logits.shape
    ws = g4.DeviceBuffer(g4.lib().g4_argmax_workspace_bytes(rows, vocab))
    tok, capped = dev(np.zeros(rows, np.int32)), dev(np.zeros_like(logits))
    g4._check(g4.lib().g4_softcap_argmax(dev(logits).ptr, rows, vocab, cap, capped.ptr, ws.ptr, ws.nbytes, tok.ptr, None))
    return tok.download(), capped.download()


@pytest.mark.parametrize("cap", [2.0, 30.0])
def test_greedy_takes_the_first_maximum_of_the_logits(gpu, cap):
    """Under a cap too, and g4_softcap_argmax's token but where capping makes an earlier logit equal to it."""
    r = np.random.default_rng(int(cap))
    rows, vocab = 12, 9001
    logits = r.standard_normal((rows, vocab)).astype(np.float32)
    at, before = r.integers(4500, vocab, rows), r.integers(0, 4500, rows)
    n = np.arange(rows)
    logits[n, at] = 6
    for i in range(rows):  # one step, some steps, far past the cap, equal
        logits[i, before[i]] = [np.nextafter(np.float32(6), np.float32(0)), 6 - 2.0 ** -6, 20 * cap, 6][i % 4]
        logits[i, at[i]] = [6, 6, 30 * cap, 6][i % 4]
    z = np.zeros(0, np.int32)
    got = verifycase.run(logits, None, z, np.zeros(rows + 1, np.int32), z, z, 0, cap, 0.0)[0][:, 0]
    assert np.array_equal(got, logits.argmax(1))
    tokens, capped = softcap_argmax(gpu, logits, cap)
    same = got == tokens
    assert same[1::4].all() and same[3::4].all()
    assert not same[2::4].any()
    assert (capped[n, got] == capped[n, tokens])[~same].all() and (tokens < got)[~same].all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", ["i8", "f16"])
@pytest.mark.parametrize("lens,absent,window", [
    ([(4, 40), (3, 1), (2, 33)], [(0, 0), (0, 1), (0, 2), (2, 1)], 0),  # none left; two rows without a position; some left
    ([(70, 100), (5, 300)], [(0, 5), (0, 6), (1, 18)], 5),  # rows of a tile whose window's pages are gone
], ids=["tokens", "chunk"])
def test_queries_that_are_not_finite(gpu, lens, absent, window, kind, bad):
    """A row whose query has a NaN or an infinity is not finite where it sees a key, and zeros where it sees none; the
    rows beside it are as without it."""
    b = Batch(lens, 1, 128, 16, kind, seed=len(lens), absent=absent).upload()
    q = queries(b, 4)
    want, bound = attention(b, q, float(np.float32(0.1)), window)
    odd = q.copy()
    odd[::2, 1::2, 5] = bad
    odd[::2, 3, 6] = -bad
    got = run(b, odd, window)
    hit = np.zeros((b.tokens, 4), bool)
    hit[::2, 1::2] = True
    seen, none_finite = np.zeros(b.tokens, bool), np.zeros((b.tokens, 4), bool)
    for s, (m, kv) in enumerate(lens):
        k, there = b.held(b.k, b.ks, s)
        for i in range(m):
            t, pos = b.start[s] + i, kv - m + i
            j = np.arange(kv)
            see = there & (j <= pos) & (j > (pos - window if window else -1))
            seen[t] = see.any()
            with np.errstate(invalid="ignore"):
                score = odd[t].astype(np.float64) @ k[see, 0].T
            # int8 keys: any; f16: a score that is NaN or +infinity (one of -infinity has no weight)
            none_finite[t] = hit[t] & seen[t] if kind == "i8" else (np.isnan(score) | (score == np.inf)).any(1)
    assert 0 < seen.sum() < b.tokens and none_finite.any()
    assert (got[~seen] == 0).all()
    assert not np.isfinite(got[none_finite]).any()
    assert (np.abs(got - want) <= to_kind(want, bound, np.float32))[~hit].all()


@pytest.mark.parametrize("dim,heads,kv", [(64, 8, 300001), (256, 2, 150001)])
def test_long_sums_of_int8_rows(gpu, dim, heads, kv):
    """Equal weights and V scales of 1 to 1/8: sums of codes times powers of two, which f32 holds exactly as long as no
    partial sum passes 2^24 eighths. So a row is off by the last division and product alone, however many keys it has
    (enough rows that the keys of one are not split over blocks)."""
    m, page = 16384 // heads, 4096
    r = np.random.default_rng(dim)
    pages = -(-kv // page)
    k, v = (r.integers(-127, 128, (pages, page, 1, dim)).astype(np.int8) for _ in range(2))
    vs = (2.0 ** -r.integers(0, 4, (pages, 1, page))).astype(np.float32)
    ks = np.full((pages, 1, page), 0.01, np.float32)
    p = gs.KVPages(dev(k), dev(v), dev(ks), dev(vs))
    c = gs.Chunk(dev(np.array([0, m], np.int32)), dev(np.array([kv], np.int32)), dev(np.arange(pages, dtype=np.int32)[None]), m, m, kv)
    q = r.standard_normal((m, heads, dim)).astype(np.float16)
    o = dev(np.zeros(q.shape, np.float32))
    ws = gpu.DeviceBuffer(gs.attention_chunk_workspace_bytes(p, c, heads))
    gs.attention_chunk(p, c, dev(q), o, ws, scale=0.0)
    sums = np.cumsum((v.astype(np.float64) * vs.transpose(0, 2, 1)[..., None]).reshape(-1, dim)[:kv], 0)[kv - m:]
    assert np.abs(sums).max() * 8 < 2 ** 24
    want = (sums / np.arange(kv - m + 1, kv + 1)[:, None])[:, None]
    assert (np.abs(o.download() - want) <= 4 * 2.0 ** -24 * np.abs(want)).all()


def scaled_attention(b, q, scale, window, rows=slice(None)):
    """attention() of servecases with a bound for V scales of very different sizes, over what a row sees alone. A weight
    is rounded to f16 with V's scale in it, relative to a power of two of at most 4 times the largest product of the
    two that the row sees: by 2^-11 of itself, or below 2^-14 of that power by up to 2^-25 of it; times a code of at most 127."""
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    for s, (m, kv) in enumerate(b.lens):
        k, there = b.held(b.k, b.ks, s)
        v, _ = b.held(b.v, b.vs, s)
        j = np.arange(kv)
        page = np.where(there, b.table[s, j // b.page], 0)
        for i in range(m):
            pos, t = kv - m + i, b.start[s] + i
            see = there & (j <= pos) & (j > (pos - window if window else -1))
            if not see.any():
                continue
            for h in range(q.shape[1]):
                g = h // (q.shape[1] // b.kv_heads)
                kk, vv, qq = k[see, g], v[see, g], q[t, h].astype(np.float64)
                vs = np.abs(b.vs[page[see], g, j[see] % b.page].astype(np.float64))
                sc = kk @ qq * scale
                p = np.exp(sc - sc.max())
                p /= p.sum()
                n = see.sum()
                ds = ((np.abs(kk) @ np.abs(qq)).max() * abs(scale) * (b.dim + 4) + 16) * 2.0 ** -24 + \
                    np.abs(qq).max() / 65024 * np.abs(kk).sum(1).max() * abs(scale)
                want[t, h] = p @ vv
                bound[t, h] = p @ np.abs(vv) * (4 * ds + 2.0 ** -11 + 2 * (n + 8) * 2.0 ** -24) + \
                    n * 2.0 ** -25 * 4 * 127 * (p * vs).max()
    return want, bound


def scales_of_all_sizes(b, seed):
    r = np.random.default_rng(seed)
    b.vs *= np.float32(10) ** r.integers(-14, 10, b.vs.shape).astype(np.float32)
    b.vs[r.random(b.vs.shape) < 0.1] = 0
    return b


@pytest.mark.parametrize("lens,heads,kv_heads,dim,window,max_kv", [
    ([(3, 150), (1, 400), (2, 33)], 4, 1, 128, 0, None),
    ([(70, 150)], 4, 1, 256, 0, None),
    ([(70, 150), (5, 90)], 4, 1, 64, 40, None),
    ([(70, 150)], 128, 128, 256, 0, 4100),  # blocks of two row tiles
])
def test_int8_scales_of_all_sizes(gpu, lens, heads, kv_heads, dim, window, max_kv):
    """Each row to its own precision: scales that it does not see change nothing, and those of keys that weigh nothing
    do not take it from the ones that do. Scores over +-20 make most keys weigh nothing."""
    for seed in (1, 2, 3):
        b = scales_of_all_sizes(Batch(lens, kv_heads, dim, 16, "i8", seed=seed, max_kv=max_kv), seed)
        # the last positions' scales are out of the range of f16 a million times: only the last rows see them
        for s, (m, kv) in enumerate(lens):
            for p in range(kv - min(m, 3) + 1, kv):
                b.vs[b.table[s, p // 16], :, p % 16] = 1e25
        b.upload()
        q = queries(b, heads)
        want, bound = scaled_attention(b, q, float(np.float32(0.6)), window)
        got = run(b, q, window, 0.6)
        assert (np.abs(got - want) <= to_kind(want, bound, np.float32)).all()


@pytest.mark.parametrize("first,big,later", [(100, 101, None), (100, 20, None), (20, 100, None), (90, 10, 170)])
def test_a_large_scale_that_weighs_nothing(gpu, first, big, later):
    """The key that takes all the weight has a V scale of about 1e-5, a key of weight e^-32 one of 1e5, in its key tile,
    before it or behind it; or the large one led until a later key outweighs it."""
    b = Batch([(2, 200)], 1, 64, 16, "i8", seed=9)
    k = np.zeros((200, 64), np.float32)
    k[:, 0], k[:, 1] = -2, 4
    k[first, 0] = 2
    if later is not None:
        k[big, 0], k[later, 0] = 0, 4
    for p in range(200):
        page, slot = b.table[0, p // 16], p % 16
        amax = np.abs(k[p]).max()
        b.k[page, slot, 0] = np.rint(127 * k[p] / amax)
        b.ks[page, 0, slot] = amax / 127
        b.vs[page, 0, slot] = 1e5 if p == big else 1e-5
    b.upload()
    q = np.zeros((2, 1, 64), np.float16)
    q[..., 0] = 8
    want, bound = scaled_attention(b, q, 1.0, 0)
    got = run(b, q, 0, 1.0)
    assert (np.abs(got - want) <= to_kind(want, bound, np.float32)).all()
    assert np.abs(want).max() > 20 * bound.max()


@pytest.mark.parametrize("kind", ["i8", "f16"])
@pytest.mark.parametrize("lens,window,dim", [([(115, 33), (31, 36), (1, 90)], 33, 128), ([(70, 200)], 0, 256), ([(5, 40), (33, 60)], 0, 64)])
def test_small_outputs_beside_a_large_weight(gpu, lens, window, dim, kind):
    """Sharp rows: where the key that takes nearly all the weight has a small element of V, that element of the output is
    made by keys of weight 1e-4 and less, and is right to its own size."""
    for seed in (1, 2):
        b = Batch(lens, 3, dim, 64, kind, seed=seed, absent=[(1, 0)] if len(lens) > 2 else ()).upload()
        q = queries(b, 24)
        got = run(b, q, window, 0.5)
        want, bound = attention(b, q, 0.5, window)
        assert (np.abs(got - want) <= to_kind(want, bound, np.float32)).all()
