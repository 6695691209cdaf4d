"""The paged cache: the chunk prologue's norm, RoPE and quantising store, and the read-back, against
plain 64-bit forms."""
import ctypes

import numpy as np
import pytest

import g4decode as gd
import g4serve as gs
from servecases import Batch, View, dev, quantise

pytestmark = pytest.mark.gpu

EPS = 1e-6


def rows(r, kind, shape):
    x = r.standard_normal(shape)
    if kind == np.int8:
        return np.clip(np.rint(30 * x), -128, 127).astype(np.int8)
    return x.astype(kind)


def norm_rope(x, gain, cos, sin, norm=True):
    """64 bits; x [tokens][heads][dim], cos / sin [tokens][dim / 2] or None."""
    y = x.astype(np.float64)
    if norm:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float32(EPS))
        if gain is not None:
            y = y * gain
    if cos is not None:
        h = y.shape[-1] // 2
        c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
        y = np.concatenate([y[..., :h] * c - y[..., h:] * s, y[..., h:] * c + y[..., :h] * s], -1)
    return y


def positions(b):
    return np.concatenate([kv - m + np.arange(m) for m, kv in b.lens]) if b.lens else np.zeros(0, int)


# f32 arithmetic before a rounding: squares, their sum over 256, a root, a divide, two products and the
# rotation's: under (256 / 64 + 8 levels + 12) steps of 2^-24 of the row's largest term
F32_REL = 32 * 2.0 ** -24


@pytest.mark.parametrize("lens,heads,kv_heads,dim,page,kind,x", [
    ([(1, 1)], 8, 1, 256, 16, "i8", np.int8),
    ([(1, 4096)], 8, 1, 256, 16, "i8", np.int8),
    ([(5, 37), (1, 16), (17, 17), (3, 100)], 8, 1, 256, 16, "i8", np.int8),
    ([(5, 37), (0, 9), (33, 64)], 6, 2, 128, 8, "i8", np.float32),
    ([(70, 70), (2, 300)], 4, 4, 64, 32, "f16", np.float16),
    ([(9, 40), (0, 0), (1, 1)], 8, 8, 128, 1024, "f16", np.float32),
    ([(1, 2 + i) for i in range(130)], 2, 1, 64, 8, "i8", np.float16),
])
def test_prologue_norm_rope_store(gpu, lens, heads, kv_heads, dim, page, kind, x):
    b = Batch(lens, kv_heads, dim, page, kind, seed=len(lens)).upload()
    r = b.rng
    t = b.tokens
    q, k, v = (rows(r, x, (t, n, dim)) for n in (heads, kv_heads, kv_heads))
    sc = [0.1, 0.05, 0.2] if x == np.int8 else [1.0] * 3
    qg, kg = (r.uniform(0.5, 1.5, dim).astype(np.float32) for _ in range(2))
    cos, sin = gd.rope_tables(b.max_kv, dim, 1e4, 1.0)
    q_out = dev(np.full((t, heads, dim), 7, np.float16))
    gs.paged_prologue(b.pages, b.chunk, dev(q), dev(k), dev(v), q_out, dev(qg), dev(kg), dev(cos), dev(sin), EPS,
                      q_scale=sc[0], k_scale=sc[1], v_scale=sc[2])
    pos = positions(b)
    qd, kd, vd = (a.astype(np.float64) * np.float32(s) for a, s in zip((q, k, v), sc))
    want = norm_rope(qd, qg, cos[pos], sin[pos])
    tol = np.abs(want) * 2.0 ** -11 + F32_REL * np.abs(want).max(-1, keepdims=True) + 2.0 ** -25
    assert (np.abs(q_out.download().astype(np.float64) - want) <= tol).all()
    ko, vo = (dev(np.zeros((t, kv_heads, dim), np.float32)) for _ in range(2))
    gs.kv_read(b.pages, b.chunk, ko, vo)
    for got, y in ((ko, norm_rope(kd, kg, cos[pos], sin[pos])), (vo, norm_rope(vd, None, None, None))):
        amax = np.abs(y).max(-1, keepdims=True)
        if kind == "i8":  # half a code, and the f32 arithmetic in front of it and in the scale
            tol = amax / 127 * 0.5 + 3 * F32_REL * amax
        else:
            tol = np.abs(y) * 2.0 ** -11 + F32_REL * amax + 2.0 ** -25
        assert (np.abs(got.download() - y) <= tol).all()


@pytest.mark.parametrize("kind", ["i8", "f16"])
def test_untouched_slots_stay(gpu, kind):
    """Only the chunk's own positions change: not the sequences' others, nor pages of no sequence."""
    b = Batch([(3, 20), (5, 5)], 2, 128, 8, kind, seed=3).upload()
    k, v = (b.rng.standard_normal((8, 2, 128)).astype(np.float32) for _ in range(2))
    gs.paged_prologue(b.pages, b.chunk, None, dev(k), dev(v), None)
    wk, wv = b.k.copy(), b.v.copy()
    ks, vs = (None, None) if b.ks is None else (b.ks.copy(), b.vs.copy())
    t = 0
    for s, (m, kv) in enumerate(b.lens):
        for p in range(kv - m, kv):
            page, slot = b.table[s, p // 8], p % 8
            for pool, scales, x in ((wk, ks, k), (wv, vs, v)):
                if kind == "i8":
                    pool[page, slot], scales[page, :, slot] = quantise(x[t])
                else:
                    pool[page, slot] = x[t].astype(np.float16)
            t += 1
    assert np.array_equal(b.dk.download().view(np.uint8), wk.view(np.uint8))
    assert np.array_equal(b.dv.download().view(np.uint8), wv.view(np.uint8))
    if kind == "i8":
        assert np.array_equal(b.dks.download().view(np.uint32), ks.view(np.uint32))
        assert np.array_equal(b.dvs.download().view(np.uint32), vs.view(np.uint32))


def test_codes_are_the_definitions(gpu):
    """Raw f32 rows: every code is RNE(127 y / amax) exactly, also where the quotient lies next to or on
    a half, and for rows of the smallest and largest magnitudes; zero and non-finite rows."""
    r = np.random.default_rng(11)
    n, dim = 600, 256
    x = r.standard_normal((n, 1, dim)).astype(np.float32)
    x[0] = 0
    # on the half (amax / 2 = 63.5 codes) and one step to either side of quotients near halves
    half = (2 * r.integers(-127, 127, (200, 1, dim)) + 1) / 254.0
    top = r.uniform(1, 100, (200, 1, 1)).astype(np.float32)
    h = (half * top).astype(np.float32)
    h = np.where(r.random(h.shape) < 0.5, np.nextafter(h, np.float32(np.inf)), h)
    x[100:300] = h
    x[100:300, :, :1] = top
    x[100:300, :, 1:2] = top / 2
    x[300:320] *= np.float32(1e-40)  # subnormal
    x[320:340] *= np.float32(3e38) / np.abs(x[320:340]).max()
    x[340:360] *= np.float32(1e-37)
    x[1, 0, 3], x[2, 0, 5], x[3, 0, 255] = np.nan, np.inf, -np.inf
    b = Batch([(n, n)], 1, dim, 16, "i8").upload()
    gs.paged_prologue(b.pages, b.chunk, None, dev(x), dev(-x), None)
    codes, scale = quantise(np.where(np.isfinite(x), x, 0))
    p = np.arange(n)
    page = b.table[0, p // 16]
    for pool, scales, sign in ((b.dk, b.dks, 1), (b.dv, b.dvs, -1)):
        got, gsc = pool.download()[page, p % 16], scales.download()[page, :, p % 16]
        assert np.array_equal(got[4:], sign * codes[4:])
        assert np.array_equal(gsc[4:], scale[4:])
        assert (got[0] == 0).all() and gsc[0, 0] == 0
        assert (got[1:4] == 0).all() and np.isnan(gsc[1:4]).all()


def test_strided_rows_and_pools(gpu):
    """q, k, v as parts of one projection's rows; pools inside a larger tensor, heads before slots."""
    kv_heads, heads, dim, page, pages_n = 2, 4, 64, 8, 5
    r = np.random.default_rng(5)
    t = 19
    width = (heads + 2 * kv_heads) * dim + 32
    qkv = dev(r.standard_normal((t, width)).astype(np.float16))
    host = qkv.download()
    part = [host[:, a * dim:(a + n) * dim].reshape(t, n, dim) for a, n in ((0, heads), (heads, kv_heads), (heads + kv_heads, kv_heads))]
    parts = [View(qkv, a * dim, (t, n, dim), (width, dim, 1), np.float16)
             for a, n in ((0, heads), (heads, kv_heads), (heads + kv_heads, kv_heads))]
    # [page][K or V][head][slot + 1 unused][dim]
    base = dev(np.full((pages_n, 2, kv_heads, page + 1, dim), 9, np.float16))
    ps, hs = 2 * kv_heads * (page + 1) * dim, (page + 1) * dim
    pools = [View(base, i * kv_heads * hs, (pages_n, kv_heads, page, dim), (ps, hs, dim, 1), np.float16) for i in (0, 1)]
    pages = gs.KVPages(*pools, heads_first=True)
    table = np.array([[3, 0, 4]], np.int32)
    chunk = gs.Chunk(dev(np.array([0, t], np.int32)), dev(np.array([t + 2], np.int32)), dev(table), t, t, t + 2)
    q_out = dev(np.zeros((t, heads, dim), np.float16))
    gs.paged_prologue(pages, chunk, *parts, q_out)
    assert np.array_equal(q_out.download(), part[0])
    got = base.download()
    want = np.full_like(got, 9)
    for i in range(t):
        p = i + 2
        want[table[0, p // page], 0, :, p % page] = part[1][i]
        want[table[0, p // page], 1, :, p % page] = part[2][i]
    assert np.array_equal(got, want)
    for dt in (np.float16, np.float32):
        k_out, v_out = (dev(np.zeros((t, kv_heads, dim), dt)) for _ in range(2))
        gs.kv_read(pages, chunk, k_out, v_out)
        assert np.array_equal(k_out.download(), part[1].astype(dt)) and np.array_equal(v_out.download(), part[2].astype(dt))


@pytest.mark.parametrize("kind", ["i8", "f16"])
@pytest.mark.parametrize("out", [np.float32, np.float16])
def test_read_whole_sequences(gpu, kind, out):
    """Whole sequences to a padded cache: rows past a sequence's end stay, absent pages read as zeros, one
    of the two outputs may be left out."""
    lens = [(n, n) for n in (1, 40, 0, 16, 131)]
    b = Batch(lens, 2, 128, 16, kind, seed=9, absent=[(1, 1), (4, 0)]).upload()
    cap = 140
    ko, vo = (dev(np.full((len(lens), cap, 2, 128), 5, out)) for _ in range(2))
    gs.kv_read(b.pages, b.chunk, ko, vo)
    for got, pool, scales in ((ko.download(), b.k, b.ks), (vo.download(), b.v, b.vs)):
        for s, (_, kv) in enumerate(lens):
            x, there = b.held(pool, scales, s)
            # one product, rounded to f32 and then to the output's type
            x32 = np.where(there[:, None, None], x, 0).astype(np.float32)
            assert np.array_equal(got[s, :kv], x32.astype(out))
            assert (got[s, kv:] == 5).all()
    only = dev(np.full((b.tokens, 2, 128), 5, out))
    gs.kv_read(b.pages, b.chunk, None, only)
    assert np.array_equal(only.download(), np.concatenate([vo.download()[s, :kv] for s, (_, kv) in enumerate(lens)]))


def test_rows_outside_the_call(gpu):
    """Rows behind the last sequence, rows past max_q, and rows at negative positions: no store, and the
    first two leave q_out as it was."""
    b = Batch([(4, 9), (6, 6), (3, 1)], 1, 128, 8, "f16", seed=2, tail_rows=5, max_q=5).upload()
    r = b.rng
    q, k = r.standard_normal((b.tokens, 2, 128)).astype(np.float16), r.standard_normal((b.tokens, 1, 128)).astype(np.float16)
    q_out = dev(np.full((b.tokens, 2, 128), 3, np.float16))
    gs.paged_prologue(b.pages, b.chunk, dev(q), dev(k), dev(k), q_out)
    want = q.copy()
    want[9] = 3  # the sixth row of the second sequence
    want[13:] = 3
    assert np.array_equal(q_out.download(), want)
    wk = b.k.copy()
    for row, s, p in [(i, 0, 5 + i) for i in range(4)] + [(4 + i, 1, i) for i in range(5)] + [(12, 2, 0)]:
        wk[b.table[s, p // 8], p % 8] = k[row]
    assert np.array_equal(b.dk.download().view(np.uint16), wk.view(np.uint16))
    ko = dev(np.full((b.tokens, 1, 128), 3, np.float16))
    gs.kv_read(b.pages, b.chunk, ko, None)
    want = k.copy()
    want[[9, 13, 14, 15, 16, 17]] = 3
    want[[10, 11]] = 0  # negative positions hold nothing
    assert np.array_equal(ko.download(), want)


def test_offsets_past_32_bits(gpu):
    """Pages 2^30 elements apart: the third starts 4 GiB in."""
    import g4w8a8 as g4
    apart, dim, page = 1 << 30, 64, 16
    size = 2 * apart + page * dim
    pools = [g4.DeviceBuffer(2 * size, np.float16) for _ in range(2)]
    pages = gs.KVPages(*[View(p, 0, (3, page, 1, dim), (apart, dim, dim, 1), np.float16) for p in pools])
    t = 3 * page
    chunk = gs.Chunk(dev(np.array([0, t], np.int32)), dev(np.array([t], np.int32)),
                     dev(np.array([[2, 0, 1]], np.int32)), t, t, t)
    x = np.random.default_rng(0).standard_normal((t, 1, dim)).astype(np.float16)
    gs.paged_prologue(pages, chunk, None, dev(x), dev(-x), None)
    k, v = (dev(np.zeros_like(x)) for _ in range(2))
    gs.kv_read(pages, chunk, k, v)
    assert np.array_equal(k.download(), x) and np.array_equal(v.download(), -x)
    q = dev(x)
    out = dev(np.zeros((t, 1, dim), np.float32))
    ws = g4.DeviceBuffer(gs.attention_chunk_workspace_bytes(pages, chunk, 1))
    gs.attention_chunk(pages, chunk, q, out, ws, scale=0.0)  # uniform weights: running means of V
    want = np.cumsum(-x.astype(np.float64), 0) / np.arange(1, t + 1)[:, None, None]
    # weights 1 and an f32 sum of up to 48 terms
    assert np.abs(out.download() - want).max() <= 64 * 2.0 ** -24 * np.abs(x).max().astype(np.float64)
