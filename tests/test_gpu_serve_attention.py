"""Attention of a chunk over the paged cache, against a plain 64-bit form."""
import numpy as np
import pytest

import g4serve as gs
import g4w8a8 as g4
from servecases import Batch, View, attention, dev, to_kind

pytestmark = pytest.mark.gpu


def run(b, q, window=0, scale=None, out=np.float16, in_scale=0.0, fill=0, stream=None):
    heads = q.shape[1]
    o = dev(np.full((b.tokens, heads, b.dim), fill, out))
    gs.attention_chunk(b.pages, b.chunk, dev(q), o, b.workspace(heads, window), scale=scale, window=window,
                       in_scale=in_scale, stream=stream)
    return o.download()


def queries(b, heads):
    return b.rng.standard_normal((b.tokens, heads, b.dim)).astype(np.float16)


def check(b, heads, window=0, out=np.float16):
    if not hasattr(b, "pages"):
        b.upload()
    q = queries(b, heads)
    scale = 1.5 / np.sqrt(b.dim)
    got = run(b, q, window, scale, out).astype(np.float64)
    want, bound = attention(b, q, float(np.float32(scale)), window)
    n = int(b.start[-1])
    tol = to_kind(want, bound, out)
    worst = np.abs(got - want)[:n] - tol[:n]
    assert (worst <= 0).all(), f"off by {np.abs(got - want)[:n].max()} at {np.unravel_index(worst.argmax(), worst.shape)}"


SINGLE = [(1, 1)], [(1, 2)], [(1, 31)], [(1, 33)], [(1, 700)]
RAGGED = [(1, 5), (3, 40), (0, 17), (8, 8), (2, 333), (1, 64), (0, 0), (5, 129)]


@pytest.mark.parametrize("kind", ["i8", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens", SINGLE + (RAGGED,), ids=lambda v: f"{len(v)}x{v[-1][1]}")
def test_small_chunks(gpu, lens, dim, kind):
    check(Batch(lens, 1, dim, 16, kind, seed=dim), 8)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (4, 2), (6, 2), (15, 3), (32, 1), (40, 1), (64, 4), (130, 2)])
@pytest.mark.parametrize("kind", ["i8", "f16"])
def test_head_layouts(gpu, heads, kv_heads, kind):
    check(Batch([(1, 70), (4, 19), (9, 100)], kv_heads, 64, 8, kind, seed=heads), heads)


@pytest.mark.parametrize("lens,heads,kv_heads,dim,kind,window", [
    ([(200, 200)], 8, 1, 256, "i8", 0),
    ([(200, 200)], 8, 1, 256, "f16", 0),
    ([(64, 64), (65, 300), (1, 500), (127, 127)], 4, 2, 128, "f16", 0),
    ([(64, 64), (65, 300), (1, 500), (127, 127)], 4, 2, 128, "i8", 0),
    ([(257, 1000)], 3, 1, 64, "i8", 100),
    ([(257, 1000)], 8, 8, 64, "f16", 0),
    ([(300, 900), (3, 700)], 8, 1, 256, "f16", 512),
    ([(513, 513)], 2, 1, 256, "i8", 37),
    ([(33, 2000)], 16, 2, 128, "f16", 1),
])
def test_prefill_chunks(gpu, lens, heads, kv_heads, dim, kind, window):
    check(Batch(lens, kv_heads, dim, 32, kind, seed=dim + heads), heads, window)


@pytest.mark.parametrize("page", [8, 64, 256, 4096])
@pytest.mark.parametrize("lens", [[(1, 257), (3, 255), (1, 256)], [(70, 300), (90, 91)]], ids=["tokens", "chunks"])
def test_page_sizes(gpu, page, lens):
    check(Batch(lens, 2, 128, page, "i8", seed=page), 8)


@pytest.mark.parametrize("window", [1, 2, 16, 33, 100, 5000])
@pytest.mark.parametrize("lens", [[(1, 200), (4, 90), (8, 8), (1, 33)], [(150, 260)]], ids=["tokens", "chunk"])
def test_windows(gpu, window, lens):
    check(Batch(lens, 1, 128, 16, "f16", seed=window), 8, window)


@pytest.mark.parametrize("kind", ["i8", "f16"])
@pytest.mark.parametrize("lens", [[(1, 4096), (2, 3000)], [(1, 9001)]], ids=["two", "one"])
def test_long_caches(gpu, lens, kind):
    check(Batch(lens, 1, 256, 64, kind, seed=7), 8)


@pytest.mark.parametrize("kind", ["i8", "f16"])
@pytest.mark.parametrize("lens,absent", [
    ([(1, 100), (3, 64), (2, 16)], [(0, 0), (0, 1), (0, 5), (1, 3), (2, 0)]),
    ([(80, 200), (40, 40)], [(0, 0), (0, 1), (0, 2), (0, 11), (1, 0), (1, 1), (1, 2)]),
], ids=["tokens", "chunks"])
def test_absent_pages_and_empty_rows(gpu, lens, absent, kind):
    """Pages let go of hold no keys; a sequence (or a row) with none left gives zeros."""
    b = Batch(lens, 1, 128, 16, kind, seed=4, absent=absent).upload()
    check(b, 8)
    check(b, 8, window=20)


@pytest.mark.parametrize("window", [0, 1, 40, 150])
@pytest.mark.parametrize("dim,kind,kv_heads", [(256, "i8", 2), (256, "f16", 2), (64, "f16", 128), (128, "f16", 128),
                                               (256, "f16", 128)])
def test_blocks_of_more_row_tiles(gpu, dim, kind, kv_heads, window):
    """Row counts around 32, 64 and 128, ends inside pages and key tiles, pages let go of."""
    lens = [(33, 35), (140, 300)] if kv_heads > 2 else [(33, 35), (64, 64), (140, 300), (0, 9), (129, 130), (1, 77)]
    check(Batch(lens, kv_heads, dim, 16, kind, seed=window + dim, absent=[(0, 1), (1, 0), (1, 2)]), kv_heads, window)


@pytest.mark.parametrize("kind", ["i8", "f16"])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("lens", [
    [(5 + i % 4, 20 + 37 * i) for i in range(11)],                    # every sequence has two row tiles or room for them
    [(8 * (i % 3 > 0), 50 + i) for i in range(17)] + [(8, 8)] * 7,
    [(1, 3 + i) for i in range(100)] + [(90, 200)] + [(2, 9), (0, 5)] * 20,  # one long chunk among many short ones
    [(1 + i % 2, 2 + 5 * i) for i in range(70)],
], ids=["eleven", "gaps", "long", "seventy"])
def test_batches(gpu, lens, dim, kind):
    check(Batch(lens, 1, dim, 16, kind, seed=len(lens)), 8)


@pytest.mark.parametrize("window", [0, 4000])
def test_int8_blocks_of_two_row_tiles(gpu, window):
    """Many blocks of 4096 keys or more (by the bounds; most sequences are short), one sequence past the window."""
    lens = [(33, 35), (64, 64), (65, 140), (0, 9), (40, 4200), (1, 77), (33, 300), (50, 90), (60, 61)]
    check(Batch(lens, 32, 256, 16, "i8", seed=window, absent=[(2, 1), (4, 0), (4, 240), (6, 18)], max_kv=4224), 32, window)


def test_int8_masked_scales_in_blocks_of_two_row_tiles(gpu):
    m = 70
    def batch():
        return Batch([(m, m + 30)], 128, 256, 16, "i8", seed=5, max_kv=4100)
    b = batch()
    for p, x in ((m + 28, np.inf), (m + 29, np.nan)):
        page = b.table[0, p // 16]
        b.ks[page, :, p % 16], b.vs[page, :, p % 16] = x, x
    q = queries(b.upload(), 128)
    got = run(b, q, 0, 0.1).astype(np.float64)
    want, bound = attention(batch(), q, float(np.float32(0.1)), 0)
    assert (np.abs(got - want) <= to_kind(want, bound, np.float16))[:m - 2].all()
    assert not np.isfinite(got[m - 1]).any()


@pytest.mark.parametrize("dim,kv_heads", [(256, 1), (64, 128), (256, 128)])
def test_masked_contents_in_blocks_of_more_row_tiles(gpu, dim, kv_heads):
    """NaN and infinities in the last two tokens' V: rows before them untouched, rows that see them not finite."""
    m = 70
    def batch():
        return Batch([(m, m + 30)], kv_heads, dim, 16, "f16", seed=dim)
    b = batch()
    for p, x in ((m + 28, np.inf), (m + 29, np.nan)):
        b.v[b.table[0, p // 16], p % 16, :, ::3] = x
    q = queries(b.upload(), kv_heads)
    got = run(b, q, 0, 0.1).astype(np.float64)
    want, bound = attention(batch(), q, float(np.float32(0.1)), 0)
    assert (np.abs(got - want) <= to_kind(want, bound, np.float16))[:m - 2].all()
    assert not np.isfinite(got[m - 1, :, ::3]).any()
    assert np.isfinite(got[m - 1, :, 1::3]).all()


@pytest.mark.parametrize("kind", ["i8", "f16"])
def test_rows_without_positions(gpu, kind):
    """More rows than positions: the rows in front see nothing and give zeros. Rows behind the last
    sequence and past max_q stay as they were."""
    b = Batch([(5, 2), (4, 0), (6, 30)], 1, 128, 16, kind, seed=6, tail_rows=7, max_q=5).upload()
    q = queries(b, 4)
    got = run(b, q, 0, 0.1, np.float32, fill=-3)
    want, bound = attention(b, q, float(np.float32(0.1)), 0)
    live = [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13]
    assert (got[:9] == want[:9]).all() or (np.abs(got[:9] - want[:9]) <= to_kind(want, bound, np.float32)[:9]).all()
    assert (got[:3] == 0).all() and (got[5:9] == 0).all()
    assert (np.abs(got - want)[live] <= to_kind(want, bound, np.float32)[live]).all()
    assert (got[14:] == -3).all()


@pytest.mark.parametrize("m", [4, 90], ids=["tokens", "chunk"])
@pytest.mark.parametrize("kind", ["i8", "f16"])
def test_masked_contents_do_not_matter(gpu, m, kind):
    """NaN and infinities in the chunk's last two tokens: the rows before them are untouched, the rows that
    see them are not finite."""
    b = Batch([(m, m + 30)], 1, 128, 16, kind, seed=m)
    for p, x in ((m + 28, np.inf), (m + 29, np.nan)):
        page = b.table[0, p // 16]
        if kind == "f16":
            b.k[page, p % 16], b.v[page, p % 16, :, ::3] = x, x
        else:
            b.ks[page, :, p % 16], b.vs[page, :, p % 16] = x, x
    b.upload()
    q = queries(b, 8)
    got = run(b, q, 0, 0.1)
    clean = Batch([(m, m + 30)], 1, 128, 16, kind, seed=m)
    want, bound = attention(clean, q, float(np.float32(0.1)), 0)
    assert (np.abs(got.astype(np.float64) - want) <= to_kind(want, bound, np.float16))[:m - 2].all()
    assert not np.isfinite(got[m - 1].astype(np.float32)).any()


@pytest.mark.parametrize("m", [2, 70], ids=["tokens", "chunk"])
def test_scores_of_every_size(gpu, m):
    """Scores spread over +-500 (one key takes all), all equal, and a negative scale."""
    b = Batch([(m, 200)], 1, 256, 16, "f16", seed=1).upload()
    q = queries(b, 8)
    for scale in (8.0, 0.0, -0.2):
        got = run(b, q, 0, scale, np.float32)
        want, bound = attention(b, q, scale, 0)
        assert (np.abs(got - want) <= to_kind(want, bound, np.float32)).all(), scale


@pytest.mark.parametrize("m", [2, 70], ids=["tokens", "chunk"])
def test_small_and_large_row_scales(gpu, m):
    """int8 rows whose scales differ by many orders: a tiny row next to a large one, V past the f16 range."""
    b = Batch([(m, 150)], 1, 128, 16, "i8", seed=8)
    b.vs *= np.float32(10) ** b.rng.integers(-12, 8, b.vs.shape).astype(np.float32)
    b.upload()
    q = queries(b, 8)
    got = run(b, q, 0, 0.1, np.float32)
    want, bound = attention(b, q, float(np.float32(0.1)), 0)
    assert (np.abs(got - want) <= to_kind(want, bound, np.float32)).all()


@pytest.mark.parametrize("m", [3, 66], ids=["tokens", "chunk"])
def test_codes_out(gpu, m):
    """int8 codes on the consumer's scale: the code of the f32 result, or its neighbour where that lies
    within the bound of a half."""
    b = Batch([(m, 90)], 1, 256, 16, "i8", seed=12).upload()
    q = queries(b, 8)
    s = np.float32(0.01)
    got = run(b, q, 0, 0.1, np.int8, in_scale=float(s)).astype(np.float64)
    want, bound = attention(b, q, float(np.float32(0.1)), 0)
    exact = want / s
    lo, hi = (np.clip(np.rint(exact + e * (bound / s + np.abs(exact) * 2.0 ** -22)), -128, 127) for e in (-1, 1))
    assert ((lo <= got) & (got <= hi)).all()
    f = run(b, q, 0, 0.1, np.float32)
    assert np.array_equal(got, np.clip(np.rint(f / s), -128, 127))


def test_strided_queries_and_pools(gpu):
    b = Batch([(3, 50), (70, 120)], 2, 64, 16, "f16", seed=13)
    # heads before slots, K and V interleaved by page
    n = b.pages_n
    both = np.stack([b.k.transpose(0, 2, 1, 3), b.v.transpose(0, 2, 1, 3)], 1)  # [page][2][head][slot][dim]
    base = dev(np.ascontiguousarray(both))
    ps, hs = 2 * 2 * 16 * 64, 16 * 64
    b.pages = gs.KVPages(*[View(base, i * 2 * hs, (n, 2, 16, 64), (ps, hs, 64, 1), np.float16) for i in (0, 1)],
                         heads_first=True)
    b.describe()
    q = queries(b, 6)
    wide = np.zeros((b.tokens, 10 * 64), np.float16)
    wide[:, 64:64 * 7] = q.reshape(b.tokens, -1)
    base_q = dev(wide)
    o = dev(np.zeros((b.tokens, 6, 64), np.float16))
    gs.attention_chunk(b.pages, b.chunk, View(base_q, 64, (b.tokens, 6, 64), (640, 64, 1), np.float16), o,
                       b.workspace(6, 0), scale=0.2)
    want, bound = attention(b, q, float(np.float32(0.2)), 0)
    assert (np.abs(o.download().astype(np.float64) - want) <= to_kind(want, bound, np.float16)).all()


@pytest.mark.parametrize("lens", [[(4, 600), (2, 90)], [(130, 400)]], ids=["tokens", "chunk"])
def test_same_bits_captured_and_replayed(gpu, lens):
    """A captured call replays to the eager bits, with new lengths written between replays, and beside
    another graph with its own workspace."""
    st, other = g4.Stream(), g4.Stream()
    b = Batch(lens, 1, 256, 16, "i8", seed=21).upload()
    q = dev(queries(b, 8))
    outs = [dev(np.zeros((b.tokens, 8, 256), np.float16)) for _ in range(2)]
    wss = [b.workspace(8, 0) for _ in range(2)]
    call = lambda i, h: gs.attention_chunk(b.pages, b.chunk, q, outs[i], wss[i], scale=0.1, stream=h)
    graphs = [g4.Graph(s, lambda i=i, s=s: call(i, s.handle)) for i, s in enumerate((st, other))]
    kv_len = b.chunk.buffers[1]
    full = np.array([kv for _, kv in lens], np.int32)
    for step in range(4):
        kv_len.upload((full - 3 * step).astype(np.int32))
        g4.synchronize()
        eager = dev(np.zeros((b.tokens, 8, 256), np.float16))
        gs.attention_chunk(b.pages, b.chunk, q, eager, b.workspace(8, 0), scale=0.1)
        g4.synchronize()
        for i in range(2):
            outs[i].fill(0)
        g4.synchronize()
        for g in graphs:
            g.launch()
        for s in (st, other):
            s.synchronize()
        for i in range(2):
            assert np.array_equal(outs[i].download().view(np.uint16), eager.download().view(np.uint16))
    for g in graphs:
        g.close()


def test_same_call_twice_same_bits(gpu):
    lens = [(4, 300), (4, 77), (4, 511)]
    b = Batch(lens, 1, 128, 16, "f16", seed=30).upload()
    q = queries(b, 8)
    first, second = run(b, q, 0, 0.1), run(b, q, 0, 0.1)
    assert np.array_equal(first.view(np.uint16), second.view(np.uint16))
