"""Pages that come and go: absent entries among released ones, and windows that move between plans."""
import numpy as np
import pytest

import g4serve as gs
import g4w8a8 as g4
from servecases import View, dev

pytestmark = pytest.mark.gpu


def release(table, first, last, free, count, num_pages):
    """The list and its count after the release, by the definition."""
    free, count = free.copy(), min(max(count, 0), len(free))
    for row, a, b in zip(table, first, last):
        a = min(max(a, 0), len(row))
        for e in row[a:max(min(b, len(row)), a)]:
            if 0 <= e < num_pages and count < len(free):
                free[count] = e
                count += 1
    return free, count


def check_release(table, first, last, free, count, num_pages, page=16, width=None):
    width = table.shape[1] if width is None else width
    first, last = (np.asarray(x, np.int32) for x in (first, last))
    want, n = release(table[:, :width], first, last, free, count, num_pages)
    d_table, d_free, out = dev(table), dev(free), dev(np.full(1, -5, np.int32))
    view = d_table if width == table.shape[1] else View(d_table, 0, (len(table), width), (table.shape[1], 1), np.int32)
    pages = gs.FreePages(d_free, dev(np.array([count], np.int32)), num_pages, page)
    for _ in range(2):  # the count it reads stays, so a second call does the same
        gs.release_pages(pages, view, dev(first), dev(last), out)
        g4.synchronize()
        assert out.download()[0] == n
        assert np.array_equal(d_free.download(), want)  # what lies behind the new count too
        assert np.array_equal(d_table.download(), table)


@pytest.mark.parametrize("seqs,width,stride", [(1, 1, 1), (1, 3000, 3000), (3, 40, 44), (16, 256, 256), (300, 70, 70), (1000, 9, 12),
                                               (4096, 3, 3), (5, 5000, 5001)])
@pytest.mark.parametrize("absent", [0.0, 0.01, 0.5, 1.0])
def test_absent_entries_stay_away(gpu, seqs, width, stride, absent):
    """Entries that are no page of the pools (-1, and others out of range) are not given back, wherever they stand."""
    r = np.random.default_rng(seqs + width)
    num_pages = seqs * width + 7
    table = r.permutation(num_pages)[:seqs * width].reshape(seqs, width).astype(np.int32)
    table = np.pad(table, ((0, 0), (0, stride - width)), constant_values=3)
    gone = r.random(table.shape) < absent
    table[gone] = r.choice([-1, -2 ** 31, num_pages, 2 ** 31 - 1], int(gone.sum()))
    free = np.full(num_pages + 20, -1, np.int32)
    for first, last in ((np.zeros(seqs), np.full(seqs, 2 ** 31 - 1)),
                        (r.integers(-2, width + 3, seqs), r.integers(-2, width + 3, seqs)),
                        (np.where(np.arange(seqs) == seqs // 2, 0, width), np.full(seqs, width))):
        check_release(table, first, last, free, 13, num_pages, width=width)


def test_a_full_list_drops_pages_not_places(gpu):
    """Room for fewer than are given back: the first pages take it, past absent entries in front of them."""
    r = np.random.default_rng(1)
    table = r.permutation(4000)[:3000].reshape(3, 1000).astype(np.int32)
    table[0, :900] = -1
    for capacity, count in ((500, 100), (500, 499), (500, 500), (500, 9999), (500, -4), (2200, 100)):
        check_release(table, [0, 5, 0], [1000, 900, 1000], np.full(capacity, -1, np.int32), count, 4000)


@pytest.mark.parametrize("seqs,width", [(700, 1500), (1, 1 << 18), (4096, 200)])
def test_many_pages(gpu, seqs, width):
    """More entries than a round of all blocks takes, in long rows and short ones."""
    r = np.random.default_rng(seqs)
    num_pages = 1 << 21
    table = r.permutation(num_pages)[:seqs * width].reshape(seqs, width).astype(np.int32)
    table[r.random(table.shape) < 0.001] = -1
    first = r.integers(0, 3, seqs)
    first[::7] = width  # some give nothing back
    check_release(table, first if seqs > 1 else [2], np.full(seqs, width), np.full(seqs * width, -1, np.int32), 5, num_pages)


def test_rows_of_very_different_lengths(gpu):
    r = np.random.default_rng(2)
    table = r.permutation(1 << 20)[:600 * 1700].reshape(600, 1700).astype(np.int32)
    table[::3, ::5] = -1
    last = np.where(np.arange(600) % 200 == 77, 1700, r.integers(0, 3, 600))
    check_release(table, np.zeros(600), last, np.full(1 << 20, -1, np.int32), 0, 1 << 20)


def test_a_moving_window(gpu):
    """Pages go back from behind a window while requests grow, and the rest when they finish. held counts the entries that
    a row was ever given, whatever went back from its front, so the next page goes behind the last; what went back is
    the program's own count, and the next release begins there. Every page is held once or free once at all times."""
    r = np.random.default_rng(4)
    seqs, page, width, total, window = 5, 8, 40, 60, 40
    free, table = dev(r.permutation(total).astype(np.int32)), dev(np.full((seqs, width), -1, np.int32))
    counts = [dev(np.array([total], np.int32)), dev(np.zeros(1, np.int32))]
    lists = [gs.FreePages(free, c, total, page) for c in counts]
    held = [dev(np.zeros(seqs, np.int32)) for _ in range(2)]
    z = lambda n: dev(np.zeros(n, np.int32))
    q_start, kv_len, served, slots = z(seqs + 1), z(seqs), z(1), z(64)
    lens, gone, now = np.zeros(seqs, np.int32), np.zeros(seqs, np.int32), 0
    content = {}  # what a slot holds: (request's number, position)
    number = list(range(seqs))
    finished = 0
    for step in range(60):
        rows = np.where(lens == 0, r.integers(1, 13, seqs), r.integers(0, 9, seqs)).astype(np.int32)
        rows = np.minimum(rows, page * width - lens)
        h = step % 2
        gs.plan_chunk(lists[now], dev(lens), dev(rows), table, q_start, kv_len, counts[1 - now], served, tokens=64, max_q=16,
                      max_kv=page * width, held=held[h], held_out=held[1 - h], row_slot=slots)
        now = 1 - now
        g4.synchronize()
        start, new, have, t = q_start.download(), kv_len.download(), held[1 - h].download(), table.download()
        at = slots.download()
        assert served.download()[0] == seqs
        for s in range(seqs):
            for i, p in enumerate(range(lens[s], new[s])):
                assert at[start[s] + i] == t[s, p // page] * page + p % page
                content[int(at[start[s] + i])] = (number[s], p)
            # what the window sees of the request, from its earliest row of the next chunk, is still its own
            for p in range(max(0, new[s] - window), new[s]):
                assert content[int(t[s, p // page]) * page + p % page] == (number[s], p), (step, s, p)
        lens = new
        done = (lens > 100) & (r.random(seqs) < 0.3) | (lens > page * width - 20)
        last = np.where(done, have, np.maximum(lens - window, 0) // page).astype(np.int32)
        assert (gone <= last).all() and (have >= -(-lens // page)).all()
        gs.release_pages(lists[now], table, dev(gone), dev(last), counts[1 - now])
        now = 1 - now
        g4.synchronize()
        gone = np.where(done, 0, last).astype(np.int32)
        have = np.where(done, 0, have).astype(np.int32)
        held[1 - h].upload(have)
        left = int(counts[now].download()[0])
        mine = [int(p) for s in range(seqs) for p in t[s, gone[s]:have[s]]]
        assert sorted(mine + [int(p) for p in free.download()[:left]]) == list(range(total)), step
        lens = np.where(done, 0, lens).astype(np.int32)
        for s in np.nonzero(done)[0]:
            number[s] += seqs
            finished += 1
    assert finished > 3


def test_release_replayed(gpu):
    """From a graph, over changing tables and ranges."""
    r = np.random.default_rng(6)
    seqs, width, num_pages = 20, 90, 5000
    d = {n: dev(np.zeros(s, np.int32)) for n, s in (("table", (seqs, width)), ("first", seqs), ("last", seqs), ("out", 1))}
    free = dev(np.full(2000, -1, np.int32))
    count = dev(np.array([40], np.int32))
    pages = gs.FreePages(free, count, num_pages, 8)
    stream = g4.Stream()
    call = lambda s=None: gs.release_pages(pages, d["table"], d["first"], d["last"], d["out"], stream=s)
    call()
    g4.synchronize()
    graph = g4.Graph(stream, lambda: call(stream.handle))
    for i in range(4):
        table = r.permutation(num_pages)[:seqs * width].reshape(seqs, width).astype(np.int32)
        table[r.random(table.shape) < 0.2] = -1
        first, last = (r.integers(0, width, seqs).astype(np.int32) for _ in range(2))
        blank = np.full(2000, -1, np.int32)
        for n, v in (("table", table), ("first", first), ("last", last)):
            d[n].upload(v)
        want, n = release(table, first, last, blank, 40, num_pages)
        for run in (lambda: (graph.launch(), stream.synchronize()), call):
            free.upload(blank)
            d["out"].fill(0)
            g4.synchronize()
            run()
            g4.synchronize()
            assert np.array_equal(free.download(), want) and d["out"].download()[0] == n
    graph.close()
