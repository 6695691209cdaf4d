"""The plan of a chunk and the release of pages, against plain loops."""
import numpy as np
import pytest

import g4serve as gs
import g4w8a8 as g4
from servecases import View, dev

pytestmark = pytest.mark.gpu


def plan(cached, rows, held, table, free, count, tokens, max_q, max_kv, page, num_pages, adapter):
    """The outputs by name, by the definition."""
    table = table.copy()
    seqs, width = table.shape
    count = min(max(count, 0), len(free))
    c = [min(max(int(x), 0), max_kv) for x in cached]
    n = [min(max(int(x), 0), max_q, max_kv - k) for x, k in zip(rows, c)]
    h = [-(-k // page) for k in c] if held is None else [min(max(int(x), 0), width) for x in held]
    need = [max(0, -(-(k + m) // page) - a) if m else 0 for k, m, a in zip(c, n, h)]
    served = used = filled = 0
    while served < seqs and filled + n[served] <= tokens and used + need[served] <= count:
        filled, used, served = filled + n[served], used + need[served], served + 1
    left = at = count - used
    out = {"q_start": [0], "kv_len": [], "held_out": [], "last_row": [], "row_pos": [], "row_slot": [], "row_adapter": []}
    for s in range(seqs):
        m, w = (n[s], need[s]) if s < served else (0, 0)
        table[s, h[s]:h[s] + w] = free[at:at + w]
        at += w
        for p in range(c[s], c[s] + m):
            e = int(table[s, p // page])
            out["row_pos"].append(p)
            out["row_slot"].append(e * page + p % page if 0 <= e < num_pages else -1)
            out["row_adapter"].append(-1 if adapter is None else adapter[s])
        out["q_start"].append(out["q_start"][-1] + m)
        out["kv_len"].append(c[s] + m)
        out["held_out"].append(h[s] + w)
        out["last_row"].append(out["q_start"][-1] - 1 if m else -1)
    for name, v in (("row_pos", -1), ("row_slot", -1), ("row_adapter", -2)):
        out[name] += [v] * (tokens - len(out[name]))
    return {**{k: np.array(v, np.int32) for k, v in out.items()}, "free_left": np.array([left], np.int32),
            "served": np.array([served], np.int32), "table": table}


class Case:
    def __init__(self, cached, rows, page=8, held=None, adapter=None, spare=5, tokens=None, max_q=None, max_kv=None, width=None,
                 short=0, num_pages=None, seed=0, stride=None):
        r = np.random.default_rng(seed)
        self.cached, self.rows = np.array(cached, np.int32), np.array(rows, np.int32)
        self.page, seqs = page, len(cached)
        top = max(int(max(0, c)) + int(max(0, n)) for c, n in zip(cached, rows))
        self.max_kv = max(1, top) if max_kv is None else max_kv
        self.width = -(-self.max_kv // page) if width is None else width
        have = [min(self.width, -(-max(0, int(c)) // page)) for c in cached] if held is None else held
        total = seqs * self.width + spare
        self.num_pages = total if num_pages is None else num_pages
        ids = r.permutation(total).astype(np.int32)
        self.table = np.full((seqs, stride or self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(have):
            n = min(max(n, 0), self.width)
            self.table[s, :n] = ids[at:at + n]
            at += n
        self.free = np.concatenate([ids[at:], np.full(at, -9, np.int32)])
        self.count = total - at - short
        self.held = None if held is None else np.array(held, np.int32)
        self.adapter = None if adapter is None else np.array(adapter, np.int32)
        self.tokens = max(1, int(sum(max(0, n) for n in rows))) if tokens is None else tokens
        self.max_q = max(1, int(max(rows))) if max_q is None else max_q

    def want(self):
        t = self.table[:, :self.width]
        w = plan(self.cached, self.rows, self.held, t, self.free, self.count, self.tokens, self.max_q, self.max_kv, self.page,
                 self.num_pages, self.adapter)
        full = self.table.copy()
        full[:, :self.width] = w["table"]
        return {**w, "table": full}

    def upload(self, optional=True):
        seqs = len(self.cached)
        z = lambda n: dev(np.full(n, 1234567, np.int32))
        self.d = {"q_start": z(seqs + 1), "kv_len": z(seqs), "free_left": z(1), "served": z(1), "table": dev(self.table)}
        if optional:
            self.d.update(held_out=z(seqs), last_row=z(seqs), row_pos=z(self.tokens), row_slot=z(self.tokens),
                          row_adapter=z(self.tokens))
        self.ins = [dev(x) for x in (self.cached, self.rows)]
        self.opt = {n: dev(x) for n, x in (("held", self.held), ("seq_adapter", self.adapter)) if x is not None}
        self.list = gs.FreePages(dev(self.free), dev(np.array([self.count], np.int32)), self.num_pages, self.page)
        return self

    def call(self, stream=None):
        d = dict(self.d)
        table = d.pop("table")
        if self.table.shape[1] != self.width:
            table = View(table, 0, (len(self.cached), self.width), (self.table.shape[1], 1), np.int32)
        names = ("q_start", "kv_len", "free_left", "served")
        gs.plan_chunk(self.list, *self.ins, table, *(d.pop(n) for n in names), tokens=self.tokens, max_q=self.max_q,
                      max_kv=self.max_kv, stream=stream, **d, **self.opt)

    def check(self):
        g4.synchronize()
        want = self.want()
        for n, x in self.d.items():
            assert np.array_equal(x.download(), want[n]), n
        assert np.array_equal(self.list.buffers[0].download(), self.free)  # the list itself is not touched


CASES = {
    "one token": dict(cached=[0], rows=[1]),
    "page ends inside": dict(cached=[7, 8, 9, 0], rows=[1, 1, 7, 16]),
    "no rows": dict(cached=[5, 0, 16], rows=[0, 0, 0]),
    "some without rows": dict(cached=[5, 0, 16, 3], rows=[0, 9, 0, 30], adapter=[3, -1, 2, 0]),
    "pages held already": dict(cached=[3, 8, 20], rows=[9, 9, 2], held=[4, 2, 3]),
    "held clamped": dict(cached=[3, 8, 20], rows=[9, 9, 2], held=[-4, 9999, 0]),
    "lengths clamped": dict(cached=[-3, 50, 7], rows=[99, 4, -2], max_q=6, max_kv=40, tokens=20),
    "rows that do not fit": dict(cached=[0, 4, 9, 2], rows=[5, 6, 7, 1], tokens=15),
    "nothing fits": dict(cached=[0, 4], rows=[5, 6], tokens=3),
    "pages run out": dict(cached=[0, 4, 9, 2], rows=[20, 30, 17, 1], spare=0, short=9),
    "no free pages": dict(cached=[4, 8], rows=[4, 1], spare=0, short=10 ** 6),
    "count past the list": dict(cached=[4, 8], rows=[4, 1], short=-10 ** 6),
    "rows behind the last": dict(cached=[4, 8], rows=[4, 1], tokens=300, adapter=[1, 7]),
    "absent and foreign pages": dict(cached=[30, 60], rows=[9, 5], num_pages=6),
    "wide table": dict(cached=[4, 8], rows=[40, 1], width=64, stride=70),
    "page 4096": dict(cached=[4095, 4096, 10], rows=[2, 1, 4096], page=4096),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("optional", [True, False])
def test_plan(gpu, name, optional):
    c = Case(**CASES[name]).upload(optional)
    c.call()
    c.check()


@pytest.mark.parametrize("seqs,most,ctx,page", [(256, 8, 4000, 16), (1000, 1, 3000, 64), (4096, 3, 100, 8), (5, 9000, 20000, 32),
                                                (257, 300, 1, 8)])
def test_plan_batches(gpu, seqs, most, ctx, page):
    r = np.random.default_rng(seqs)
    c = Case(cached=r.integers(0, ctx + 1, seqs), rows=r.integers(0, most + 1, seqs), page=page,
             adapter=r.integers(-1, 9, seqs), tokens=int(seqs * most * 0.4) + 1).upload()
    c.call()
    c.check()


def test_plan_again_and_replayed(gpu):
    """A plan reads only what it does not write: the same again, eager and from a graph."""
    r = np.random.default_rng(3)
    c = Case(cached=r.integers(0, 90, 40), rows=r.integers(0, 30, 40)).upload()
    stream = g4.Stream()
    c.call()
    c.check()
    graph = g4.Graph(stream, lambda: c.call(stream.handle))
    for _ in range(3):
        for n in ("q_start", "row_slot", "held_out"):
            c.d[n].fill(0)
        c.d["table"].upload(c.table)
        g4.synchronize()
        graph.launch()
        stream.synchronize()
        c.check()
        c.call()
        c.check()
    graph.close()


def release(table, first, last, free, count):
    free, count = free.copy(), min(max(count, 0), len(free))
    for row, a, b in zip(table, first, last):
        a = min(max(a, 0), table.shape[1])
        for e in row[a:max(min(b, table.shape[1]), a)]:
            if count < len(free):
                free[count] = e
                count += 1
    return free, count


@pytest.mark.parametrize("seqs,width,capacity,count,stride", [
    (1, 1, 10, 3, 1), (3, 40, 500, 17, 40), (3, 40, 30, 5, 44), (300, 70, 30000, 0, 70), (4096, 3, 20000, 100, 3),
    (2, 9000, 20000, 11, 9000), (5, 8, 40, 40, 8), (5, 8, 40, 99, 8), (5, 8, 40, -3, 8)])
def test_release(gpu, seqs, width, capacity, count, stride):
    r = np.random.default_rng(width)
    table = r.integers(0, 10 ** 6, (seqs, stride)).astype(np.int32)
    first, last = (r.integers(-2, width + 3, seqs).astype(np.int32) for _ in range(2))
    last[::3] = 2 ** 31 - 1
    free = np.full(capacity, -1, np.int32)
    want, n = release(table[:, :width], first, last, free, count)
    d_free, d_table, out = dev(free), dev(table), dev(np.zeros(1, np.int32))
    view = d_table if stride == width else View(d_table, 0, (seqs, width), (stride, 1), np.int32)
    pages = gs.FreePages(d_free, dev(np.array([count], np.int32)), 10 ** 6, 16)
    for _ in range(2):  # the count it reads stays, so a second call does the same
        gs.release_pages(pages, view, dev(first), dev(last), out)
        g4.synchronize()
        assert np.array_equal(d_free.download(), want) and out.download()[0] == n
        assert np.array_equal(d_table.download(), table)


def test_pages_go_round(gpu):
    """Requests come, grow and leave, over two counts and two held arrays in turn: no page is ever held twice."""
    r = np.random.default_rng(11)
    seqs, page, width, total = 6, 8, 12, 50
    free, table = dev(r.permutation(total).astype(np.int32)), dev(np.full((seqs, width), -1, np.int32))
    counts = [dev(np.array([total], np.int32)), dev(np.zeros(1, np.int32))]
    lists = [gs.FreePages(free, c, total, page) for c in counts]
    held = [dev(np.zeros(seqs, np.int32)) for _ in range(2)]
    lens, now, h = np.zeros(seqs, np.int32), 0, 0
    q_start, kv_len, served = (dev(np.zeros(n, np.int32)) for n in (seqs + 1, seqs, 1))
    for step in range(40):
        rows = np.where(lens == 0, r.integers(1, 40, seqs), r.integers(0, 5, seqs)).astype(np.int32)
        rows = np.minimum(rows, page * width - lens)
        gs.plan_chunk(lists[now], dev(lens), dev(rows), table, q_start, kv_len, counts[1 - now], served, tokens=100, max_q=64,
                      max_kv=page * width, held=held[h], held_out=held[1 - h])
        now, h = 1 - now, 1 - h
        g4.synchronize()
        lens, have = kv_len.download(), held[h].download()
        t, left = table.download(), int(counts[now].download()[0])
        inside = [p for s in range(seqs) for p in t[s, :have[s]]] + list(free.download()[:left])
        assert sorted(inside) == list(range(total)), step
        assert (have * page >= lens).all()
        gone = (r.random(seqs) < 0.3) | (lens >= page * width - 2)
        last = np.where(gone, have, 0).astype(np.int32)
        gs.release_pages(lists[now], table, dev(np.zeros(seqs, np.int32)), dev(last), counts[1 - now])
        now = 1 - now
        lens = np.where(gone, 0, lens).astype(np.int32)
        held[h].upload(np.where(gone, 0, have).astype(np.int32))
