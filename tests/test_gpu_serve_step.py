"""A server's steps with every serving operator in its place: pages and slots planned on the GPU, projections with the
requests' adapters, the cache, attention, the head, and a drawn token a request, fed back as the next step's input;
requests come and go."""
import numpy as np
import pytest

import g4decode as gd
import g4serve as gs
import g4synth as syn
import g4w8a8 as g4
from servecases import dev
from test_gpu_serve_sample import sample

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, DIM, VOCAB, PAGE, SEQS, ADAPTERS, RANK = 512, 4, 64, 1000, 8, 4, 3, 16
TOKENS, MAX_Q, WIDTH, PAGES = 64, 40, 10, 36
ACT, OUT, SCALE, CAP = 0.05, 2.0 ** -4, DIM ** -0.5, 30.0
ADAPTER_OF = [2, -1, 0, 2]
FILTERS = dict(temperature=np.array([0.8, 1.0, 0.0, 1.3], np.float32), top_k=np.array([0, 50, 0, 7], np.int32),
               top_p=np.array([0.9, 1.0, 1.0, 0.8], np.float32), min_p=np.array([0.0, 0.02, 0.0, 0.0], np.float32))


class Server:
    def __init__(self, kind):
        r = np.random.default_rng(3)
        z = lambda n, dt=np.int32: dev(np.zeros(n, dt))
        shapes = {"q": (HEADS * DIM, HIDDEN), "k": (DIM, HIDDEN), "v": (DIM, HIDDEN), "o": (HIDDEN, HEADS * DIM),
                  "head": (VOCAB, HIDDEN)}
        self.w = {n: (dev(syn.weights("step", n, a, b, 8)), dev(syn.row_scales("step", n, a)), b, a)
                  for n, (a, b) in shapes.items()}
        self.a = (r.standard_normal((ADAPTERS, RANK, HIDDEN)) / 20).astype(np.float16)
        self.b = r.standard_normal((ADAPTERS, HEADS * DIM, RANK)).astype(np.float16)
        self.adapters = gs.Adapters(dev(self.a), dev(self.b))
        shape = (PAGES, PAGE, 1, DIM)
        pools = [z(shape, np.int8 if kind == "i8" else np.float16) for _ in range(2)]
        self.pages = gs.KVPages(*pools, *([z((PAGES, 1, PAGE), np.float32) for _ in range(2)] if kind == "i8" else []))
        self.free = dev(r.permutation(PAGES).astype(np.int32))
        self.counts = [dev(np.array([PAGES], np.int32)), z(1)]
        self.lists = [gs.FreePages(self.free, c, PAGES, PAGE) for c in self.counts]
        self.held = [z(SEQS), z(SEQS)]
        self.now = 0
        self.table = dev(np.full((SEQS, WIDTH), -1, np.int32))
        self.cached, self.rows, self.first, self.last = (z(SEQS) for _ in range(4))
        self.q_start, self.kv_len, self.served, self.last_row = z(SEQS + 1), z(SEQS), z(1), z(SEQS)
        self.row_pos, self.row_slot, self.row_adapter = (z(TOKENS) for _ in range(3))
        self.seq_adapter = dev(np.array(ADAPTER_OF, np.int32))
        self.groups = g4.DeviceBuffer(gs.adapter_groups_bytes(TOKENS, ADAPTERS))
        self.chunk = gs.Chunk(self.q_start, self.kv_len, self.table, TOKENS, MAX_Q, WIDTH * PAGE)
        f = lambda *n: z(n, np.float32)
        self.x, self.q, self.qa = z((TOKENS, HIDDEN), np.int8), f(TOKENS, HEADS * DIM), f(TOKENS, HEADS * DIM)
        self.k, self.v = f(TOKENS, DIM), f(TOKENS, DIM)
        self.qr, self.att = z((TOKENS, HEADS, DIM), np.float16), z((TOKENS, HEADS, DIM), np.int8)
        self.o, self.logits = z((TOKENS, HIDDEN), np.int8), f(TOKENS, VOCAB)
        self.gains = [dev(r.uniform(0.5, 1.5, DIM).astype(np.float32)) for _ in range(2)]
        self.rope = [dev(t) for t in gd.rope_tables(WIDTH * PAGE, DIM, 1e4, 1.0)]
        self.u, self.filters = f(SEQS), {n: dev(v) for n, v in FILTERS.items()}
        self.tokens, self.lps = z(SEQS), f(SEQS)
        self.ws = [g4.DeviceBuffer(n) for n in (gs.adapter_workspace_bytes(self.adapters, TOKENS),
                                                gs.attention_chunk_workspace_bytes(self.pages, self.chunk, HEADS),
                                                gs.sample_workspace_bytes(SEQS, VOCAB))]

    def linear(self, name, x, out, in_scale, out_scale, stream):
        w, s, k, n = self.w[name]
        g4.linear(8, w, s, x, out, k, n, TOKENS, in_scale, out_scale, stream=stream)

    def step(self, now, stream=None):
        """Everything of a step that the GPU does, on the counts and held pages `now`."""
        gs.plan_chunk(self.lists[now], self.cached, self.rows, self.table, self.q_start, self.kv_len, self.counts[1 - now],
                      self.served, tokens=TOKENS, max_q=MAX_Q, max_kv=WIDTH * PAGE, held=self.held[now],
                      held_out=self.held[1 - now], seq_adapter=self.seq_adapter, row_pos=self.row_pos, row_slot=self.row_slot,
                      row_adapter=self.row_adapter, last_row=self.last_row, stream=stream)
        gs.adapter_groups(self.row_adapter, self.groups, ADAPTERS, stream=stream)
        for n, out in (("q", self.q), ("k", self.k), ("v", self.v)):
            self.linear(n, self.x, out, ACT, 0.0, stream)
        gs.adapter_linear(self.adapters, self.groups, self.x, self.q, self.qa, self.ws[0], x_scale=ACT, stream=stream)
        heads = lambda b, h: type("V", (), dict(ptr=b.ptr, shape=(TOKENS, h, DIM), dtype=b.dtype))
        gs.paged_prologue(self.pages, self.chunk, heads(self.qa, HEADS), heads(self.k, 1), heads(self.v, 1), self.qr, *self.gains,
                          *self.rope, stream=stream)
        gs.attention_chunk(self.pages, self.chunk, self.qr, self.att, self.ws[1], scale=SCALE, in_scale=OUT, stream=stream)
        self.linear("o", self.att, self.o, OUT, ACT, stream)
        self.linear("head", self.o, self.logits, ACT, 0.0, stream)
        gs.sample_tokens(self.logits, self.u, self.tokens, self.lps, self.ws[2], row_index=self.last_row, cap=CAP, stream=stream,
                         **self.filters)


def embed(tokens, positions):
    r = [np.random.default_rng(int(t) * 1000 + int(p)) for t, p in zip(tokens, positions)]
    return np.stack([np.clip(np.rint(30 * g.standard_normal(HIDDEN)), -128, 127) for g in r]).astype(np.int8)


@pytest.mark.parametrize("kind", ["i8", "f16"])
def test_requests_come_and_go(gpu, kind):
    r = np.random.default_rng(5)
    s = Server(kind)
    stream = g4.Stream()
    graphs = [g4.Graph(stream, lambda: s.step(i, stream.handle)) for i in range(2)]
    lens, tokens = np.zeros(SEQS, np.int64), [[] for _ in range(SEQS)]
    prompts = [[int(t) for t in r.integers(0, VOCAB, n)] for n in (37, 5, 1, 20)]
    for step in range(9):
        new = [prompts[i] if not lens[i] else tokens[i][-1:] for i in range(SEQS)]
        rows = np.array([len(n) for n in new], np.int32)
        x = np.zeros((TOKENS, HIDDEN), np.int8)
        flat = [(t, lens[i] + j) for i in range(SEQS) for j, t in enumerate(new[i])][:TOKENS]
        x[:len(flat)] = embed(*zip(*flat))
        s.x.upload(x)
        s.cached.upload(lens.astype(np.int32))
        s.rows.upload(rows)
        u = r.random(SEQS).astype(np.float32)
        s.u.upload(u)
        g4.synchronize()
        before = [b.download() for b in (s.free, s.counts[s.now], s.held[s.now])]
        graphs[s.now].launch()
        stream.synchronize()
        outs = (s.tokens, s.lps, s.logits, s.row_slot, s.qa, s.counts[1 - s.now])
        replayed = [b.download() for b in outs]
        s.step(s.now)  # and eager, on the same inputs
        g4.synchronize()
        for b, w in zip(outs, replayed):
            assert np.array_equal(b.download().view(np.uint8), w.view(np.uint8)), step
        served, start = int(s.served.download()[0]), s.q_start.download()
        assert served == SEQS and start[-1] == rows.sum() <= TOKENS
        # pages: no two sequences share one, none is free too
        held, table = s.held[1 - s.now].download(), s.table.download()
        left = int(replayed[5][0])
        mine = [int(p) for i in range(SEQS) for p in table[i, :held[i]]]
        assert sorted(mine + [int(p) for p in before[0][:left]]) == list(range(PAGES))
        slots = [int(table[i, p // PAGE]) * PAGE + p % PAGE for i in range(SEQS) for p in range(lens[i], lens[i] + rows[i])]
        assert list(replayed[3][:start[-1]]) == slots
        # the q projection with each request's adapter: three sums in f32 of up to HIDDEN products
        q, ids = s.q.download().astype(np.float64), s.row_adapter.download()
        for row in range(int(start[-1])):
            want, off = q[row], np.abs(q[row]) * 2.0 ** -22
            if ids[row] >= 0:
                a, b, xr = (y.astype(np.float64) for y in (s.a[ids[row]], s.b[ids[row]], x[row]))
                h, ha = ACT * (xr @ a.T), ACT * (np.abs(xr) @ np.abs(a).T)
                want = want + h @ b.T
                off = off + (HIDDEN + RANK + 10) * 2.0 ** -24 * (ha @ np.abs(b).T)
            assert (np.abs(replayed[4][row] - want) <= off).all()
        # the drawn tokens, from the logits of each request's last row
        for i in range(SEQS):
            row = replayed[2][start[i + 1] - 1]
            f = {n: v[i] for n, v in FILTERS.items()}
            want, _ = sample(row, CAP, f["temperature"], f["top_k"], f["top_p"], f["min_p"], u[i])
            near = {sample(row, CAP, f["temperature"], f["top_k"], f["top_p"], f["min_p"], u[i], (a, b))[0]
                    for a in (-1e-11, 0, 1e-11) for b in (-1e-11, 0, 1e-11)}
            assert replayed[0][i] == want or replayed[0][i] in near
            tokens[i].append(int(replayed[0][i]))
        lens += rows
        s.now = 1 - s.now
        # requests 0 and 3 finish in turn; a new prompt takes the place
        gone = {3: 0, 5: 3, 6: 0}.get(step)
        if gone is not None:
            first, last = np.zeros(SEQS, np.int32), np.zeros(SEQS, np.int32)
            last[gone] = held[gone]
            s.first.upload(first)
            s.last.upload(last)
            gs.release_pages(s.lists[s.now], s.table, s.first, s.last, s.counts[1 - s.now])
            g4.synchronize()
            held[gone] = lens[gone] = 0
            s.counts[s.now].upload(s.counts[1 - s.now].download())
            s.held[s.now].upload(held)
            tokens[gone], prompts[gone] = [], [int(t) for t in r.integers(0, VOCAB, 11 + step)]
    for g in graphs:
        g.close()
