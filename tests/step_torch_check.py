"""Page plans, adapters and sampling on torch tensors, in a process of its own (torch has to be loaded before the
library; the other tests run on the system's HIP runtime): on a side stream behind the work that makes the operands, on
two streams at once, and in captured graphs. Run by test_gpu_step_torch.py; prints "ok" at the end."""
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [os.path.join(os.path.dirname(HERE), "gemma4-webgpu-engine_amd")]
import g4serve as gs  # noqa: E402

SEQS, TOKENS, MAX_Q, PAGES, PAGE, WIDTH, ADAPTERS, VOCAB = 6, 70, 32, 64, 8, 12, 5, 20001


class Program:
    """The operators as one pass over operands that `feed` brings in. k, rank: with 64 and 8 the adapters take one launch,
    with 6144 and 72 two."""

    def __init__(self, k, rank, n=520):
        z = lambda *shape, dt=torch.int32: torch.zeros(shape, dtype=dt, device="cuda")
        f = lambda *shape: z(*shape, dt=torch.float32)
        h = lambda *shape: z(*shape, dt=torch.float16)
        self.list, self.count = z(PAGES), z(1)
        self.free = gs.FreePages(self.list, self.count, PAGES, PAGE)
        self.table, self.cached, self.rows, self.held, self.seq_adapter = z(SEQS, WIDTH), z(SEQS), z(SEQS), z(SEQS), z(SEQS)
        self.q_start, self.kv_len, self.left, self.served, self.held_out, self.last_row = (
            z(SEQS + 1), z(SEQS), z(1), z(1), z(SEQS), z(SEQS))
        self.row_pos, self.row_slot, self.row_adapter = z(TOKENS), z(TOKENS), z(TOKENS)
        self.back, self.back_count = z(PAGES), z(1)
        self.back_free = gs.FreePages(self.back, self.left, PAGES, PAGE)
        self.first, self.last = z(SEQS), z(SEQS)
        self.a, self.b, self.x, self.base, self.out = (h(ADAPTERS, rank, k), h(ADAPTERS, n, rank), h(TOKENS, k), f(TOKENS, n),
                                                       f(TOKENS, n))
        self.scales = f(ADAPTERS)
        self.adapters = gs.Adapters(self.a, self.b, scales=self.scales)
        byte = lambda n: z(n, dt=torch.uint8)
        self.groups = byte(gs.adapter_groups_bytes(TOKENS, ADAPTERS))
        self.aws = byte(gs.adapter_workspace_bytes(self.adapters, TOKENS))
        self.logits, self.u, self.tokens, self.lps = f(TOKENS, VOCAB), f(SEQS), z(SEQS), f(SEQS)
        self.temperature, self.top_k, self.top_p, self.min_p = f(SEQS), z(SEQS), f(SEQS), f(SEQS)
        self.sws = byte(gs.sample_workspace_bytes(SEQS, VOCAB))

    def inputs(self):
        return [self.list, self.count, self.table, self.cached, self.rows, self.held, self.seq_adapter, self.first, self.last,
                self.a, self.b, self.x, self.base, self.scales, self.logits, self.u, self.temperature, self.top_k, self.top_p,
                self.min_p]

    def data(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        ints = lambda lo, hi, *shape: torch.randint(lo, hi, shape or (SEQS,), generator=g, device="cuda").int()
        real = lambda x, s=1.0: (s * torch.randn(x.shape, generator=g, device="cuda")).to(x.dtype)
        rand = lambda: torch.rand(SEQS, generator=g, device="cuda")
        cached = ints(0, 30)
        held = (cached + PAGE - 1) // PAGE
        order = torch.randperm(PAGES, generator=g, device="cuda").int()
        table = order[:SEQS * 5].view(SEQS, 5)
        wide = torch.full((SEQS, WIDTH), -1, dtype=torch.int32, device="cuda")
        wide[:, :5] = torch.where(torch.arange(5, device="cuda") < held[:, None], table, -1)
        free = torch.cat([order[SEQS * 5:], order[:SEQS * 5]])
        return [free, ints(20, 30, 1), wide, cached, ints(0, 20), held, ints(-1, ADAPTERS), ints(0, 1), held.clone(),
                real(self.a, 0.1), real(self.b, 0.1), real(self.x), real(self.base), rand()[:ADAPTERS].clone(),
                real(self.logits, 4.0), rand(), rand() * 1.5, ints(0, 300), rand(), rand() * 0.1]

    def feed(self, data):
        for x, y in zip(self.inputs(), data):
            x.copy_(y)
        for x in (self.out, self.back, self.row_pos, self.row_slot, self.row_adapter):
            x.fill_(-5)

    def run(self):
        gs.plan_chunk(self.free, self.cached, self.rows, self.table, self.q_start, self.kv_len, self.left, self.served,
                      tokens=TOKENS, max_q=MAX_Q, max_kv=WIDTH * PAGE, held=self.held, held_out=self.held_out,
                      seq_adapter=self.seq_adapter, row_pos=self.row_pos, row_slot=self.row_slot,
                      row_adapter=self.row_adapter, last_row=self.last_row)
        gs.adapter_groups(self.row_adapter, self.groups, ADAPTERS)
        gs.adapter_linear(self.adapters, self.groups, self.x, self.base, self.out, self.aws)
        gs.sample_tokens(self.logits, self.u, self.tokens, self.lps, self.sws, row_index=self.last_row,
                         temperature=self.temperature, top_k=self.top_k, top_p=self.top_p, min_p=self.min_p, cap=30.0)
        gs.release_pages(self.back_free, self.table, self.first, self.last, self.back_count)

    def outputs(self):
        return [x.clone() for x in (self.q_start, self.kv_len, self.left, self.served, self.held_out, self.last_row, self.row_pos,
                                    self.row_slot, self.row_adapter, self.table, self.out, self.tokens, self.lps, self.back,
                                    self.back_count)]

    def check(self):
        """The products in 64 bits on the host, the rest for what it has to be at least."""
        ids, x = self.row_adapter.cpu(), self.x.cpu().double()
        want, off = self.base.cpu().double(), self.base.cpu().double().abs() * 2.0 ** -22
        for r, i in enumerate(ids.tolist()):
            if i < 0:
                continue
            a, b, s = self.a[i].cpu().double(), self.b[i].cpu().double(), float(self.scales[i])
            want[r] += s * (b @ (a @ x[r]))
            # sums in f32 of k products, then of a rank's
            off[r] += (self.x.shape[1] + a.shape[0] + 10) * 2.0 ** -24 * s * (b.abs() @ (a.abs() @ x[r].abs()))
        given = ids > -2
        assert ((self.out.cpu().double() - want).abs() <= off)[given].all()
        assert (self.out.cpu()[~given] == -5).all()  # rows behind the last are left
        assert int(self.served) > 0 and int(self.q_start[-1]) == int(given.sum())
        drawn = self.tokens.cpu()
        assert ((drawn >= 0) == (self.last_row.cpu() >= 0)).all() and (drawn < VOCAB).all()
        n = int((self.last - self.first).sum())
        assert int(self.back_count) == int(self.left) + n
        gone = self.back[int(self.left):int(self.back_count)].cpu().tolist()
        assert sorted(gone) == sorted(p for s in range(SEQS) for p in self.table[s, :int(self.held[s])].cpu().tolist())


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


progs = [Program(64, 8), Program(6144, 72)]
slow = torch.randn(4096, 4096, device="cuda")
sides = [torch.cuda.Stream(), torch.cuda.Stream()]
for prog in progs:
    sets = [prog.data(s) for s in range(4)]
    want = []
    for data in sets:
        prog.feed(data)
        prog.run()
        want.append(prog.outputs())
        prog.check()
    print("eager", flush=True)
    torch.cuda.synchronize()
    for data, w in zip(sets, want):
        with torch.cuda.stream(sides[0]):
            x = slow
            for _ in range(12):  # some milliseconds in front of the operands
                x = x @ slow * 0.01
            prog.feed(data)
            prog.run()
            got = prog.outputs()
        sides[0].synchronize()
        assert same(got, w)
    print("side stream", flush=True)
    # two graphs of one program share its workspaces, as its eager calls do
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:
        with torch.cuda.graph(graph):
            prog.run()
    for i, (data, w) in enumerate(list(zip(sets, want)) * 2):
        prog.feed(data)
        graphs[i % 2].replay()
        assert same(prog.outputs(), w)
        prog.feed(data)
        prog.run()  # eager work between the replays
        torch.cuda.synchronize()
    print("captured", flush=True)
    prog.kept = sets, want
# two programs at once, each on a stream and in workspaces of its own
torch.cuda.synchronize()
got = [[], []]
for i in range(4):
    for p, side in enumerate(sides):
        with torch.cuda.stream(side):
            progs[p].feed(progs[p].kept[0][i])
            progs[p].run()
            got[p].append(progs[p].outputs())
torch.cuda.synchronize()
assert all(same(g, w) for p in range(2) for g, w in zip(got[p], progs[p].kept[1]))
print("ok")
