"""The serving operators on torch tensors, in a process of its own (torch has to be loaded before the library;
the other tests run on the system's HIP runtime): on a side stream behind the work that makes the operands, and
in a captured graph. Run by test_gpu_serve_torch.py; prints "ok" at the end."""
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [os.path.join(os.path.dirname(HERE), "gemma4-webgpu-engine_amd")]
import g4serve as gs  # noqa: E402

SEQS, ROWS, KV, HEADS, KVH, DIM, PAGE, VOCAB, DRAFTS = 3, 5, 75, 4, 2, 64, 16, 1500, 2
T = SEQS * ROWS


class Program:
    """The four operators as one pass over operands that `feed` brings in."""

    def __init__(self, kind):
        z = lambda *shape, dt=torch.float32: torch.zeros(shape, dtype=dt, device="cuda")
        need = -(-KV // PAGE)
        n = SEQS * need
        dt = torch.int8 if kind == "i8" else torch.float16
        scales = [z(n, KVH, PAGE) for _ in range(2)] if kind == "i8" else [None, None]
        self.pools = [z(n, PAGE, KVH, DIM, dt=dt) for _ in range(2)] + [x for x in scales if x is not None]
        self.pages = gs.KVPages(*self.pools[:2], *scales)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        self.chunk = gs.Chunk(i32(range(0, T + 1, ROWS)), i32([KV] * SEQS),
                              torch.randperm(n, generator=torch.Generator().manual_seed(1)).int().view(SEQS, need).cuda(),
                              T, ROWS, KV)
        self.wide = z(T, (HEADS + 2 * KVH) * DIM, dt=torch.float16)  # one projection's rows: q, k, v
        a, b = HEADS * DIM, (HEADS + KVH) * DIM
        self.parts = [x.view(T, -1, DIM) for x in (self.wide[:, :a], self.wide[:, a:b], self.wide[:, b:])]
        self.q, self.o = z(T, HEADS, DIM, dt=torch.float16), z(T, HEADS, DIM)
        self.ws = torch.empty(gs.attention_chunk_workspace_bytes(self.pages, self.chunk, HEADS), dtype=torch.uint8, device="cuda")
        self.back = [z(T, KVH, DIM) for _ in range(2)]
        rows = SEQS * (DRAFTS + 1)
        self.logits, self.draft_logits = z(rows, VOCAB), z(SEQS * DRAFTS, VOCAB)
        self.drafts, self.start = z(SEQS * DRAFTS, dt=torch.int32), i32(range(0, SEQS * DRAFTS + 1, DRAFTS))
        self.u, self.u_next = z(SEQS * DRAFTS), z(SEQS)
        self.verdict = [z(SEQS, DRAFTS + 1, dt=torch.int32), z(SEQS, dt=torch.int32), z(SEQS, DRAFTS + 1)]
        self.vws = torch.empty(gs.verify_workspace_bytes(SEQS, SEQS * DRAFTS, VOCAB), dtype=torch.uint8, device="cuda")

    def data(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        out = [torch.randn(self.wide.shape, generator=g, device="cuda").half()]
        for x in self.pools:
            y = torch.randn(x.shape, generator=g, device="cuda")
            out.append((30 * y).clamp(-127, 127).to(x.dtype) if x.dtype == torch.int8 else
                       y.abs() / 50 if x.dtype == torch.float32 else y.half())
        logits = 3 * torch.randn(self.logits.shape, generator=g, device="cuda")
        at = torch.arange(SEQS * DRAFTS, device="cuda")
        dl = logits[at + at // DRAFTS] + torch.randn(self.draft_logits.shape, generator=g, device="cuda")
        out += [logits, dl, dl.argmax(1).int(), torch.rand(self.u.shape, generator=g, device="cuda"),
                torch.rand(self.u_next.shape, generator=g, device="cuda")]
        return out

    def feed(self, data):
        for x, y in zip([self.wide, *self.pools, self.logits, self.draft_logits, self.drafts, self.u, self.u_next], data):
            x.copy_(y)

    def run(self):
        gs.paged_prologue(self.pages, self.chunk, *self.parts, self.q)
        gs.attention_chunk(self.pages, self.chunk, self.q, self.o, self.ws, scale=0.1)
        gs.kv_read(self.pages, self.chunk, *self.back)
        gs.verify_drafts(self.logits, self.draft_logits, self.drafts, self.start, self.u, self.u_next, *self.verdict,
                         self.vws, cap=30.0, temperature=0.9)

    def outputs(self):
        return [x.clone() for x in (self.q, self.o, *self.back, *self.verdict)]

    def plain_attention(self):
        """In 64 bits on the host, from the cache as it stands."""
        k, v, *s = (x.cpu().double() for x in self.pools)
        if s:
            k, v = (x * y.permute(0, 2, 1)[..., None] for x, y in zip((k, v), s))
        table, q = self.chunk.buffers[2].cpu().long(), self.q.cpu().double()
        out = torch.zeros(T, HEADS, DIM, dtype=torch.float64)
        for r in range(T):
            p = torch.arange(KV - ROWS + r % ROWS + 1)
            page = table[r // ROWS, p // PAGE]
            for h in range(HEADS):
                kk, vv = (x[page, p % PAGE, h // (HEADS // KVH)] for x in (k, v))
                out[r, h] = torch.softmax(kk @ q[r, h] * 0.1, 0) @ vv
        return out, v.abs().max()


for kind in ("i8", "f16"):
    prog = Program(kind)
    sets = [prog.data(s) for s in range(4)]
    want = []
    for data in sets:
        prog.feed(data)
        prog.run()
        want.append(prog.outputs())
    # a weight is off by 2^-12 and by its score's error, numerator and sum (Q's digits: half of 2^-15 of its largest
    # on each of the 64 dims, |q| and |k| under 6: 64 * 6 * 6 * 0.1 * 2^-16)
    ref, vmax = prog.plain_attention()
    off = (prog.o.cpu().double() - ref).abs().max()
    assert off <= 2 * vmax * (2.0 ** -12 + 64 * 36 * 0.1 * 2.0 ** -16 + 2.0 ** -16), off
    print(kind, "eager", flush=True)

    side, slow = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for data, w in zip(sets, want):
        with torch.cuda.stream(side):
            x = slow
            for _ in range(12):  # some milliseconds in front of the operands
                x = x @ slow * 0.01
            prog.feed(data)
            prog.run()
            got = prog.outputs()
        side.synchronize()
        assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(got, w))
    print(kind, "side stream", flush=True)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prog.run()
    for data, w in list(zip(sets, want)) * 2:
        prog.feed(data)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(prog.outputs(), w))
        prog.feed(data)
        prog.run()  # eager work between the replays
        torch.cuda.synchronize()
    print(kind, "captured", flush=True)
print("ok")
