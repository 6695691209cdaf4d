"""The serving operators as a draft-and-verify pass runs them: projections' int8 codes into the paged
cache, attention back to codes, the o projection, logits, and the verdict on the drafts."""
import numpy as np
import pytest

import g4decode as gd
import g4serve as gs
import g4synth as syn
import g4w8a8 as g4
from servecases import dev
from test_gpu_serve_verify import verify

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, DIM, VOCAB, PAGE = 512, 4, 64, 1000, 8
PROMPTS, DRAFTS = [45, 20, 3], [3, 1, 0]
ACT, PROJ, OUT = 0.05, 0.11, 2.0 ** -4  # scales: the input's codes, the projections', attention's
SCALE = DIM ** -0.5


class Layer:
    """One attention layer and a head over random int8 weights, on a cache of `kind`."""

    def __init__(self, kind, window):
        self.window = window
        shapes = {"q": (HEADS * DIM, HIDDEN), "k": (DIM, HIDDEN), "v": (DIM, HIDDEN), "o": (HIDDEN, HEADS * DIM),
                  "head": (VOCAB, HIDDEN)}
        self.w = {n: (dev(syn.weights("pass", n, r, k, 8)), dev(syn.row_scales("pass", n, r)), k, r)
                  for n, (r, k) in shapes.items()}
        total = [p + d + 1 for p, d in zip(PROMPTS, DRAFTS)]
        need = [-(-n // PAGE) for n in total]
        order = np.random.default_rng(1).permutation(sum(need) + 2)
        table = np.full((len(need), max(need)), -1, np.int32)
        for s, n in enumerate(need):
            table[s, :n], order = order[:n], order[n:]
        shape = (sum(need) + 2, PAGE, 1, DIM)
        pools = [dev(np.zeros(shape, np.int8 if kind == "i8" else np.float16)) for _ in range(2)]
        scales = [dev(np.zeros((shape[0], 1, PAGE), np.float32)) for _ in range(2)] if kind == "i8" else [None, None]
        self.pages = gs.KVPages(*pools, *scales)
        self.table = dev(table)
        r = np.random.default_rng(2)
        self.gains = [dev(r.uniform(0.5, 1.5, DIM).astype(np.float32)) for _ in range(2)]
        self.rope = [dev(x) for x in gd.rope_tables(max(total), DIM, 1e4, 1.0)]

    def chunk(self, rows, kv):
        start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        return gs.Chunk(dev(start), dev(np.array(kv, np.int32)), self.table, int(start[-1]), max(rows), max(kv))

    def buffers(self, chunk):
        t = chunk.tokens
        b = {n: dev(np.zeros((t, h, DIM), x)) for n, h, x in (
            ("q", HEADS, np.int8), ("k", 1, np.int8), ("v", 1, np.int8), ("qr", HEADS, np.float16), ("a", HEADS, np.int8))}
        b["o"], b["logits"] = dev(np.zeros((t, HIDDEN), np.int8)), dev(np.zeros((t, VOCAB), np.float32))
        b["ws"] = g4.DeviceBuffer(gs.attention_chunk_workspace_bytes(self.pages, chunk, HEADS, self.window))
        return b

    def linear(self, name, x, out, t, in_scale, out_scale, stream):
        w, s, k, n = self.w[name]
        g4.linear(8, w, s, x, out, k, n, t, in_scale, out_scale, stream=stream)

    def run(self, chunk, x, b, stream=None):
        t = chunk.tokens
        for n in "qkv":
            self.linear(n, x, b[n], t, ACT, PROJ, stream)
        gs.paged_prologue(self.pages, chunk, b["q"], b["k"], b["v"], b["qr"], *self.gains, *self.rope, x_scale=PROJ,
                          stream=stream)
        gs.attention_chunk(self.pages, chunk, b["qr"], b["a"], b["ws"], scale=SCALE, window=self.window, in_scale=OUT,
                           stream=stream)
        self.linear("o", b["a"], b["o"], t, OUT, ACT, stream)
        self.linear("head", b["o"], b["logits"], t, ACT, 0.0, stream)


def codes(r, t):
    return np.clip(np.rint(30 * r.standard_normal((t, HIDDEN))), -128, 127).astype(np.int8)


@pytest.mark.parametrize("window", [0, 24])
@pytest.mark.parametrize("kind", ["i8", "f16"])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_prompt_drafts_verdict(gpu, kind, window, temperature):
    r = np.random.default_rng(7)
    layer = Layer(kind, window)
    prompt = layer.chunk(PROMPTS, PROMPTS)
    layer.run(prompt, dev(codes(r, prompt.tokens)), layer.buffers(prompt))

    rows = [d + 1 for d in DRAFTS]
    kv = [p + n for p, n in zip(PROMPTS, rows)]
    c = layer.chunk(rows, kv)
    x, b = dev(codes(r, c.tokens)), layer.buffers(c)
    n = sum(DRAFTS)
    start = np.concatenate([[0], np.cumsum(DRAFTS)]).astype(np.int32)
    layer.run(c, x, b)
    g4.synchronize()
    logits = b["logits"].download()
    at = [start[s] + s + i for s, d in enumerate(DRAFTS) for i in range(d)]
    draft_logits = (logits[at] + logits.std() * r.standard_normal((n, VOCAB))).astype(np.float32)
    drafts = draft_logits.argmax(1).astype(np.int32)
    drafts[0] = logits[at[0]].argmax()
    u, u_next = r.random(n).astype(np.float32), r.random(len(DRAFTS)).astype(np.float32)
    given = [dev(a) for a in (draft_logits, drafts, start, u, u_next)]
    if temperature == 0:
        given[0] = given[3] = given[4] = None
    most = max(DRAFTS)
    outs = [dev(np.zeros((len(DRAFTS), most + 1), np.int32)), dev(np.zeros(len(DRAFTS), np.int32)),
            dev(np.zeros((len(DRAFTS), most + 1), np.float32))]
    vws = g4.DeviceBuffer(gs.verify_workspace_bytes(len(DRAFTS), n, VOCAB))

    def whole(stream=None):
        layer.run(c, x, b, stream)
        gs.verify_drafts(b["logits"], *given, *outs, vws, cap=30.0, temperature=temperature, stream=stream)

    whole()
    g4.synchronize()
    first = [a.download() for a in (*outs, b["a"], b["logits"])]

    # attention's codes, from the cache as it reads back and the queries as they were given
    whole_chunk = layer.chunk(kv, kv)
    k, v = (dev(np.zeros((sum(kv), 1, DIM), np.float32)) for _ in range(2))
    gs.kv_read(layer.pages, whole_chunk, k, v)
    k, v, q = (a.download().astype(np.float64) for a in (k, v, b["qr"]))
    got = first[3].astype(np.float64) * OUT
    for s, m in enumerate(rows):
        o = sum(kv[:s])
        kk, vv = k[o:o + kv[s], 0], v[o:o + kv[s], 0]
        for i in range(m):
            t, pos = sum(rows[:s]) + i, kv[s] - m + i
            lo = max(0, pos - window + 1) if window else 0
            z = (q[t] @ kk[lo:pos + 1].T) * SCALE
            p = np.exp(z - z.max(1, keepdims=True))
            want = np.clip((p / p.sum(1, keepdims=True)) @ vv[lo:pos + 1], -128 * OUT, 127 * OUT)
            # half a code; weights off by 2^-12 in their rounding and by exp(ds) in their scores, in the product
            # and in the sum: ds is half of 2^-15 of q's largest on every k, and f32's (DIM + 8) 2^-24
            ds = SCALE * np.abs(kk).sum(1).max() * np.abs(q[t]).max() * (1 / 65024 + (DIM + 8) * 2.0 ** -24)
            tol = OUT / 2 + 2 * np.abs(vv).max() * (2.0 ** -12 + 1.1 * ds + 2.0 ** -16)
            assert (np.abs(got[t] - want) <= tol).all()

    tokens, accepted, lp, margin = verify(first[4], None if temperature == 0 else draft_logits, drafts, start, u, u_next,
                                          most, 30.0, temperature)
    assert temperature == 0 or margin > 2.0 ** -32
    assert np.array_equal(first[0], tokens) and np.array_equal(first[1], accepted)
    assert (np.abs(first[2] - lp) <= np.abs(lp) * 2.0 ** -24 * 1.01 + 2.0 ** -36).all()

    # captured: every replay gives the eager bits, with eager passes in between
    stream = g4.Stream()
    graph = g4.Graph(stream, lambda: whole(stream.handle))
    for _ in range(3):
        for a in (*outs, b["a"], b["logits"], b["qr"]):
            a.fill(0)
        g4.synchronize()
        graph.launch()
        stream.synchronize()
        for a, w in zip((*outs, b["a"], b["logits"]), first):
            assert np.array_equal(a.download().view(np.uint8), w.view(np.uint8))
        whole()
        g4.synchronize()
    graph.close()
