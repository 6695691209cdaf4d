"""Serving operators over a paged KV cache, as measurable cases: the chunk prologue with its
quantising store and the read-back, attention of a chunk of new tokens, and the verification of
drafted tokens.

The shape of the listed cases is the model of the tests and the benchmark (8 query heads on one KV
head of 256, a vocabulary of 262144, a 512-position window), plus a grouped layout of narrower heads.

A batch is described the same way for every cache operator: sequence s has the rows
q_start[s] .. q_start[s + 1] of the chunk, kv_len[s] positions once the chunk is in the cache, and
row i of it is position kv_len[s] - (rows of s) + i. Position p of sequence s is slot p % page of
page page_table[s][p / page].

A case is a dict with "kind" and that kind's sizes:
  store   norm, RoPE and the store of a chunk, and the chunk's rows read back
  read    the last `m` positions of every sequence read back
  attn    causal attention of the chunk over everything the cache holds
  verify  `drafts` drafted tokens a sequence against the target's logits; temperature 0 is greedy
"ragged" cases take different lengths for each sequence, by a fixed rule.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
VOCAB = 262144
DTYPES = {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8}


# ---- the cases ----------------------------------------------------------------------------------

def _cache(kind, name, **kw):
    c = {"name": name, "kind": kind, "seqs": 1, "m": 1, "ctx": 0, "ragged": False, "heads": 8,
         "kv_heads": 1, "dim": 256, "page": 16, "cache": "i8"}
    c.update(kw)
    return c


def listed():
    return [
        # A decode step's new token, the 4096th of its sequence: projections' int8 codes in.
        _cache("store", "store_m1", ctx=4095, x="i8", norm=True, out="f16"),
        # The first chunk of a 2048-token prompt.
        _cache("store", "store_m2048", m=2048, x="i8", norm=True, out="f16"),
        # A whole sequence handed to a program with a contiguous f32 cache.
        _cache("read", "read_4095_f32", m=4095, out="f32"),
        # 32 sequences of up to 4096 positions, four narrower KV heads, to f16.
        _cache("read", "read_b32_f16", seqs=32, m=4096, ragged=True, heads=16, kv_heads=4, dim=128,
               out="f16"),
        # A draft-verify pass of one sequence: four tokens on 4096 positions.
        _cache("attn", "attn_b1_m4", m=4, ctx=4092, window=0),
        # Draft-verify of 32 sequences, one to eight tokens each, at different lengths.
        _cache("attn", "attn_b32_m8", seqs=32, m=8, ctx=4088, ragged=True, window=0),
        # Single tokens of 32 long sequences, four query heads on each of two KV heads.
        _cache("attn", "attn_b32_long", seqs=32, m=1, ctx=16383, kv_heads=2, dim=128, cache="f16",
               page=64, window=0),
        # A 512-token prompt chunk in a layer with a sliding window.
        _cache("attn", "attn_m512_window", m=512, ctx=3584, cache="f16", window=512),
        # A 2048-token prompt chunk that ends at position 8192, in a layer without one.
        _cache("attn", "attn_m2048", m=2048, ctx=6144, window=0),
        # Greedy verification of a decode batch with four drafts each, from a drafter that has no
        # probabilities.
        {"name": "verify_b32_greedy", "kind": "verify", "seqs": 32, "drafts": 4, "ragged": False,
         "vocab": VOCAB, "cap": 30.0, "temperature": 0.0, "draft_logits": False},
        # Sampled verification of one sequence's four drafts.
        {"name": "verify_b1", "kind": "verify", "seqs": 1, "drafts": 4, "ragged": False,
         "vocab": VOCAB, "cap": 0.0, "temperature": 1.0, "draft_logits": True},
        # And of 32 sequences with up to seven.
        {"name": "verify_b32", "kind": "verify", "seqs": 32, "drafts": 7, "ragged": True,
         "vocab": VOCAB, "cap": 30.0, "temperature": 0.8, "draft_logits": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _scores(c):
    """Score elements of a plain pass over the padded batch."""
    return c["seqs"] * c["heads"] * c["m"] * (c["ctx"] + c["m"])


def draw(rng):
    kind = rng.choice(["store", "read", "attn", "attn", "attn", "verify"])
    if kind == "verify":
        seqs = _log(rng, 1, 32)
        return {"kind": kind, "seqs": seqs, "drafts": rng.randint(1, 7), "ragged": rng.random() < 0.5,
                "vocab": _log(rng, 1000, VOCAB), "cap": rng.choice([0.0, 30.0]),
                "temperature": rng.choice([0.0, 0.6, 1.0]), "draft_logits": rng.random() < 0.7}
    kv = rng.choice([1, 1, 2, 4, 8])
    c = {"kind": kind, "heads": kv * rng.choice([1, 2, 3, 4, 8]), "kv_heads": kv,
         "dim": rng.choice([64, 128, 256, 256]), "page": rng.choice([8, 16, 32, 64, 128]),
         "cache": rng.choice(["i8", "f16"]), "ragged": rng.random() < 0.5}
    while True:
        c["seqs"], c["m"] = _log(rng, 1, 64), _log(rng, 1, 2048)
        c["ctx"] = 0 if kind == "read" else _log(rng, 1, 16384) - 1
        held = 2 * c["seqs"] * (c["ctx"] + c["m"]) * kv * c["dim"]
        if kind == "attn":
            fits = _scores(c) <= 1 << 27 and held <= 1 << 28
        else:
            fits = c["seqs"] * c["m"] * c["heads"] * c["dim"] <= 1 << 24 and held <= 1 << 28
        if fits:
            break
    if kind == "attn":
        c["window"] = rng.choice([0, 0, 100, 512])
    else:
        c["out"] = "f16" if kind == "store" else rng.choice(["f16", "f32"])
    if kind == "store":
        c["norm"] = rng.random() < 0.7
        c["x"] = rng.choice(["i8", "f32", "f16"]) if c["norm"] else "f16"
    return c


def _lengths(c):
    """Rows and final lengths of each sequence: the same for every seed."""
    ms, kvs = [], []
    for s in range(c["seqs"]):
        f = (0.6180339887 * s) % 1.0
        m = c["m"] if not c["ragged"] else max(1, round(c["m"] * (1.0 - f)))
        ctx = c["ctx"] if not c["ragged"] else round(c["ctx"] * (1.0 - 0.75 * ((0.4142135624 * s) % 1.0)))
        ms.append(m)
        kvs.append(ctx + m)
    return ms, kvs


def _draft_counts(c):
    if not c["ragged"]:
        return [c["drafts"]] * c["seqs"]
    return [max(1, round(c["drafts"] * (1.0 - (0.6180339887 * s) % 1.0))) for s in range(c["seqs"])]


def work(case):
    c = case
    if c["kind"] == "verify":
        n = sum(_draft_counts(c))
        rows = n + c["seqs"] + (n if c["draft_logits"] else 0)
        return {"bytes": rows * c["vocab"] * 4 + 16 * (n + c["seqs"]), "flops": 6 * rows * c["vocab"]}
    ms, kvs = _lengths(c)
    tokens, d, kvh = sum(ms), c["dim"], c["kv_heads"]
    row = d + 4 if c["cache"] == "i8" else 2 * d  # one K or V row of the cache
    if c["kind"] == "read":
        return {"bytes": tokens * kvh * 2 * (row + d * (2 if c["out"] == "f16" else 4)),
                "flops": tokens * kvh * 2 * d}
    if c["kind"] == "store":
        size = {"i8": 1, "f16": 2, "f32": 4}[c["x"]]
        # q, k and v in; q' out; the rows written, and read back
        b = tokens * ((c["heads"] + 2 * kvh) * d * size + c["heads"] * d * 2 + 2 * kvh * (2 * row + 2 * d))
        return {"bytes": b, "flops": tokens * (c["heads"] + 2 * kvh) * d * 8}
    seen = held = 0
    for m, kv in zip(ms, kvs):
        w = c["window"] or kv
        seen += sum(min(w, kv - m + i + 1) for i in range(m))
        held += min(kv, w + m - 1)
    return {"bytes": tokens * c["heads"] * d * 4 + held * kvh * 2 * row,
            "flops": 4 * seen * c["heads"] * d}


# ---- inputs -------------------------------------------------------------------------------------

class State:
    """What a serving program has in hand: tensors by name, the case, and (made on first use) the
    descriptors that it keeps for the batch."""

    def __init__(self, case, **tensors):
        self.case, self.kept = case, None
        self.__dict__.update(tensors)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 29)
    return g


def _rope(positions, dim):
    inv = 1e4 ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64, device="cuda") / dim)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return a.cos().float(), a.sin().float()


def _pool(g, c, pages):
    """One pool of pages as a running server holds it: [page][slot][head][dim], codes of rows that
    were quantised by their own largest value."""
    x = torch.randn((pages, c["page"], c["kv_heads"], c["dim"]), device="cuda", generator=g)
    if c["cache"] == "f16":
        return x.half(), None
    amax = x.abs().amax(-1)
    codes = torch.round(127.0 * x / amax[..., None]).to(torch.int8)
    return codes, (amax / 127.0).permute(0, 2, 1).contiguous()  # [page][head][slot]


def _inputs(g, c, n):
    """`n` heads of every token, as the projection left them."""
    x = torch.randn((c["tokens"], n, c["dim"]), device="cuda", generator=g)
    return torch.clamp(torch.round(15 * x), -128, 127).to(torch.int8) if c["x"] == "i8" else x.to(DTYPES[c["x"]])


def _prepare_verify(c, seed):
    g = _gen(seed)
    counts = _draft_counts(c)
    n, rows, v = sum(counts), sum(counts) + c["seqs"], c["vocab"]
    start = torch.tensor([0] + counts, device="cuda").cumsum(0)
    # a few plausible tokens over a wide floor; the drafter sees a blurred copy of the target
    logits = torch.randn((rows, v), device="cuda", generator=g) * 2.0
    top = torch.randint(0, v, (rows, 12), device="cuda", generator=g)
    logits.scatter_add_(1, top, 9.0 + 4.0 * torch.rand((rows, 12), device="cuda", generator=g))
    at = torch.arange(n, device="cuda") + torch.searchsorted(start[1:], torch.arange(n, device="cuda"), right=True)
    blurred = logits[at] + 0.5 * torch.randn((n, v), device="cuda", generator=g)
    noise = torch.rand((n, v), device="cuda", generator=g).clamp_min_(1e-7)
    if c["temperature"] > 0 and c["draft_logits"]:
        tokens = (blurred / c["temperature"] - torch.log(-torch.log(noise))).argmax(1)
    else:
        tokens = blurred.argmax(1)
    del noise
    return State(c, logits=logits, draft_logits=blurred if c["draft_logits"] else None,
                 draft_tokens=tokens.int(), draft_start=start.int(),
                 u=torch.rand(n, device="cuda", generator=g),
                 u_next=torch.rand(c["seqs"], device="cuda", generator=g),
                 tokens=torch.zeros((c["seqs"], c["drafts"] + 1), dtype=torch.int32, device="cuda"),
                 accepted=torch.zeros(c["seqs"], dtype=torch.int32, device="cuda"),
                 logprobs=torch.zeros((c["seqs"], c["drafts"] + 1), device="cuda"))


def prepare(case, seed):
    if case["kind"] == "verify":
        return _prepare_verify(case, seed)
    g = _gen(seed)
    ms, kvs = _lengths(case)
    c = dict(case, tokens=sum(ms), max_kv=max(kvs))
    need = [-(-kv // c["page"]) for kv in kvs]
    width, pages = max(need), sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).int()
    table = torch.full((c["seqs"], width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    k, k_scales = _pool(g, c, pages)
    v, v_scales = _pool(g, c, pages)
    d, t = c["dim"], c["tokens"]
    st = State(c, q_start=torch.tensor([0] + ms, device="cuda").cumsum(0).int(),
               kv_len=torch.tensor(kvs, device="cuda").int(), page_table=table, k=k, v=v,
               k_scales=k_scales, v_scales=v_scales)
    if c["kind"] == "attn":
        st.q = torch.randn((t, c["heads"], d), device="cuda", generator=g).half()
        st.scale = 1.5 / math.sqrt(d)
        st.out = torch.zeros((t, c["heads"], d), dtype=torch.float16, device="cuda")
        return st
    st.k_out = torch.zeros((t, c["kv_heads"], d), dtype=DTYPES[c["out"]], device="cuda")
    st.v_out = torch.zeros_like(st.k_out)
    if c["kind"] == "store":
        st.q_in, st.k_in, st.v_in = (_inputs(g, c, n) for n in (c["heads"], c["kv_heads"], c["kv_heads"]))
        st.x_scale = 0.1
        st.q_gain = st.k_gain = st.cos = st.sin = None
        if c["norm"]:
            st.q_gain = 0.15 + 0.2 * torch.rand(d, device="cuda", generator=g)
            st.k_gain = 0.15 + 0.2 * torch.rand(d, device="cuda", generator=g)
            st.cos, st.sin = _rope(c["max_kv"], d)
        st.q_out = torch.zeros((t, c["heads"], d), dtype=torch.float16, device="cuda")
    return st


# ---- the plain form: elementary torch operations ------------------------------------------------

def _rows(st):
    """Sequence and position of every row of the chunk."""
    start = st.q_start.long()
    row = torch.arange(st.case["tokens"], device="cuda")
    seq = torch.searchsorted(start[1:], row, right=True)
    i = row - start[seq]
    return seq, i, st.kv_len.long()[seq] - (start[1:] - start[:-1])[seq] + i


def _gather(st, pool, scales, seq, pos):
    """Cache rows at (seq, pos), any shape, as f32 [..., kv_heads, dim]."""
    page = st.page_table.long()[seq, pos // st.case["page"]]
    x = pool[page, pos % st.case["page"]].float()
    return x if scales is None else x * scales[page, :, pos % st.case["page"]][..., None]


def _plain_norm_rope(x, gain, cos, sin):
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    x = x if gain is None else x * gain
    if cos is None:
        return x
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_put(st, pool, scales, seq, pos, y):
    page, slot = st.page_table.long()[seq, pos // st.case["page"]], pos % st.case["page"]
    if scales is None:
        pool[page, slot] = y.half()
        return
    amax = y.abs().amax(-1)
    scales[page, :, slot] = amax / 127.0
    # 64 bits: a quotient next to a half goes to the code that the definition says
    pool[page, slot] = torch.round(127.0 * y.double() / amax.double()[..., None]).to(torch.int8)


def _plain_store(st):
    seq, _, pos = _rows(st)
    unit = st.x_scale if st.q_in.dtype == torch.int8 else 1.0
    q, k, v = (x.float() * unit for x in (st.q_in, st.k_in, st.v_in))
    if st.q_gain is not None:
        cos, sin = st.cos[pos][:, None], st.sin[pos][:, None]
        q = _plain_norm_rope(q, st.q_gain, cos, sin)
        k = _plain_norm_rope(k, st.k_gain, cos, sin)
        v = _plain_norm_rope(v, None, None, None)
    _plain_put(st, st.k, st.k_scales, seq, pos, k)
    _plain_put(st, st.v, st.v_scales, seq, pos, v)
    return {"q": q.half(), **_plain_read(st)}


def _plain_read(st):
    seq, _, pos = _rows(st)
    dt = st.k_out.dtype
    return {"k": _gather(st, st.k, st.k_scales, seq, pos).to(dt),
            "v": _gather(st, st.v, st.v_scales, seq, pos).to(dt)}


def _plain_attn(st):
    c = st.case
    s, m, kvh, d = c["seqs"], c["m"], c["kv_heads"], c["dim"]
    group, kv_len = c["heads"] // kvh, st.kv_len.long()
    start = st.q_start.long()
    count = start[1:] - start[:-1]
    key = torch.arange(c["max_kv"], device="cuda")
    there = key < kv_len[:, None]  # [s, keys]
    seq = torch.arange(s, device="cuda")[:, None]
    at = torch.where(there, key, 0)
    k = _gather(st, st.k, st.k_scales, seq, at).permute(0, 2, 1, 3).contiguous()  # [s, kvh, keys, d]
    v = _gather(st, st.v, st.v_scales, seq, at).permute(0, 2, 1, 3).contiguous()
    i = torch.arange(m, device="cuda")
    row = torch.minimum(start[:-1, None] + i, start[-1] - 1)  # [s, m]
    q = st.q[row].float().view(s, m, kvh, group, d).permute(0, 2, 1, 3, 4).reshape(s, kvh, m * group, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(s, kvh, m, group, -1) * st.scale
    pos = (kv_len - count)[:, None] + i  # [s, m]
    seen = there[:, None] & (key <= pos[..., None])
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(s, kvh, m * group, -1), v).view(s, kvh, m, group, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(s, m, c["heads"], d)
    return o[i < count[:, None]].half()


def _plain_verify(st):
    c = st.case
    start = st.draft_start.long()
    count = start[1:] - start[:-1]  # [s]
    slot = torch.arange(c["drafts"], device="cuda")
    real = slot < count[:, None]  # [s, drafts]
    at = torch.where(real, start[:-1, None] + slot, 0)
    seqs = torch.arange(c["seqs"], device="cuda")
    first = start[:-1] + seqs  # the target's first row of each sequence

    def capped(x):
        x = x.double()
        return torch.tanh(x / c["cap"]) * c["cap"] if c["cap"] else x

    def log_total(y):  # log of the running sum of exp(y), by rows
        top = y.amax(-1, keepdim=True)
        return top + torch.log(torch.exp(y - top).sum(-1, keepdim=True))

    y = capped(st.logits)
    z = y / (c["temperature"] or 1.0)
    logp = z - log_total(z)  # what is reported: log probabilities of what is sampled from
    draft = st.draft_tokens.long()[at]
    row = first[:, None] + torch.where(real, slot, 0)
    if c["temperature"] == 0:
        best = y.argmax(1)
        good = real & (best[row] == draft)
    else:
        p = torch.exp(logp)
        if st.draft_logits is not None:
            z = capped(st.draft_logits) / c["temperature"]
            q = torch.exp(z - log_total(z))
            qt = q[at, draft]
        else:
            qt = torch.ones_like(at, dtype=torch.float64)
        good = real & (st.u.double()[at] * qt < p[row, draft])
    accepted = good.int().cumprod(1).sum(1)  # [s]
    last = first + accepted
    refused = accepted < count
    if c["temperature"] == 0:
        token = best[last]
    else:
        w = p[last]
        j = torch.where(refused, start[:-1] + accepted, 0)
        if st.draft_logits is not None:
            less = q[j]
        else:
            less = torch.zeros_like(w).scatter_(1, st.draft_tokens.long()[j][:, None], 2.0)
        w = torch.where(refused[:, None], (w - less).clamp_min(0), w)
        run_ = w.cumsum(1)
        token = (run_ <= st.u_next.double()[:, None] * run_[:, -1:]).sum(1)
    out = torch.arange(c["drafts"] + 1, device="cuda")
    pad = torch.nn.functional.pad(draft, (0, 1))
    tokens = torch.where(out < accepted[:, None], pad, torch.where(out == accepted[:, None], token[:, None], -1))
    lp = logp[(first[:, None] + out).clamp_max(logp.shape[0] - 1), tokens.clamp_min(0)]
    return {"tokens": tokens.int(), "accepted": accepted.int(),
            "logprobs": torch.where(tokens >= 0, lp, 0.0).float()}


# ---- the framework's operators ------------------------------------------------------------------

def _serve():
    import os
    import sys
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemma4-webgpu-engine_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import g4serve
    return g4serve


def _keep(st):
    """The cache and batch descriptors of the program, and the workspace of its calls."""
    gs, c = _serve(), st.case
    if c["kind"] == "verify":
        n = gs.verify_workspace_bytes(c["seqs"], st.draft_tokens.numel(), c["vocab"])
        return gs, torch.empty(n, dtype=torch.uint8, device="cuda")
    pages = gs.KVPages(st.k, st.v, st.k_scales, st.v_scales)
    chunk = gs.Chunk(st.q_start, st.kv_len, st.page_table, tokens=c["tokens"], max_q=c["m"],
                     max_kv=c["max_kv"])
    ws = None
    if c["kind"] == "attn":
        n = gs.attention_chunk_workspace_bytes(pages, chunk, c["heads"], c["window"])
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    return gs, pages, chunk, ws


def _own(st):
    c = st.case
    if st.kept is None:
        st.kept = _keep(st)
    stream = torch.cuda.current_stream().cuda_stream or None
    if c["kind"] == "verify":
        gs, ws = st.kept
        gs.verify_drafts(st.logits, st.draft_logits, st.draft_tokens, st.draft_start, st.u, st.u_next,
                         st.tokens, st.accepted, st.logprobs, ws, cap=c["cap"],
                         temperature=c["temperature"], stream=stream)
        return {"tokens": st.tokens, "accepted": st.accepted, "logprobs": st.logprobs}
    gs, pages, chunk, ws = st.kept
    if c["kind"] == "attn":
        gs.attention_chunk(pages, chunk, st.q, st.out, ws, scale=st.scale, window=c["window"], stream=stream)
        return st.out
    if c["kind"] == "store":
        gs.paged_prologue(pages, chunk, st.q_in, st.k_in, st.v_in, st.q_out, q_gain=st.q_gain,
                          k_gain=st.k_gain, cos=st.cos, sin=st.sin, eps=EPS,
                          x_scale=st.x_scale, stream=stream)
    gs.kv_read(pages, chunk, st.k_out, st.v_out, stream=stream)
    out = {"k": st.k_out, "v": st.v_out}
    return {"q": st.q_out, **out} if c["kind"] == "store" else out


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attn, "store": _plain_store, "read": _plain_read,
            "verify": _plain_verify}[state.case["kind"]](state)


# ---- the definition in 64 bits ------------------------------------------------------------------

def _exact_rows(st, s):
    """Page and slot of every position of sequence s."""
    n, page = int(st.kv_len[s]), st.case["page"]
    p = torch.arange(n, device="cuda")
    return st.page_table[s].long()[p // page], p % page


def _exact_cache(st, pool, scales, s):
    page, slot = _exact_rows(st, s)
    x = pool[page, slot].double()
    return x if scales is None else x * scales.double()[page, :, slot][:, :, None]


def _exact_attn(st):
    c, out = st.case, []
    for s in range(c["seqs"]):
        a, b = int(st.q_start[s]), int(st.q_start[s + 1])
        k, v = _exact_cache(st, st.k, st.k_scales, s), _exact_cache(st, st.v, st.v_scales, s)
        n, m = k.shape[0], b - a
        behind = (n - m + torch.arange(m, device="cuda"))[:, None] - torch.arange(n, device="cuda")
        hidden = behind < 0
        if c["window"]:
            hidden |= behind >= c["window"]
        o = torch.empty((m, c["heads"], c["dim"]), dtype=torch.float64, device="cuda")
        for h in range(c["heads"]):
            kv = h // (c["heads"] // c["kv_heads"])
            logit = (st.q[a:b, h].double() @ k[:, kv].T) * st.scale
            weight = torch.softmax(logit.masked_fill(hidden, -math.inf), 1)
            o[:, h] = weight @ v[:, kv]
        out.append(o)
    return torch.cat(out)


def _exact_kv(st, x, gain, pos, norm, rope):
    """One of q, k, v after norm and rotation, f64 [tokens, heads, dim]."""
    y = x.double() * (float(torch.tensor(st.x_scale)) if x.dtype == torch.int8 else 1.0)
    if norm:
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / y.shape[-1] + EPS)
        if gain is not None:
            y = y * gain.double()
    if rope:
        h = y.shape[-1] // 2
        z = torch.complex(y[..., :h], y[..., h:]) * torch.complex(st.cos.double()[pos], st.sin.double()[pos])[:, None]
        y = torch.cat((z.real, z.imag), -1)
    return y


def _exact_held(st, y):
    """What the cache holds of y."""
    if st.k_scales is None:
        return y.half().double()
    amax = y.abs().amax(-1, keepdim=True)
    return torch.round(y * 127 / amax) * amax / 127


def _exact_store(st):
    c = st.case
    pos = torch.cat([torch.arange(int(kv) - int(b - a), int(kv), device="cuda") for a, b, kv in
                     zip(st.q_start[:-1], st.q_start[1:], st.kv_len)])
    n = c["norm"]
    return {"q": _exact_kv(st, st.q_in, st.q_gain, pos, n, n),
            "k": _exact_held(st, _exact_kv(st, st.k_in, st.k_gain, pos, n, n)),
            "v": _exact_held(st, _exact_kv(st, st.v_in, None, pos, n, False))}


def _exact_read(st):
    m = [int(b - a) for a, b in zip(st.q_start[:-1], st.q_start[1:])]
    return {"k": torch.cat([_exact_cache(st, st.k, st.k_scales, s)[-n:] for s, n in enumerate(m)]),
            "v": torch.cat([_exact_cache(st, st.v, st.v_scales, s)[-n:] for s, n in enumerate(m)])}


def _exact_verify(st):
    c = st.case
    tokens = torch.full((c["seqs"], c["drafts"] + 1), -1, dtype=torch.int32, device="cuda")
    accepted = torch.zeros(c["seqs"], dtype=torch.int32, device="cuda")
    lp = torch.zeros((c["seqs"], c["drafts"] + 1), dtype=torch.float64, device="cuda")

    def squash(x):
        x = x.double()
        return c["cap"] * torch.tanh(x / c["cap"]) if c["cap"] else x

    for s in range(c["seqs"]):
        a, b = int(st.draft_start[s]), int(st.draft_start[s + 1])
        for i in range(b - a + 1):
            y = squash(st.logits[a + s + i])
            t = int(st.draft_tokens[a + i]) if i < b - a else -1
            if c["temperature"] == 0:
                choice = int(y.argmax())
                keep = choice == t
            else:
                p = torch.softmax(y / c["temperature"], 0)
                if t >= 0:
                    q = torch.zeros_like(p)
                    if st.draft_logits is None:
                        q[t] = 1.0
                    else:
                        q = torch.softmax(squash(st.draft_logits[a + i]) / c["temperature"], 0)
                    keep = bool(st.u[a + i].double() * q[t] < p[t])
                    w = torch.relu(p - q)
                else:
                    keep, w = False, p
                if not keep:
                    r = torch.cumsum(w, 0)
                    choice = int((r <= st.u_next[s].double() * r[-1]).sum())
            tokens[s, i] = t if keep else choice
            lp[s, i] = torch.log_softmax(y / (c["temperature"] or 1.0), 0)[int(tokens[s, i])]
            if not keep:
                accepted[s] = i
                break
    return {"tokens": tokens, "accepted": accepted, "logprobs": lp}


def exact(case, seed):
    st = prepare(case, seed)
    return {"attn": _exact_attn, "store": _exact_store, "read": _exact_read,
            "verify": _exact_verify}[case["kind"]](st)
