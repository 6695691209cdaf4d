"""More serving operators, as measurable cases: the plan of a chunk (pages, block tables and slot maps from
the requests' lengths) and the release of pages, low-rank adapters of many requests beside a shared
projection, and sampling with temperature, top-k, top-p and min-p from given random numbers.

The listed sizes are the model of the tests and the benchmark (hidden 1536, feed-forward 6144, query
projection 2048, a vocabulary of 262144), plus odd ones.

A case is a dict with "kind" and that kind's sizes:
  plan     the rows and cached positions of every request to a chunk: q_start, kv_len, new pages from
           the free list into the block table, and each row's position, cache slot and adapter
  release  pages of finished requests, or behind a window, back to the free list
  adapter  base + scale * (x A^T) B^T, with the A and B of each row's request
  sample   one token a row; "mode" says which filters the rows have ("mixed": different ones)
Lengths, ids and filters of a batch follow a fixed rule; values are random.
"""
from __future__ import annotations

import math

import torch

own = False

HIDDEN, FFN, VOCAB = 1536, 6144, 262144
DTYPES = {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8}
# temperature, top-k, top-p, min-p (0 or 1: off)
FILTERS = {
    "greedy": (0.0, 0, 1.0, 0.0),
    "top": (0.8, 64, 0.95, 0.0),
    "topk": (1.3, 1000, 1.0, 0.0),
    "nucleus": (1.0, 0, 0.95, 0.0),
    "minp": (1.2, 0, 1.0, 0.05),
    "all": (0.9, 200, 0.9, 0.01),
    "free": (1.0, 0, 1.0, 0.0),
}
MIX = ("top", "nucleus", "greedy", "minp", "topk", "free", "all")


# ---- the cases ----------------------------------------------------------------------------------

def _plan(name, **kw):
    return dict({"name": name, "kind": "plan", "seqs": 1, "m": 1, "ctx": 0, "page": 16, "spare": 64}, **kw)


def _adapter(name, **kw):
    return dict({"name": name, "kind": "adapter", "tokens": 1, "adapters": 8, "seqs": 1, "k": HIDDEN, "n": 2048,
                 "rank": 16, "x": "i8", "base": "f32", "out": "f32"}, **kw)


def _sample(name, **kw):
    return dict({"name": name, "kind": "sample", "rows": 1, "vocab": VOCAB, "cap": 30.0, "mode": "top",
                 "shape": "peaked"}, **kw)


def listed():
    return [
        # A step of a busy server: 256 requests, one to eight rows each, some of which open a page.
        _plan("plan_b256", seqs=256, m=8, ctx=4088),
        # 64 new prompts of up to 2048 tokens at once, in small pages.
        _plan("plan_prompts", seqs=64, m=2048, page=8),
        # The pages of 16 finished requests of up to 4096 positions.
        {"name": "release_b16", "kind": "release", "seqs": 16, "width": 256, "page": 16, "part": False},
        # What a sliding window leaves behind in 1000 requests: a page of most of them.
        {"name": "release_window", "kind": "release", "seqs": 1000, "width": 1024, "page": 16, "part": True},
        # One decoded token of one request, on the query projection.
        _adapter("adapter_b1"),
        # A decode batch: 64 requests with 16 adapters between them, on a feed-forward projection.
        _adapter("adapter_b64", tokens=64, seqs=64, adapters=16, n=FFN, rank=32),
        # A few prompts of odd lengths, f32 activations, a narrow projection.
        _adapter("adapter_m509", tokens=509, seqs=5, adapters=8, k=2048, n=250, rank=24, x="f32", out="f16"),
        # Long prompts with three adapters: the projection down, f16 activations, f16 out.
        _adapter("adapter_m2048", tokens=2048, seqs=3, adapters=4, k=FFN, n=HIDDEN, rank=64, x="f16", out="f16"),
        # The next token of one request.
        _sample("sample_b1"),
        # A decode batch whose requests ask for different filters.
        _sample("sample_b32", rows=32, mode="mixed"),
        # Another vocabulary, flat rows: a nucleus of thousands of tokens.
        _sample("sample_b64_odd", rows=64, vocab=32003, cap=0.0, mode="nucleus", shape="flat"),
        # The largest batch.
        _sample("sample_b256", rows=256, mode="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "release", "adapter", "adapter", "adapter", "sample", "sample", "sample"])
    page = rng.choice([8, 16, 32, 64])
    while True:
        if kind == "plan":
            c = {"kind": kind, "seqs": _log(rng, 1, 1024), "m": _log(rng, 1, 4096), "ctx": _log(rng, 1, 16384) - 1,
                 "page": page, "spare": rng.choice([0, 64, 1000])}
            if c["seqs"] * c["m"] <= 1 << 17 and c["seqs"] * (c["ctx"] + c["m"]) <= 1 << 22:
                return c
        elif kind == "release":
            c = {"kind": kind, "seqs": _log(rng, 1, 1024), "width": _log(rng, 1, 2048), "page": page,
                 "part": rng.random() < 0.5}
            if c["seqs"] * c["width"] <= 1 << 20:
                return c
        elif kind == "adapter":
            c = {"kind": kind, "tokens": _log(rng, 1, 4096), "adapters": _log(rng, 1, 64),
                 "k": 8 * _log(rng, 16, FFN // 8), "n": _log(rng, 60, FFN), "rank": 8 * rng.randint(1, 8),
                 "x": rng.choice(["i8", "f16", "f32"]), "base": rng.choice(["f32", "f32", "f16", "i8"]),
                 "out": rng.choice(["f32", "f16"])}
            c["seqs"] = min(c["tokens"], _log(rng, 1, 256))
            if c["tokens"] * (c["k"] + c["n"]) <= 1 << 23 and c["tokens"] * c["adapters"] <= 1 << 15:
                return c
        else:
            c = {"kind": kind, "rows": _log(rng, 1, 256), "vocab": _log(rng, 1000, VOCAB),
                 "cap": rng.choice([0.0, 30.0]), "mode": rng.choice(["mixed", *MIX]),
                 "shape": rng.choice(["peaked", "peaked", "flat"])}
            if c["rows"] * c["vocab"] <= 1 << 25:
                return c


def _golden(s):
    return (0.6180339887 * s) % 1.0


def _lengths(c):
    """Rows and cached positions of each request of a plan: the same for every seed."""
    s = range(c["seqs"])
    rows = [max(1, round(c["m"] * (1.0 - _golden(i)))) for i in s]
    return rows, [round(c["ctx"] * (1.0 - 0.75 * ((0.4142135624 * i) % 1.0))) for i in s]


def _ranges(c):
    """First and last page to release of each request."""
    out = []
    for i in range(c["seqs"]):
        if c["part"]:
            first = int(_golden(i) * (c["width"] - 1))
            out.append((first, min(c["width"], first + (0 if i % 5 == 4 else 1))))
        else:
            out.append((0, max(1, round(c["width"] * (1.0 - 0.75 * _golden(i))))))
    return out


def _ids(c):
    """The adapter of each row: runs of rows, one a request; of more than two requests one has none."""
    cuts = [round(c["tokens"] * i / c["seqs"]) for i in range(c["seqs"] + 1)]
    ids = []
    for i in range(c["seqs"]):
        a = -1 if c["seqs"] > 2 and i == 1 else int(_golden(i) * c["adapters"])
        ids += [a] * (cuts[i + 1] - cuts[i])
    return ids


def _ranks(c):
    """The rank of each adapter: most have the pool's."""
    return [c["rank"] if i % 3 != 2 else max(1, c["rank"] * 3 // 4) for i in range(c["adapters"])]


def work(case):
    c = case
    if c["kind"] == "sample":
        return {"bytes": c["rows"] * (c["vocab"] * 4 + 32), "flops": 4 * c["rows"] * c["vocab"]}
    if c["kind"] == "release":
        pages = sum(b - a for a, b in _ranges(c))
        return {"bytes": 8 * pages + 8 * c["seqs"], "flops": pages}
    if c["kind"] == "plan":
        rows, cached = _lengths(c)
        pages = sum(-(-(k + n) // c["page"]) + (-k // c["page"]) for n, k in zip(rows, cached))
        return {"bytes": 12 * sum(rows) + 8 * pages + 32 * c["seqs"], "flops": sum(rows)}
    size = {"i8": 1, "f16": 2, "f32": 4}
    ids, ranks = _ids(c), _ranks(c)
    t = sum(i >= 0 for i in ids)
    b = t * c["k"] * size[c["x"]] + c["tokens"] * c["n"] * (size[c["base"]] + size[c["out"]])
    b += sum(ranks[a] * (c["k"] + c["n"]) * 2 for a in set(ids) if a >= 0)
    return {"bytes": b, "flops": sum(2 * ranks[a] * (c["k"] + c["n"]) for a in ids if a >= 0)}


# ---- inputs -------------------------------------------------------------------------------------

class State:
    """What a serving program has in hand: tensors by name, the case, and (made on first use) the
    descriptors, workspaces and row groups that it keeps for the batch."""

    def __init__(self, case, **tensors):
        self.case, self.kept = case, None
        self.__dict__.update(tensors)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 53)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _new(*shape):
    return torch.zeros(shape, dtype=torch.int32, device="cuda")


def _prepare_plan(c, g):
    rows, cached = _lengths(c)
    held = [-(-k // c["page"]) for k in cached]
    width = max(-(-(k + n) // c["page"]) for n, k in zip(rows, cached))
    new = sum(-(-(k + n) // c["page"]) - h for n, k, h in zip(rows, cached, held))
    pages = sum(held) + new + c["spare"]
    order = torch.randperm(pages, device="cuda", generator=g).int()
    col = torch.arange(width, device="cuda")
    mine = col < _ints(held)[:, None]
    table = torch.full((c["seqs"], width), -1, dtype=torch.int32, device="cuda")
    table[mine] = order[:sum(held)]
    free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    free[:new + c["spare"]] = order[sum(held):]
    tokens = sum(rows) + 3
    adapter = torch.randint(-1, 16, (c["seqs"],), device="cuda", generator=g).int()
    return State(dict(c, tokens=tokens, pages=pages, max_kv=max(a + b for a, b in zip(rows, cached))),
                 rows=_ints(rows), cached=_ints(cached), held=_ints(held), free=free,
                 count=_ints([new + c["spare"]]), table=table, adapter=adapter, q_start=_new(c["seqs"] + 1),
                 kv_len=_new(c["seqs"]), held_out=_new(c["seqs"]), left=_new(1), served=_new(1), row_pos=_new(tokens),
                 row_slot=_new(tokens), row_adapter=_new(tokens), last_row=_new(c["seqs"]))


def _prepare_release(c, g):
    ranges = _ranges(c)
    pages = c["seqs"] * c["width"]
    order = torch.randperm(pages + 100, device="cuda", generator=g).int()
    free = torch.full((pages + 100,), -1, dtype=torch.int32, device="cuda")
    free[:100] = order[pages:]
    return State(dict(c, pages=pages + 100), table=order[:pages].view(c["seqs"], c["width"]).clone(), free=free,
                 count=_ints([100]), first=_ints([a for a, _ in ranges]), last=_ints([b for _, b in ranges]),
                 left=_new(1))


def _values(g, kind, shape):
    x = torch.randn(shape, device="cuda", generator=g)
    return torch.clamp(torch.round(30 * x), -128, 127).to(torch.int8) if kind == "i8" else x.to(DTYPES[kind])


def _prepare_adapter(c, g):
    t, k, n, r, m = c["tokens"], c["k"], c["n"], c["rank"], c["adapters"]
    a = torch.randn((m, r, k), device="cuda", generator=g).mul_(k ** -0.5).half()
    b = torch.randn((m, n, r), device="cuda", generator=g).mul_(0.1).half()
    ranks = _ints(_ranks(c))
    behind = torch.arange(r, device="cuda") >= ranks[:, None]
    a[behind] = 0  # a smaller adapter leaves the rest of its rows empty
    b.masked_fill_(behind[:, None], 0)
    return State(c, x=_values(g, c["x"], (t, k)), base=_values(g, c["base"], (t, n)), a=a, b=b, ranks=ranks,
                 scale=0.5 + torch.rand(m, device="cuda", generator=g), ids=_ints(_ids(c)),
                 x_scale=0.04 if c["x"] == "i8" else 1.0, base_scale=0.05 if c["base"] == "i8" else 1.0,
                 out=torch.zeros((t, n), dtype=DTYPES[c["out"]], device="cuda"))


def _prepare_sample(c, g):
    n, v = c["rows"], c["vocab"]
    if c["shape"] == "flat":
        logits = torch.randn((n, v), device="cuda", generator=g).mul_(1.5)
    else:  # a few plausible tokens, of different weight in each row, over a floor
        logits = torch.randn((n, v), device="cuda", generator=g).mul_(2.0)
        top = torch.randint(0, v, (n, 40), device="cuda", generator=g)
        best = 12.0 + 6.0 * torch.rand((n, 1), device="cuda", generator=g)
        logits.scatter_add_(1, top, best * (0.6 + 0.4 * torch.rand((n, 40), device="cuda", generator=g)))
    modes = [MIX[i % len(MIX)] if c["mode"] == "mixed" else c["mode"] for i in range(n)]
    t, k, p, m = zip(*(FILTERS[x] for x in modes))

    def given(values, off, dtype):  # a program whose requests never ask for a filter has no array for it
        return None if all(x == off for x in values) else torch.tensor(values, dtype=dtype, device="cuda")

    return State(c, logits=logits, u=torch.rand(n, device="cuda", generator=g),
                 temperature=given(t, 1.0, torch.float32), top_k=given(k, 0, torch.int32),
                 top_p=given(p, 1.0, torch.float32), min_p=given(m, 0.0, torch.float32), tokens=_new(n),
                 logprobs=torch.zeros(n, device="cuda"))


def prepare(case, seed):
    return {"plan": _prepare_plan, "release": _prepare_release, "adapter": _prepare_adapter,
            "sample": _prepare_sample}[case["kind"]](case, _gen(seed))


# ---- the plain form: elementary torch operations ------------------------------------------------

def _before(x):
    """Exclusive running sums."""
    return torch.nn.functional.pad(x.cumsum(0), (1, 0))


def _plan_outputs(st):
    return {n: getattr(st, n) for n in ("q_start", "kv_len", "held_out", "left", "served", "table", "row_pos",
                                        "row_slot", "row_adapter", "last_row")}


def _plain_plan(st):
    c, page = st.case, st.case["page"]
    cached = st.cached.long().clamp(0, c["max_kv"])
    rows = torch.minimum(st.rows.long().clamp(0, c["m"]), c["max_kv"] - cached)
    held = st.held.long()
    need = torch.where(rows > 0, ((cached + rows + page - 1) // page - held).clamp_min(0), 0)
    count = st.count.long()
    fits = (rows.cumsum(0) <= c["tokens"]) & (need.cumsum(0) <= count)
    fits = fits.long().cumprod(0)
    rows, need = rows * fits, need * fits
    start, pages = _before(rows), _before(need)
    left = count - pages[-1]
    j = torch.arange(st.table.shape[1], device="cuda") - held[:, None]
    new = (j >= 0) & (j < need[:, None])
    at = torch.where(new, left + pages[:-1, None] + j, 0)
    st.table.copy_(torch.where(new, st.free[at], st.table))
    t = torch.arange(c["tokens"], device="cuda")
    seq = torch.searchsorted(start[1:], t, right=True)
    real = seq < c["seqs"]
    seq = torch.where(real, seq, 0)
    pos = torch.where(real, cached[seq] + t - start[seq], 0)
    entry = st.table[seq, pos // page].long()
    there = real & (entry >= 0) & (entry < c["pages"])
    st.q_start.copy_(start)
    st.kv_len.copy_(cached + rows)
    st.held_out.copy_(held + need)
    st.left.copy_(left)
    st.served.copy_(fits.sum())
    st.row_pos.copy_(torch.where(real, pos, -1))
    st.row_slot.copy_(torch.where(there, entry * page + pos % page, -1))
    st.row_adapter.copy_(torch.where(real, st.adapter[seq], -2))
    st.last_row.copy_(torch.where(rows > 0, start[1:] - 1, -1))
    return _plan_outputs(st)


def _plain_release(st):
    width = st.case["width"]
    first, last = st.first.long().clamp(0, width), st.last.long().clamp(0, width)
    n = (last - first).clamp_min(0)
    col = torch.arange(width, device="cuda")
    going = (col >= first[:, None]) & (col < last[:, None])
    at = st.count.long() + _before(n)[:-1, None] + col - first[:, None]
    # what stays goes to a place behind the list
    room = torch.cat((st.free, st.free.new_zeros(1)))
    room.scatter_(0, torch.where(going, at, st.free.numel()).view(-1), st.table.view(-1))
    st.free.copy_(room[:-1])
    st.left.copy_(st.count + n.sum())
    return {"free": st.free, "left": st.left}


def _plain_adapter(st):
    c = st.case
    x, ids = st.x.float() * st.x_scale, st.ids.long()
    out = st.base.float() * st.base_scale
    if c["tokens"] * c["rank"] * (c["k"] + c["n"]) <= 1 << 27:  # each row's own matrices
        at = ids.clamp_min(0)
        h = torch.bmm(st.a[at].float(), x[:, :, None])
        y = torch.bmm(st.b[at].float(), h)[:, :, 0] * st.scale[at][:, None]
        return (out + torch.where(ids[:, None] >= 0, y, 0.0)).to(st.out.dtype)
    for i in range(c["adapters"]):
        y = (x @ st.a[i].float().T) @ st.b[i].float().T * st.scale[i]
        out = torch.where(ids[:, None] == i, out + y, out)
    return out.to(st.out.dtype)


def _plain_sample(st):
    c = st.case
    n, v = c["rows"], c["vocab"]

    def per_row(x, off):
        return torch.full((n, 1), off, device="cuda", dtype=torch.float64) if x is None else x.double()[:, None]

    t, k, p, m = per_row(st.temperature, 1.0), per_row(st.top_k, 0), per_row(st.top_p, 1.0), per_row(st.min_p, 0.0)
    x, token = torch.sort(torch.where(st.logits.isnan(), -math.inf, st.logits), dim=1, descending=True, stable=True)
    # 64 bits: the drawn token is one of thousands next to each other in a running sum
    y = torch.tanh(x.double() / c["cap"]) * c["cap"] if c["cap"] else x.double()
    z = (y - y[:, :1]) / torch.where(t > 0, t, 1.0)
    w = torch.exp(z)
    rank = torch.arange(v, device="cuda")
    total = w.sum(1, keepdim=True)
    kept = torch.where((k <= 0) | (rank < k), w, 0.0)
    run_ = kept.cumsum(1)
    low = torch.nn.functional.pad(run_[:, :-1], (1, 0)) < p * run_[:, -1:]
    kept = torch.where((p >= 1) | low | (rank == 0), kept, 0.0)
    kept = torch.where((m <= 0) | (z >= torch.log(m.clamp(1e-300, 1.0))), kept, 0.0)
    del run_, low, w, y, x
    by_token = torch.zeros_like(kept).scatter_(1, token, kept).cumsum(1)
    del kept
    drawn = (by_token <= st.u.double()[:, None] * by_token[:, -1:]).sum(1, keepdim=True)
    drawn = torch.where(t > 0, drawn.clamp_max(v - 1), token[:, :1])
    # the drawn token's place in the order gives its log weight
    place = (token == drawn).int().argmax(1, keepdim=True)
    return {"tokens": drawn[:, 0].int(), "logprobs": (z.gather(1, place) - torch.log(total))[:, 0].float()}


# ---- the framework's operators ------------------------------------------------------------------

def _serve():
    import os
    import sys
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemma4-webgpu-engine_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import g4serve
    return g4serve


def _room(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def _keep(st, stream):
    """The descriptors and workspaces of the program, and the batch's rows grouped by adapter (one
    grouping serves every projection of every layer of a step)."""
    gs, c = _serve(), st.case
    if c["kind"] in ("plan", "release"):
        return gs, gs.FreePages(st.free, st.count, num_pages=c["pages"], page_size=c["page"])
    if c["kind"] == "sample":
        return gs, _room(gs.sample_workspace_bytes(c["rows"], c["vocab"]))
    adapters = gs.Adapters(st.a, st.b, scales=st.scale, ranks=st.ranks)
    groups = _room(gs.adapter_groups_bytes(c["tokens"], c["adapters"]))
    gs.adapter_groups(st.ids, groups, adapters=c["adapters"], stream=stream)
    return gs, adapters, groups, _room(gs.adapter_workspace_bytes(adapters, c["tokens"]))


def _own(st):
    c = st.case
    stream = torch.cuda.current_stream().cuda_stream or None
    if st.kept is None:
        st.kept = _keep(st, stream)
    gs = st.kept[0]
    if c["kind"] == "plan":
        gs.plan_chunk(st.kept[1], st.cached, st.rows, st.table, st.q_start, st.kv_len, st.left, st.served,
                      tokens=c["tokens"], max_q=c["m"], max_kv=c["max_kv"], held=st.held, held_out=st.held_out,
                      seq_adapter=st.adapter, row_pos=st.row_pos, row_slot=st.row_slot,
                      row_adapter=st.row_adapter, last_row=st.last_row, stream=stream)
        return _plan_outputs(st)
    if c["kind"] == "release":
        gs.release_pages(st.kept[1], st.table, st.first, st.last, st.left, stream=stream)
        return {"free": st.free, "left": st.left}
    if c["kind"] == "sample":
        gs.sample_tokens(st.logits, st.u, st.tokens, st.logprobs, st.kept[1], temperature=st.temperature,
                         top_k=st.top_k, top_p=st.top_p, min_p=st.min_p, cap=c["cap"], stream=stream)
        return {"tokens": st.tokens, "logprobs": st.logprobs}
    _, adapters, groups, ws = st.kept
    gs.adapter_linear(adapters, groups, st.x, st.base, st.out, ws, x_scale=st.x_scale, base_scale=st.base_scale,
                      stream=stream)
    return st.out


def run(state):
    if own:
        return _own(state)
    return {"plan": _plain_plan, "release": _plain_release, "adapter": _plain_adapter,
            "sample": _plain_sample}[state.case["kind"]](state)


# ---- the definition in 64 bits ------------------------------------------------------------------

def _exact_plan(st):
    c, page = st.case, st.case["page"]
    cached, rows, held, table, free, adapter = (x.tolist() for x in (st.cached, st.rows, st.held, st.table, st.free,
                                                                     st.adapter))
    wants = [max(0, -(-(k + n) // page) - h) if n else 0 for k, n, h in zip(cached, rows, held)]
    count, served, used, filled = int(st.count), 0, 0, 0
    for n, w in zip(rows, wants):
        if filled + n > c["tokens"] or used + w > count:
            break
        served, used, filled = served + 1, used + w, filled + n
    pages = iter(free[count - used:count])
    out = {"q_start": [0], "kv_len": [], "held_out": [], "left": [count - used], "served": [served], "table": table,
           "row_pos": [], "row_slot": [], "row_adapter": [], "last_row": []}
    for s in range(c["seqs"]):
        n, w = (rows[s], wants[s]) if s < served else (0, 0)
        for i in range(w):
            table[s][held[s] + i] = next(pages)
        for p in range(cached[s], cached[s] + n):
            entry = table[s][p // page]
            out["row_pos"].append(p)
            out["row_slot"].append(entry * page + p % page if 0 <= entry < c["pages"] else -1)
            out["row_adapter"].append(adapter[s])
        out["kv_len"].append(cached[s] + n)
        out["held_out"].append(held[s] + w)
        out["q_start"].append(out["q_start"][-1] + n)
        out["last_row"].append(out["q_start"][-1] - 1 if n else -1)
    for name, value in (("row_pos", -1), ("row_slot", -1), ("row_adapter", -2)):
        out[name] += [value] * (c["tokens"] - len(out[name]))
    return {n: _ints(v) for n, v in out.items()}


def _exact_release(st):
    free, n = st.free.tolist(), int(st.count)
    for row, a, b in zip(st.table.tolist(), st.first.tolist(), st.last.tolist()):
        free[n:n + b - a] = row[a:b]
        n += b - a
    return {"free": _ints(free), "left": _ints([n])}


def _exact_adapter(st):
    out = st.base.double() * (float(torch.tensor(st.base_scale)) if st.base.dtype == torch.int8 else 1.0)
    unit = float(torch.tensor(st.x_scale)) if st.x.dtype == torch.int8 else 1.0
    for i, rank in enumerate(st.ranks.tolist()):
        rows = (st.ids == i).nonzero()[:, 0]
        h = unit * torch.matmul(st.x[rows].double(), st.a[i, :rank].double().T.contiguous())
        out[rows] += st.scale[i].double() * torch.matmul(h, st.b[i, :, :rank].double().T.contiguous())
    return out


def _exact_sample(st):
    c = st.case
    tokens, logprobs = [], []
    for i in range(c["rows"]):
        t, k, p, m = (float(x[i]) if x is not None else off for x, off in
                      ((st.temperature, 1.0), (st.top_k, 0), (st.top_p, 1.0), (st.min_p, 0.0)))
        x = st.logits[i].double()
        y = c["cap"] * torch.tanh(x / c["cap"]) if c["cap"] else x
        logp = torch.log_softmax(y / (t or 1.0), 0)
        if t == 0:
            choice = int((x == x.max()).nonzero()[0])
        else:
            order = torch.sort(-x, stable=True).indices
            if k > 0:
                order = order[:int(k)]
            q = torch.softmax(logp[order], 0)
            if p < 1:
                order = order[:1 + int((q.cumsum(0)[:-1] < p).sum())]
            order = order[logp[order] - logp.max() >= math.log(m)] if m > 0 else order
            order = order.sort().values
            total = torch.exp(logp[order]).cumsum(0)
            choice = int(order[int((total <= float(st.u[i]) * total[-1]).sum())])
        tokens.append(choice)
        logprobs.append(logp[choice])
    return {"tokens": _ints(tokens), "logprobs": torch.stack(logprobs)}


def exact(case, seed):
    st = prepare(case, seed)
    return {"plan": _exact_plan, "release": _exact_release, "adapter": _exact_adapter,
            "sample": _exact_sample}[case["kind"]](st)
