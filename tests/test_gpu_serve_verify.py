"""Verification of drafted tokens, against the sampling rule in 64 bits."""
import numpy as np
import pytest

import g4serve as gs
import g4w8a8 as g4
from servecases import dev

pytestmark = pytest.mark.gpu


def softcap(x, cap):
    x = x.astype(np.float64)
    return cap * np.tanh(x / cap) if cap else x


def probabilities(x, cap, t):
    """p and log p of rows; a NaN has no weight; rows without weight: zeros."""
    y = softcap(x, cap)
    y = np.where(np.isnan(x), -np.inf, y) / (t or 1.0)
    top = y.max(-1, keepdims=True)
    with np.errstate(invalid="ignore"):
        z = np.where(y == top, 0.0, y - np.where(np.isfinite(top), top, 0))
    z = np.where(top == -np.inf, -np.inf, np.where((top == np.inf) & (y != top), -np.inf, z))
    w = np.exp(z)
    s = w.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        return w / np.where(s == 0, 1, s), z - np.log(s)


def verify(logits, draft_logits, drafts, start, u, u_next, max_drafts, cap, t):
    """(tokens, accepted, logprobs, margin): margin is how near a decision came to going the other way: of a
    draft in parts of its probability, of a draw in parts of the total."""
    t = float(np.float32(t))
    seqs = len(start) - 1
    tokens = np.full((seqs, max_drafts + 1), -1, np.int32)
    lp = np.zeros((seqs, max_drafts + 1))
    accepted = np.zeros(seqs, np.int32)
    margin = 1.0
    vocab = logits.shape[1]
    for s in range(seqs):
        a, n = start[s], min(start[s + 1] - start[s], max_drafts)
        for i in range(n + 1):
            row = logits[a + s + i]
            p, logp = probabilities(row, cap, t)
            choice = int(np.argmax(np.where(np.isnan(row), -np.inf, row))) if p.any() else -1
            if i < n:
                d = int(drafts[a + i])
                inside = 0 <= d < vocab
                if t == 0:
                    take = choice == d and inside
                else:
                    q = np.zeros(vocab)
                    if draft_logits is not None:
                        q, _ = probabilities(draft_logits[a + i], cap, t)
                    elif inside:
                        q[d] = 1.0
                    take = inside and float(u[a + i]) * q[d] < p[d]
                    if inside and (q[d] or p[d]):  # 0 < 0 is decided exactly
                        margin = min(margin, abs(float(u[a + i]) * q[d] - p[d]) / max(q[d], p[d]))
                if take:
                    tokens[s, i], lp[s, i] = d, logp[d]
                    accepted[s] = i + 1
                    continue
            if t:
                w = np.maximum(p - q, 0) if i < n else p
                if not w.any():
                    w = p
                run = np.cumsum(w)
                if run[-1] > 0:
                    target = float(u_next[s]) * run[-1]
                    choice = int((run <= target).sum())
                    if target > 0:  # a running sum of 0 is exact
                        margin = min(margin, np.abs(run - target).min() / run[-1])
            tokens[s, i] = choice
            lp[s, i] = logp[choice] if choice >= 0 else 0.0
            break
    return tokens, accepted, lp, margin


def run(logits, draft_logits, drafts, start, u, u_next, max_drafts, cap, t, with_lp=True):
    seqs = len(start) - 1
    out = dev(np.full((seqs, max_drafts + 1), 77, np.int32)), dev(np.full(seqs, 77, np.int32))
    lp = dev(np.full((seqs, max_drafts + 1), 77, np.float32)) if with_lp else None
    ws = g4.DeviceBuffer(gs.verify_workspace_bytes(seqs, len(drafts), logits.shape[1]))
    ws.fill(0xFF)
    gs.verify_drafts(dev(logits), None if draft_logits is None else dev(draft_logits), dev(drafts), dev(start),
                     None if t == 0 else dev(u), None if t == 0 else dev(u_next), *out, lp, ws, cap=cap, temperature=t)
    return out[0].download(), out[1].download(), lp.download() if with_lp else None


def case(counts, vocab, seed, blur=0.7, spread=3.0):
    r = np.random.default_rng(seed)
    n = sum(counts)
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    logits = (spread * r.standard_normal((n + len(counts), vocab))).astype(np.float32)
    at = np.concatenate([start[s] + s + np.arange(c) for s, c in enumerate(counts)]).astype(int) if n else np.zeros(0, int)
    draft_logits = (logits[at] + blur * r.standard_normal((n, vocab))).astype(np.float32)
    drafts = np.array([np.argmax(x + r.gumbel(size=vocab)) for x in draft_logits], np.int32)
    return logits, draft_logits, drafts, start, r.random(n).astype(np.float32), r.random(len(counts)).astype(np.float32)


# Weights of relative error 2^-39 and 64-bit sums: a decision whose margin is over 2^-34 of the total is the
# same.
# f32 log probabilities: half a step of the value, and 2^-38 before it.
def check(c, max_drafts, cap, t, drafter=True):
    logits, dl, drafts, start, u, un = c
    dl = dl if drafter else None
    want = verify(logits, dl, drafts, start, u, un, max_drafts, cap, t)
    assert t == 0 or want[3] > 2.0 ** -32  # the inputs decide, not the last bits
    got = run(logits, dl, drafts, start, u, un, max_drafts, cap, t)
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], want[0])
    assert (np.abs(got[2] - want[2]) <= np.abs(want[2]) * 2.0 ** -24 * 1.01 + 2.0 ** -36).all()
    return got


@pytest.mark.parametrize("drafter", [True, False], ids=["logits", "tokens"])
@pytest.mark.parametrize("t", [0.0, 0.3, 1.0, 1.7])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 8192, 8193, 30001])
def test_rule(gpu, vocab, t, drafter):
    for seed, cap in ((1, 0.0), (2, 30.0), (3, 2.0)):
        check(case([4, 1, 0, 7, 2], vocab, seed), 7, cap, t, drafter)


def test_full_vocabulary(gpu):
    taken = 0
    for seed in range(4):
        got = check(case([4, 3, 5], 262144, seed), 5, 30.0 if seed % 2 else 0.0, 0.9)
        taken += int(got[1].sum())
    assert 0 < taken < 48


def test_flat_distribution(gpu):
    """Every token nearly alike: the drawn one hangs on sums of 262144 terms."""
    for seed in range(3):
        check(case([2] * 3, 262144, seed, blur=0.01, spread=0.05), 2, 0.0, 1.0)


def test_many_sequences_and_the_longest_drafts(gpu):
    check(case([63, 0, 17, 63], 512, 5, blur=0.05), 63, 0.0, 1.0)
    check(case([1] * 200, 700, 6), 1, 0.0, 1.0)


def test_counts_past_max_drafts_are_cut(gpu):
    check(case([5, 2, 9], 300, 8, blur=0.0), 3, 0.0, 1.0)


def test_no_drafts_is_plain_sampling(gpu):
    c = case([0, 0, 0], 5000, 9)
    got = check(c, 0, 30.0, 1.0)
    assert (got[1] == 0).all() and (got[0] >= 0).all()
    check(c, 2, 0.0, 0.0)


def test_equal_models_take_everything(gpu):
    """p = q: every draft is taken, whatever u is; one that the drafter could not have drawn is refused and
    the residual is nowhere positive, so the draw is from p."""
    logits, _, drafts, start, u, un = case([4, 4], 9000, 10, blur=0.0)
    at = np.array([0, 1, 2, 3, 5, 6, 7, 8])
    u[:] = np.float32(1 - 2.0 ** -24)
    got = check((logits, logits[at].copy(), drafts, start, u, un), 4, 0.0, 1.0)
    assert (got[1] == 4).all()
    logits[at[5], 123] = -np.inf
    drafts[5] = 123
    got = check((logits, logits[at].copy(), drafts, start, u, un), 4, 0.0, 1.0)
    assert got[1].tolist() == [4, 1] and got[0][1, 1] != 123


def test_ends_of_the_random_numbers(gpu):
    """u_next 0 draws the first token of any weight, the largest u_next the last ones; u 0 takes any draft
    of positive probability."""
    logits, dl, drafts, start, u, un = case([3, 3], 20000, 12)
    logits[:, :100] = -np.inf
    dl[:, :50] = -np.inf
    drafts = np.maximum(drafts, 150)
    u[:] = 0
    for x in (0.0, 1 - 2.0 ** -24):
        un[:] = x
        got = check((logits, dl, drafts, start, u, un), 3, 0.0, 1.0)
        assert (got[1] == 3).all()
    un[:] = 0
    assert (run(logits, dl, drafts, start, u, un, 3, 0.0, 1.0)[0][:, 3] == 100).all()
    logits[[3, 7], 8500] = np.inf  # the others weigh nothing beside it
    assert (run(logits, dl, drafts, start, u, un, 3, 0.0, 1.0)[0][:, 3] == 8500).all()
    logits[[3, 7], 8500], logits[[3, 7], 100:8500] = 3000, -3000
    assert (run(logits, dl, drafts, start, u, un, 3, 0.0, 1.0)[0][:, 3] == 8500).all()


def test_nan_infinite_and_empty_rows(gpu):
    """NaN has no weight; +inf takes everything; a row without weight gives -1 and 0; drafts outside the
    vocabulary are refused."""
    logits, dl, drafts, start, u, un = case([1, 1, 1, 1, 1, 1], 9000, 13)
    u[:] = 0.5
    drafts[:] = [5, 6, 7, -1, 9000, 4]
    logits[0, ::2] = np.nan
    logits[2, 8500] = np.inf           # sequence 1 drafted 6
    logits[4] = -np.inf                # sequence 2: nothing to draw from
    logits[5] = np.nan
    dl[5] = -np.inf                    # sequence 5: the drafter's row has no weight: q = 0, p > 0 takes it
    with np.errstate(divide="ignore", invalid="ignore"):
        for t in (1.0, 0.0):
            got = check((logits, dl, drafts, start, u, un), 1, 0.0, t)
            assert got[0][1, 0] == 8500 and got[0][2, 0] == -1 and got[2][2, 0] == 0
            assert got[1][3] == 0 and got[1][4] == 0
        assert check((logits, dl, drafts, start, u, un), 1, 0.0, 1.0)[1][5] == 1


def test_greedy_is_softcap_argmax(gpu):
    """Ties go to the lowest index, and the drawn token is g4_softcap_argmax's."""
    logits, _, drafts, start, _, _ = case([2, 3], 20000, 14)
    r = np.random.default_rng(0)
    logits[:] = r.integers(-3, 4, logits.shape)
    first = logits.argmax(1)
    drafts[:] = first[[0, 1, 3, 4, 5]]
    drafts[3] += 1
    got = check((logits, None, drafts, start, None, None), 3, 0.0, 0.0, drafter=False)
    assert got[1].tolist() == [2, 1]
    ws = g4.DeviceBuffer(g4.lib().g4_argmax_workspace_bytes(7, 20000))
    tok = dev(np.zeros(7, np.int32))
    g4._check(g4.lib().g4_softcap_argmax(dev(logits).ptr, 7, 20000, 0.0, None, ws.ptr, ws.nbytes, tok.ptr, None))
    tok = tok.download()
    assert got[0][0, 2] == tok[2] and got[0][1, 1] == tok[4]


def test_draws_follow_the_target(gpu):
    """The rule's point: over many sequences the emitted tokens are distributed as the target's, whatever
    the drafter says. 4096 sequences of one draft over 8 tokens; a count of probability p is within 5
    standard deviations."""
    n, vocab = 4096, 8
    r = np.random.default_rng(15)
    row, drow = r.standard_normal(vocab).astype(np.float32), r.standard_normal(vocab).astype(np.float32)
    logits = np.repeat(row[None], 2 * n, 0)
    dl = np.repeat(drow[None], n, 0)
    q, _ = probabilities(drow, 0.0, 1.0)
    p, _ = probabilities(row, 0.0, 1.0)
    drafts = r.choice(vocab, n, p=q / q.sum()).astype(np.int32)
    start = np.arange(n + 1, dtype=np.int32)
    got = run(logits, dl, drafts, start, r.random(n).astype(np.float32), r.random(n).astype(np.float32), 1, 0.0, 1.0, False)
    count = np.bincount(got[0][:, 0], minlength=vocab)
    assert (np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all()


def test_replayed_graphs_and_unaligned_rows(gpu):
    """A captured call replays to the eager result with new random numbers between replays; the vocabulary
    leaves every row but the first unaligned."""
    for t in (1.0, 0.0):
        logits, dl, drafts, start, u, un = case([3, 2, 4], 20001, 16)
        st = g4.Stream()
        d = [dev(x) for x in (logits, dl, drafts, start, u, un)]
        out = dev(np.zeros((3, 5), np.int32)), dev(np.zeros(3, np.int32)), dev(np.zeros((3, 5), np.float32))
        ws = g4.DeviceBuffer(gs.verify_workspace_bytes(3, 9, 20001))
        call = lambda h: gs.verify_drafts(*d, *out, ws, cap=30.0, temperature=t, stream=h)
        g = g4.Graph(st, lambda: call(st.handle))
        r = np.random.default_rng(3)
        for _ in range(4):
            u, un = r.random(9).astype(np.float32), r.random(3).astype(np.float32)
            d[4].upload(u)
            d[5].upload(un)
            want = run(logits, dl, drafts, start, u, un, 4, 30.0, t)
            for o in out:
                o.fill(0x55)
            g4.synchronize()
            g.launch()
            st.synchronize()
            for o, w in zip(out, want):
                assert np.array_equal(o.download(), w)
        g.close()
