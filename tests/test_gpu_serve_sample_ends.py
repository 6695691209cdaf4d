"""Sampling where the answer is one token, and how often a token is accepted only as a neighbour of the definition's."""
import numpy as np
import pytest

from test_gpu_serve_sample import LAST, both, mixed, numbers, run

pytestmark = pytest.mark.gpu

# Weights are 1.2e-12 off and counted in steps of 2^-44 at least: so is the sum of n equal ones, relative to itself.
OFF = 2e-12

PARAMS = ({}, {"min_p": 0.5}, {"min_p": 1.0}, {"top_k": 1}, {"top_k": 40}, {"top_p": 0.7}, {"top_k": 900, "top_p": 0.999},
          {"top_k": 2, "min_p": 1e-30})


def draw(logits, u, t, cap, params):
    n = len(u)
    return run(logits, u, temperature=[t] * n, cap=cap, **{k: [v] * n for k, v in params.items()})


@pytest.mark.parametrize("params", PARAMS, ids=str)
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("t", [1e-45, 1e-38, 1e-20, 1e-12])
def test_tiny_temperatures_draw_the_maximum(gpu, t, cap, params):
    """All others' weights are 0, also of the neighbouring f32 below the maximum: its y is 7e-8 lower at
    least (1e-10 next to a maximum of 0.001), a hundred temperatures, and far past the softcap's error of 8e-14 of itself. Maxima
    below half the cap, next to it on both sides, where another series takes over, and far above."""
    half = np.float32(15)
    tops = np.array([1e-3, 3, -2, half, np.nextafter(half, np.float32(0)), np.nextafter(half, np.float32(99)), 14.9999, 15.0001,
                     20, 45, 60, 90, -20, 10.123], np.float32)
    r = np.random.default_rng(1)
    vocab = 3001
    logits = (tops[:, None] - np.abs(8 * r.standard_normal((len(tops), vocab))) - 1).astype(np.float32)
    at = r.integers(0, vocab, len(tops))
    for i, top in enumerate(tops):
        logits[i, r.integers(0, vocab, 700)] = np.nextafter(top, np.float32(-np.inf))
        logits[i, r.integers(0, vocab, 300)] = -np.inf
        logits[i, r.integers(0, vocab, 300)] = np.nan
        logits[i, at[i]] = top
    for u in (0.0, 0.37, LAST):
        tokens, lps = draw(logits, np.full(len(tops), u, np.float32), t, cap, params)
        assert np.array_equal(tokens, at)
        assert (np.abs(lps) <= OFF).all()


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("t", [1e-45, 1e-30])
@pytest.mark.parametrize("top", [2.5, 15.0, 40.0])
def test_tiny_temperatures_share_out_ties(gpu, t, cap, top):
    """n tokens of the largest logit have the whole weight alike: the first floor(u n) + 1 of them by id, of those that the
    filters keep. (u n is no whole number in any case, but where u is 0.)"""
    r = np.random.default_rng(2)
    n, vocab, most = 24, 5000, np.float32(top)
    logits = (top - 1 - np.abs(4 * r.standard_normal((n, vocab)))).astype(np.float32)
    u = ((np.arange(n) + 0.3) / n).astype(np.float32)
    u[0] = 0
    ids = []
    for i in range(n):
        ids.append(np.sort(r.permutation(vocab)[:(1, 2, 7, 100, 1023)[i % 5]]))
        logits[i, r.integers(0, vocab, 50)] = np.nextafter(most, np.float32(0))
        logits[i, ids[i]] = most
    for params, kept in (({}, lambda m: m), ({"top_k": 5}, lambda m: min(m, 5)), ({"min_p": 1.0}, lambda m: m),
                         ({"top_p": 0.45}, lambda m: int(np.ceil(np.float32(0.45) * np.float64(m))))):
        tokens, lps = draw(logits, u, t, cap, params)
        for i in range(n):
            m = len(ids[i])
            assert tokens[i] == ids[i][int(np.float64(u[i]) * kept(m))], (i, params)
            assert abs(lps[i] + np.log(m)) <= np.log(m) * 2.0 ** -24 * 1.01 + OFF, (i, params)


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("vocab", [1000, 32003, 262144])
def test_neighbours_are_rare(gpu, vocab, cap):
    """A running sum within the weights' error (1e-8 of the total at 262144 tokens) of a target is rare: with an average weight of
    4e-6 of the total there, two targets a row, one row in 200. A token next to the definition's every time is none."""
    off = rows = 0
    for seed in range(4):
        r = np.random.default_rng(100 + seed)
        logits = (3 * r.standard_normal((40, vocab))).astype(np.float32)
        logits[::2, r.integers(0, vocab, 20)] += 15
        off += both(logits, numbers(r, 40), cap=cap, **mixed(r, 40, vocab))
        rows += 40
    assert off <= rows // 20
