"""Plans, adapters and sampling at the ends of what their arguments may be."""
import numpy as np
import pytest

import g4serve as gs
import g4w8a8 as g4
from servecases import dev
from test_gpu_serve_sample import both, mixed, numbers, run, sample

pytestmark = pytest.mark.gpu


def put(buffer, offset, a):
    """a's bytes at an offset of a device buffer."""
    a = np.ascontiguousarray(a)
    g4._check(g4.lib().g4_memcpy_h2d(buffer.ptr + offset, a.ctypes.data, a.nbytes, None))


def get(buffer, offset, n, dtype):
    out = np.empty(n, dtype)
    g4._check(g4.lib().g4_memcpy_d2h(out.ctypes.data, buffer.ptr + offset, out.nbytes, None))
    return out


@pytest.mark.parametrize("cap", [1e-40, 1e-30, 1e-3, 1.0, 100.0, 1e9, 1e30, 3e38])
def test_caps_of_every_size(gpu, cap):
    """A cap far below the logits leaves them nearly alike, but in their order; one far above changes nothing."""
    r = np.random.default_rng(1)
    for rows, vocab in ((24, 5000), (70, 40001)):
        logits = (3 * r.standard_normal((rows, vocab))).astype(np.float32)
        logits[::2, r.integers(0, vocab, 20)] += 15
        logits[:, r.integers(0, vocab, 50)] = -np.inf
        params, u = mixed(r, rows, vocab), numbers(r, rows)
        both(logits, u, cap=cap, **params)
        if cap >= 1e9:
            capped = run(logits, u, cap=cap, **params)
            assert np.array_equal(capped[0], run(logits, u, **params)[0])


def test_as_many_rows_as_a_call_takes(gpu):
    r = np.random.default_rng(2)
    rows, vocab = 65535, 33
    logits = (3 * r.standard_normal((500, vocab))).astype(np.float32)
    index = r.integers(-1, 500, rows).astype(np.int32)
    params, u = mixed(r, rows, vocab), numbers(r, rows)
    tokens, _ = run(logits, u, index=index, **params)
    off = 0
    for i in range(0, rows, 37):
        p = [params[n][i] for n in ("temperature", "top_k", "top_p", "min_p")]
        want = -1 if index[i] < 0 else sample(logits[index[i]], 0.0, *p, u[i])[0]
        off += tokens[i] != want
    assert off <= 1  # (a target within 2e-12 of a running sum)


def test_as_many_tokens_and_adapters_as_a_batch_takes(gpu):
    r = np.random.default_rng(3)
    t, m, k, n, rank = 1 << 19, 4096, 16, 9, 8
    ids = r.integers(-2, m, t).astype(np.int32)
    a, b = (r.integers(-3, 4, s).astype(np.float16) for s in ((m, rank, k), (m, n, rank)))
    x = r.integers(-4, 5, (t, k)).astype(np.int8)
    adapters = gs.Adapters(dev(a), dev(b))
    groups = g4.DeviceBuffer(gs.adapter_groups_bytes(t, m))
    gs.adapter_groups(dev(ids), groups, m)
    out = dev(np.full((t, n), 77, np.float32))
    gs.adapter_linear(adapters, groups, dev(x), None, out, g4.DeviceBuffer(gs.adapter_workspace_bytes(adapters, t)))
    g4.synchronize()
    at = np.maximum(ids, 0)
    want = np.empty((t, n))
    for i in range(0, t, 1 << 16):  # whole numbers below 2^11: exact
        s = np.s_[i:i + (1 << 16)]
        h = (a[at[s]].astype(np.float32) @ x[s, :, None].astype(np.float32))
        want[s] = (b[at[s]].astype(np.float32) @ h)[:, :, 0]
    want[ids == -1], want[ids == -2] = 0, 77
    assert np.array_equal(out.download(), want)


@pytest.mark.parametrize("x_type", [np.float16, np.int8, np.float32])
def test_the_longest_inner_size(gpu, x_type):
    k, n, rank = 1 << 23, 24, 8
    r = np.random.default_rng(4)
    at = np.unique(np.concatenate([r.integers(0, k, 60), [0, 255, 256, k // 2, k - 257, k - 1]]))
    x, a = np.zeros((2, k), x_type), np.zeros((1, rank, k), np.float16)
    x[:, at], a[:, :, at] = r.integers(-3, 4, (2, len(at))), r.integers(-3, 4, (1, rank, len(at)))
    b = r.integers(-3, 4, (1, n, rank)).astype(np.float16)
    adapters = gs.Adapters(dev(a), dev(b))
    groups = g4.DeviceBuffer(gs.adapter_groups_bytes(2, 1))
    gs.adapter_groups(dev(np.zeros(2, np.int32)), groups, 1)
    out = dev(np.full((2, n), 77, np.float32))
    gs.adapter_linear(adapters, groups, dev(x), None, out, g4.DeviceBuffer(gs.adapter_workspace_bytes(adapters, 2)))
    g4.synchronize()
    want = (x[:, at].astype(np.float64) @ a[0, :, at].astype(np.float64)) @ b[0].astype(np.float64).T
    assert np.array_equal(out.download(), want)


def test_the_longest_outer_size(gpu):
    """2^30 outputs of a row: B of 16 GiB, of which some rows are not zero."""
    n, k, rank = 1 << 30, 64, 8
    r = np.random.default_rng(5)
    x, a = r.integers(-3, 4, (1, k)).astype(np.float16), r.integers(-3, 4, (1, rank, k)).astype(np.float16)
    b, out = g4.DeviceBuffer.empty((1, n, rank), np.float16), g4.DeviceBuffer.empty((1, n), np.int8)
    b.fill(0)
    out.fill(5)
    adapters = gs.Adapters(dev(a), b)
    groups = g4.DeviceBuffer(gs.adapter_groups_bytes(1, 1))
    gs.adapter_groups(dev(np.zeros(1, np.int32)), groups, 1)
    h = x[0].astype(np.float64) @ a[0].astype(np.float64).T
    places = [0, 504, 512, (1 << 28) - 3, (1 << 29) + 17, n - 600, n - 8]
    rows = [r.integers(-2, 3, (8, rank)).astype(np.float16) for _ in places]
    for at, w in zip(places, rows):
        put(b, 2 * rank * at, w)
    g4.synchronize()
    gs.adapter_linear(adapters, groups, dev(x), None, out, g4.DeviceBuffer(gs.adapter_workspace_bytes(adapters, 1)),
                      out_scale=8.0)
    g4.synchronize()
    for at, w in zip(places, rows):
        want = np.clip(np.rint(w.astype(np.float64) @ h / 8.0), -128, 127)
        assert np.array_equal(get(out, at, 8, np.int8), want), at
    for at in (600, n // 3, n - 16):
        assert (get(out, at, 8, np.int8) == 0).all(), at


def test_a_chunk_of_very_many_rows(gpu):
    """One prompt of 2^24 positions and another, in a chunk with room behind them."""
    page, most = 4096, 1 << 24
    width, tokens = most // page, most + 5000
    table = np.full((2, width), -1, np.int32)
    free = np.arange(2 * width, dtype=np.int32)[::-1].copy()
    z = lambda n: dev(np.full(n, -9, np.int32))
    d_table = dev(table)
    d = dict(q_start=z(3), kv_len=z(2), free_left=z(1), served=z(1), row_pos=z(tokens), row_slot=z(tokens), row_adapter=z(tokens),
             held_out=z(2), last_row=z(2))
    pages = gs.FreePages(dev(free), dev(np.array([2 * width], np.int32)), 2 * width, page)
    gs.plan_chunk(pages, dev(np.zeros(2, np.int32)), dev(np.array([most, 4000], np.int32)), d_table, tokens=tokens, max_q=most,
                  max_kv=most, seq_adapter=dev(np.array([3, 1], np.int32)), **d)
    g4.synchronize()
    got = {n: b.download() for n, b in d.items()}
    assert list(got["q_start"]) == [0, most, most + 4000] and list(got["kv_len"]) == [most, 4000] and got["served"][0] == 2
    assert got["free_left"][0] == width - 1 and list(got["held_out"]) == [width, 1]
    given = free[width - 1:]
    t = d_table.download()
    assert np.array_equal(t[0], given[:-1]) and t[1, 0] == given[-1] and (t[1, 1:] == -1).all()
    pos = np.concatenate([np.arange(most), np.arange(4000)])
    slot = np.concatenate([np.repeat(given[:-1].astype(np.int64) * page, page), np.full(4000, int(given[-1]) * page)]) + pos % page
    behind = np.full(1000, -1)
    assert np.array_equal(got["row_pos"], np.concatenate([pos, behind]))
    assert np.array_equal(got["row_slot"], np.concatenate([slot, behind]))
    assert np.array_equal(got["row_adapter"], np.repeat([3, 1, -2], [most, 4000, 1000]))
