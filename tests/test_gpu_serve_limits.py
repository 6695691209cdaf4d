"""The serving operators at the ends of what their arguments may be."""
import numpy as np
import pytest

import g4serve as gs
from servecases import Batch, attention, dev, to_kind

pytestmark = pytest.mark.gpu


def run(b, q, window=0, scale=0.1, out=np.float32):
    o = dev(np.full(q.shape, -3, out))
    gs.attention_chunk(b.pages, b.chunk, dev(q), o, b.workspace(q.shape[1], window), scale=scale, window=window)
    return o.download()


def queries(b, heads):
    return b.rng.standard_normal((b.tokens, heads, b.dim)).astype(np.float16)


@pytest.mark.parametrize("kind", ["i8", "f16"])
@pytest.mark.parametrize("window", [30, 31, 1 << 30, (1 << 31) - 40, (1 << 31) - 1])
def test_windows_of_any_size_and_rows_without_positions(gpu, kind, window):
    """A window that hides nothing is none, also where rows stand at negative positions: sequences with more
    rows than positions, alone in their tile and beside rows that have some."""
    b = Batch([(8, 0), (5, 2), (40, 3), (6, 30), (1, 1)], 1, 128, 16, kind, seed=6).upload()
    q = queries(b, 4)
    got = run(b, q, window)
    want, bound = attention(b, q, float(np.float32(0.1)), window)
    assert (np.abs(got - want) <= to_kind(want, bound, np.float32)).all()
    assert (got[:11] == 0).all()
    assert np.array_equal(got.view(np.uint32), run(b, q, 0).view(np.uint32))
