"""What the serving operators refuse at the ends of their arguments (no device needed)."""
import numpy as np

import g4serve as gs
from test_serve_refusals import Fake, Strided, chunk, expect, pages


def test_workspaces_that_are_not_contiguous_are_refused(g4):
    """An expanded tensor counts bytes that it does not hold."""
    p, c, q = pages(), chunk(), Fake((6, 4, 128), np.float16)
    expanded = Strided((1 << 24,), np.uint8, (0,))
    expect(g4, lambda: gs.attention_chunk(p, c, q, q, expanded), 1, "the workspace must be contiguous")
    expect(g4, lambda: gs.verify_drafts(Fake((3, 100), np.float32), None, Fake((1,), np.int32), Fake((3,), np.int32),
                                        Fake((1,), np.float32), Fake((2,), np.float32), Fake((2, 2), np.int32),
                                        Fake((2,), np.int32), None, expanded), 1, "the workspace must be contiguous")
