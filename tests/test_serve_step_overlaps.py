"""Buffers that the adapters' kernels read while others are written: refused where they overlap (no device needed)."""
import numpy as np
import pytest

import g4serve as gs
from test_serve_refusals import Fake, expect


@pytest.mark.parametrize("k,launches", [(256, 1), (8192, 2)])
def test_groups_and_workspace_are_apart(g4, k, launches):
    """Rows of a batch come from the groups: with a first product written over them they would be any number."""
    p = gs.Adapters(Fake((4, 16, k), np.float16, 1 << 20), Fake((4, 64, 16), np.float16, 1 << 21))
    x, out = Fake((300, k), np.float32, 1 << 22), Fake((300, 64), np.float32, 1 << 28)
    need, room = gs.adapter_groups_bytes(300, 4), gs.adapter_workspace_bytes(p, 300)
    assert (room > 16) == (launches > 1)
    at = 1 << 30
    for groups, workspace in ((at, at), (at, at + (need - 1) // 16 * 16), (at + (room - 1) // 16 * 16, at)):
        call = lambda: gs.adapter_linear(p, Fake((need,), np.uint8, groups), x, None, out, Fake((room,), np.uint8, workspace))
        expect(g4, call, 1, "groups and workspace overlap")
