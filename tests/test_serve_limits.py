"""What the serving operators refuse at the ends of their arguments (no device needed)."""
import os
import subprocess
import sys
from types import SimpleNamespace

import numpy as np
import pytest

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


@pytest.mark.parametrize("first", ["torch", "library"])
def test_tensors_need_the_librarys_runtime(g4, first):
    """torch brings a HIP runtime of its own. Imported after the library is loaded it stays a second one, and
    its tensors are refused (a stand-in for one here: there is no device)."""
    pytest.importorskip("torch")
    load = ["import torch", "g4.lib()"]
    code = f"""
import sys
from types import SimpleNamespace
sys.path.insert(0, {os.path.dirname(gs.__file__)!r})
import numpy as np
import g4w8a8 as g4
{chr(10).join(load if first == "torch" else load[::-1])}
import g4serve as gs

class Tensor:
    shape, dtype, is_cuda = (4, 16, 2, 128), torch.float16, True
    data_ptr = lambda self: 0x1000
    get_device = lambda self: 0
    stride = lambda self: (4096, 256, 128, 1)

try:
    gs.KVPages(Tensor(), Tensor())
    print("taken")
except g4.G4Error as e:
    print(e)
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, check=True).stdout
    assert ("taken" if first == "torch" else "import torch before the first call into the library") in out


def test_tensors_are_used_on_torchs_current_stream(g4, monkeypatch):
    """Without a stream argument, where any operand is a tensor; DeviceBuffers alone go to the default stream."""
    class Tensor(Fake):
        is_cuda = True
        data_ptr = lambda self: self.ptr
        get_device = lambda self: 0
        stride = lambda self: tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))
        is_contiguous = lambda self: True

    seen = []
    take = staticmethod(lambda *a: seen.append(a[-1]) or 0)
    library = type("Library", (), dict.fromkeys(("g4_paged_prologue", "g4_kv_read", "g4_attention_chunk", "g4_verify_drafts"), take))
    cuda = SimpleNamespace(is_initialized=lambda: True, current_device=lambda: 0)
    monkeypatch.setitem(sys.modules, "torch", SimpleNamespace(cuda=cuda, _C=SimpleNamespace(_cuda_getCurrentRawStream=lambda d: 0x77)))
    monkeypatch.setattr(gs.g4, "lib", lambda: library)
    monkeypatch.setattr(gs, "_one_runtime", True, raising=False)

    def calls(kind, **kw):
        p = gs.KVPages(*[kind((4, 16, 2, 128), np.float16)] * 2)
        c, f = chunk(), Fake
        gs.paged_prologue(p, c, None, f((6, 2, 128), np.float16), f((6, 2, 128), np.float16), None, **kw)
        gs.kv_read(p, c, f((6, 2, 128), np.float16), None, **kw)
        gs.attention_chunk(p, c, f((6, 4, 128), np.float16), f((6, 4, 128), np.float16), f((99,), np.uint8), **kw)
        gs.verify_drafts(f((3, 100), np.float32), None, f((1,), np.int32), f((3,), np.int32), f((1,), np.float32),
                         kind((2,), np.float32), f((2, 2), np.int32), f((2,), np.int32), None, f((99,), np.uint8), **kw)

    calls(Tensor)
    calls(Fake)
    calls(Tensor, stream=0)
    calls(Tensor, stream=5)
    assert seen == [0x77] * 4 + [None] * 4 + [0] * 4 + [5] * 4


def test_grids_of_2_to_the_32_threads_are_refused(g4):
    """The store has a wave per head row, the read-back a block per 16 rows."""
    L, p = g4.lib(), pages(shape=(4, 16, 2, 64))

    def store(tokens, heads, k):
        c = chunk(tokens=tokens)
        g4._check(L.g4_paged_prologue(p.ref, c.ref, 0, 0x1000 if heads else None, 0, 1.0, k, 0, 1.0, k, 0, 1.0, heads, None, None,
                                      None, None, 0, 1e-6, 0x1000 if heads else None, None))
    expect(g4, lambda: store(1 << 20, 61, 0x1000), 5, "more than 67108860 head rows")
    expect(g4, lambda: store((1 << 26) - 3, 1, None), 5, "more than 67108860 head rows")
    expect(g4, lambda: store((1 << 24), 0, 0x1000), 5, "more than 67108860 head rows")
    expect(g4, lambda: g4._check(L.g4_kv_read(p.ref, chunk(tokens=(1 << 28) - 15).ref, 0x1000, None, 0, 0, None)), 5,
           "more than 268435440 rows")
    expect(g4, lambda: g4._check(L.g4_kv_read(p.ref, chunk(tokens=(1 << 31) - 1).ref, 0x1000, None, 0, 0, None)), 5,
           "more than 268435440 rows")
