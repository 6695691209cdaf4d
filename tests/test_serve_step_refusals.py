"""What the plan, the release, the adapters and the sampling refuse before anything is launched (no device needed)."""
import ctypes
import sys
from types import SimpleNamespace

import numpy as np
import pytest

import g4serve as gs
from test_serve_refusals import Fake, Strided, expect

I, F = np.int32, np.float32


def i32(*shape, ptr=0x1000):
    return Fake(shape, I, ptr)


def free(pages=100, count=None, num_pages=100, page=16):
    return gs.FreePages(i32(pages), i32(1, ptr=0x9000) if count is None else count, num_pages, page)


def test_plan_refusals(g4):
    def call(f=None, cached=i32(3, ptr=0x2000), rows=i32(3), table=i32(3, 4), kv_len=i32(3), left=i32(1), tokens=9, max_q=4,
             max_kv=60, **kw):
        gs.plan_chunk(f or free(), cached, rows, table, i32(4), kv_len, left, i32(1), tokens=tokens, max_q=max_q, max_kv=max_kv, **kw)
    expect(g4, lambda: call(free(page=24)), 1, "page_size 24 is not a power of two")
    expect(g4, lambda: call(free(num_pages=0)), 1, "a free list of 100 of 0 pages")
    expect(g4, lambda: call(free(num_pages=1 << 27)), 5, "slots are 32-bit")
    expect(g4, lambda: free(count=i32(2)), 1, "count has shape [2]")
    expect(g4, lambda: call(cached=i32(2)), 1, "cached has shape [2], expected [3]")
    expect(g4, lambda: call(cached=None), 1, "plan-chunk needs cached, rows")
    expect(g4, lambda: call(rows=Fake((3,), np.int64)), 1, "int64")
    expect(g4, lambda: call(max_kv=65), 1, "4 table pages of 16 slots do not hold max_kv 65")
    expect(g4, lambda: call(tokens=0), 1, "0 tokens")
    expect(g4, lambda: call(max_q=0), 1, "max_q 0")
    expect(g4, lambda: call(table=i32(3)), 1, "expected [seqs][pages]")
    expect(g4, lambda: call(table=Strided((3, 4), I, (3, 1))), 1, "page_table rows must be packed")
    expect(g4, lambda: call(left=i32(1, ptr=0x9000)), 1, "cannot be the arrays they are made from")
    expect(g4, lambda: call(kv_len=i32(3, ptr=0x2000)), 1, "cannot be the arrays they are made from")
    expect(g4, lambda: call(held=i32(3), held_out=i32(3)), 1, "cannot be the arrays they are made from")
    expect(g4, lambda: call(row_pos=i32(8)), 1, "row_pos has shape [8], expected [9]")
    apart = lambda i, *shape: i32(*shape, ptr=0x10000 * (i + 1))
    outs = dict(q_start=4, kv_len=3, free_left=1, served=1, held_out=3, row_pos=9, row_slot=9, row_adapter=9, last_row=3)
    for i, at in enumerate(outs):
        for j, name in enumerate(("cached", "rows", "held", "seq_adapter", "count")):
            to = {n: apart(m, size) for m, (n, size) in enumerate(outs.items())}
            given = {n: apart(20 + m, 3) for m, n in enumerate(("cached", "rows", "held", "seq_adapter"))}
            to[at] = i32(outs[at], ptr=0x9000 if name == "count" else 0x10000 * (21 + j))
            expect(g4, lambda: gs.plan_chunk(free(), page_table=i32(3, 4), tokens=9, max_q=4, max_kv=60, **to, **given), 1,
                   "cannot be the arrays they are made from")
    n = 4097
    expect(g4, lambda: gs.plan_chunk(free(), i32(n, ptr=0x2000), i32(n), i32(n, 4), i32(n + 1), i32(n), i32(1), i32(1), tokens=9,
                                     max_q=4, max_kv=60), 5, "4097 sequences in one call (at most 4096)")
    s = g4.lib().g4_plan_chunk
    raw = lambda **kw: g4._check(s(kw.get("list", free().ref), 0x2000, 0x1000, None, None, 3, 9, 4, 60, kw.get("table", 0x1000), 4,
                                   kw.get("stride", 0), kw.get("q", 0x1000), 0x3000, *[None] * 1, 0x1000, 0x1000, *[None] * 5))
    expect(g4, lambda: raw(list=None), 1, "needs the free pages")
    expect(g4, lambda: raw(table=None), 1, "plan-chunk: 3 sequences")
    expect(g4, lambda: raw(stride=3), 1, "table_stride 3 < 4")
    expect(g4, lambda: raw(q=None), 1, "plan-chunk needs cached")


def test_release_refusals(g4):
    call = lambda f=None, table=i32(3, 4), first=i32(3), last=i32(3), out=i32(1): gs.release_pages(f or free(), table, first, last, out)
    expect(g4, lambda: call(free(page=4)), 1, "page_size 4")
    expect(g4, lambda: call(first=i32(2)), 1, "first has shape [2]")
    expect(g4, lambda: call(table=Fake((3, 4), np.int64)), 1, "int64")
    expect(g4, lambda: call(out=i32(1, ptr=0x9000)), 1, "count_out cannot be the list's count")
    expect(g4, lambda: call(table=i32(5000, 4), first=i32(5000), last=i32(5000)), 5, "at most 4096")
    expect(g4, lambda: g4._check(g4.lib().g4_release_pages(free().ref, 0x1000, 4, 0, None, 0x1000, 3, 0x1000, None)), 1,
           "release-pages needs first, last")


def test_adapter_refusals(g4):
    h = lambda *s, ptr=0x1000: Fake(s, np.float16, ptr)

    def pool(a=h(4, 16, 256), b=h(4, 64, 16), **kw):
        return gs.Adapters(a, b, **kw)

    expect(g4, lambda: pool(a=Fake((4, 16, 256), F)), 1, "a cannot be float32")
    expect(g4, lambda: pool(b=h(4, 64, 8)), 1, "adapters need a [count][max_rank][k]")
    expect(g4, lambda: pool(b=h(3, 64, 16)), 1, "adapters need a [count][max_rank][k]")
    expect(g4, lambda: pool(scales=Fake((3,), F)), 1, "scales has shape [3]")
    expect(g4, lambda: pool(ranks=Fake((4,), F)), 1, "ranks cannot be float32")
    expect(g4, lambda: pool(a=Strided((4, 16, 256), np.float16, (4096, 300, 1))), 1, "an adapter must be packed")
    expect(g4, lambda: pool(a=Strided((4, 16, 256), np.float16, (4000, 256, 1))), 1, "adapters apart")
    ws, x, base = Fake((1 << 24,), np.uint8), Fake((6, 256), F), Fake((6, 64), F)

    def call(p=None, g=ws, x=x, base=base, out=base, ws=ws, **kw):
        gs.adapter_linear(p or pool(), g, x, base, out, ws, **kw)

    for p, text in ((pool(h(4, 20, 256), h(4, 64, 20)), "max_rank 20"), (pool(h(4, 136, 256), h(4, 64, 136)), "max_rank 136"),
                    (pool(h(4, 16, 256, ptr=0x1008)), "16-byte aligned"),
                    (pool(h(5000, 16, 256), h(5000, 64, 16)), "5000 adapters"),
                    (pool(Strided((4, 16, 256), np.float16, (4100, 256, 1))), "multiples of 8")):
        expect(g4, lambda: call(p), 1, text)
        expect(g4, lambda: gs.adapter_workspace_bytes(p, 6), 1, "no such call")
    expect(g4, lambda: call(pool(h(4, 16, 252)), x=Fake((6, 252), F)), 1, "k a multiple of 8")
    expect(g4, lambda: call(pool(h(1, 16, (1 << 23) + 8), h(1, 64, 16)), x=Fake((6, (1 << 23) + 8), F)), 1, "up to 8388608")
    wide = pool(Fake((1, 16, 256), np.float16), Fake((1, (1 << 30) + 1, 16), np.float16))
    expect(g4, lambda: call(wide, base=None, out=Fake((6, (1 << 30) + 1), F, 0x5000)), 1, "n up to 1073741824")
    expect(g4, lambda: call(x=Fake((6, 128), F)), 1, "x has shape [6, 128]")
    expect(g4, lambda: call(x=Fake((6, 256), I)), 1, "x cannot be int32")
    expect(g4, lambda: call(x=Strided((6, 256), F, (257, 1))), 1, "x must be 16-byte aligned, its rows too")
    expect(g4, lambda: call(x=Fake((6, 256), F, 0x1004)), 1, "x must be 16-byte aligned")
    expect(g4, lambda: call(base=Fake((5, 64), F)), 1, "base has shape [5, 64]")
    expect(g4, lambda: call(out=Fake((6, 64), np.int8, 0x5000)), 1, "int8 output codes need a calibrated outScale")
    expect(g4, lambda: call(out=Fake((6, 64), np.float16)), 1, "out can be base only with its type and stride")
    expect(g4, lambda: call(out=Strided((6, 64), F, (80, 1))), 1, "out can be base only with its type and stride")
    expect(g4, lambda: call(), 1, "out cannot be x")
    expect(g4, lambda: call(g=Fake((16,), np.uint8)), 1, "groups 16 B <")
    expect(g4, lambda: call(ws=Fake((8,), np.uint8)), 1, "workspace 8 B <")
    expect(g4, lambda: call(ws=Strided((1 << 24,), np.uint8, (0,))), 1, "the workspace must be contiguous")
    expect(g4, lambda: call(g=Fake((1 << 20,), np.uint8, 0x1008)), 1, "16-byte aligned")
    expect(g4, lambda: g4._check(g4.lib().g4_adapter_linear(pool().ref, 0x1000, 1 << 20, 6, 0x1000, 3, 0, 1.0, 0x1000, 0, 0, 1.0, 0x1000,
                                                            0, 0, 0.0, 0x1000, 1 << 20, None)), 1, "f32, f16 or int8 codes")
    expect(g4, lambda: gs.adapter_groups(i32(6), Fake((64,), np.uint8), 4), 1, "groups 64 B <")
    expect(g4, lambda: gs.adapter_groups(Fake((6,), np.int64), ws, 4), 1, "int64")
    expect(g4, lambda: gs.adapter_groups_bytes((1 << 19) + 1, 4), 1, "no such call")
    expect(g4, lambda: gs.adapter_groups_bytes(4, 4097), 1, "no such call")


def test_sample_refusals(g4):
    base = dict(logits=Fake((3, 100), F), u=Fake((3,), F), tokens=i32(3), logprobs=Fake((3,), F), workspace=Fake((1 << 20,), np.uint8))
    call = lambda cap=0.0, **kw: gs.sample_tokens(*{**base, **{k: v for k, v in kw.items() if k in base}}.values(), cap=cap,
                                                  **{k: v for k, v in kw.items() if k not in base})
    expect(g4, lambda: call(logits=Fake((3, 100), np.float16)), 1, "logits cannot be float16")
    expect(g4, lambda: call(logits=Fake((300,), F)), 1, "expected [rows][vocab]")
    expect(g4, lambda: call(logits=Fake((2, 100), F)), 1, "3 rows from 2 rows of logits need row_index")
    expect(g4, lambda: call(tokens=i32(2)), 1, "tokens has shape [2]")
    expect(g4, lambda: call(temperature=Fake((2,), F)), 1, "temperature has shape [2]")
    expect(g4, lambda: call(top_k=Fake((3,), F)), 1, "top_k cannot be float32")
    expect(g4, lambda: call(cap=-1.0), 1, "cap must be finite")
    expect(g4, lambda: call(cap=float("nan")), 1, "cap must be finite")
    expect(g4, lambda: call(workspace=Fake((64,), np.uint8)), 1, "workspace 64 B <")
    expect(g4, lambda: call(workspace=Fake((1 << 20,), np.uint8, 0x1008)), 1, "16-byte aligned")
    expect(g4, lambda: call(workspace=Strided((1 << 20,), np.uint8, (0,))), 1, "the workspace must be contiguous")
    expect(g4, lambda: call(logits=Fake((3, (1 << 22) + 1), F)), 5, "at most 65535")
    expect(g4, lambda: gs.sample_workspace_bytes(1, (1 << 22) + 1), 1, "no such call")
    expect(g4, lambda: gs.sample_workspace_bytes(65536, 10), 1, "no such call")
    s = lambda stride=0, u=0x1000: g4._check(g4.lib().g4_sample_tokens(0x1000, 3, stride, None, 3, 100, 0.0, None, None, None, None, u,
                                                                       0x1000, 1 << 20, 0x1000, None, None))
    expect(g4, lambda: s(stride=99), 1, "logit_stride 99 < vocabulary 100")
    expect(g4, lambda: s(u=None), 1, "needs logits, u and tokens")


def test_other_devices_are_refused(g4, monkeypatch):
    f, p = free(), gs.Adapters(Fake((4, 16, 256), np.float16), Fake((4, 64, 16), np.float16))
    monkeypatch.setattr(gs, "_device", lambda: 1)
    ws, y = Fake((1 << 24,), np.uint8), Fake((6, 64), F)
    expect(g4, lambda: gs.release_pages(f, i32(3, 4), i32(3), i32(3), i32(1)), 1, "the free pages are on another device")
    expect(g4, lambda: gs.plan_chunk(f, i32(3), i32(3), i32(3, 4), i32(4), i32(3), i32(1), i32(1), tokens=9, max_q=4, max_kv=60), 1,
           "the free pages are on another device")
    expect(g4, lambda: gs.adapter_linear(p, ws, Fake((6, 256), F), y, y, ws), 1, "the adapters are on another device")


def test_struct_layout(g4):
    """The ctypes structs are the header's, field by field."""
    assert ctypes.sizeof(gs.FreePagesStruct) == 2 * 8 + 3 * 4 + 4
    assert ctypes.sizeof(gs.AdaptersStruct) == 4 * 8 + 4 * 4 + 2 * 8
    assert gs.AdaptersStruct.a_stride.offset == 48 and gs.FreePagesStruct.page_size.offset == 24


def test_tensors_are_used_on_torchs_current_stream(g4, monkeypatch):
    """Without a stream argument, where any operand is a tensor; DeviceBuffers alone go to the default stream."""
    class Tensor(Fake):
        is_cuda = True
        data_ptr = lambda self: self.ptr
        get_device = lambda self: 0
        stride = lambda self: tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))
        is_contiguous = lambda self: True

    names = ("g4_plan_chunk", "g4_release_pages", "g4_adapter_groups", "g4_adapter_linear", "g4_sample_tokens")
    seen = []
    library = type("Library", (), dict.fromkeys(names, staticmethod(lambda *a: seen.append(a[-1]) or 0)))
    cuda = SimpleNamespace(is_initialized=lambda: True, current_device=lambda: 0)
    monkeypatch.setitem(sys.modules, "torch", SimpleNamespace(cuda=cuda, _C=SimpleNamespace(_cuda_getCurrentRawStream=lambda d: 0x77)))
    monkeypatch.setattr(gs.g4, "lib", lambda: library)
    monkeypatch.setattr(gs, "_one_runtime", True, raising=False)

    def calls(kind, **kw):
        f, ws = free(), Fake((1 << 24,), np.uint8)
        p = gs.Adapters(Fake((4, 16, 256), np.float16), Fake((4, 64, 16), np.float16))
        gs.plan_chunk(f, i32(3), i32(3), i32(3, 4), i32(4), i32(3), i32(1), i32(1), tokens=9, max_q=4, max_kv=60,
                      last_row=kind((3,), I), **kw)
        gs.release_pages(f, i32(3, 4), kind((3,), I), i32(3), i32(1), **kw)
        gs.adapter_groups(i32(6), kind((1 << 20,), np.uint8), 4, **kw)
        gs.adapter_linear(p, ws, Fake((6, 256), F), None, kind((6, 64), F), ws, **kw)
        gs.sample_tokens(Fake((3, 99), F), Fake((3,), F), i32(3), None, ws, min_p=kind((3,), F), **kw)

    calls(Tensor)
    calls(Fake)
    calls(Tensor, stream=0)
    calls(Tensor, stream=5)
    assert seen == [0x77] * 5 + [None] * 5 + [0] * 5 + [5] * 5
