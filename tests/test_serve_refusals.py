"""The serving operators refuse bad arguments before anything is launched (no device needed)."""
import ctypes

import numpy as np
import pytest

import g4serve as gs


class Fake:
    """A packed operand at a made-up address."""

    def __init__(self, shape, dtype, ptr=0x1000):
        self.shape, self.dtype, self.ptr = tuple(shape), np.dtype(dtype), ptr
        self.nbytes = int(np.prod(shape)) * self.dtype.itemsize


class Strided(Fake):
    def __init__(self, shape, dtype, strides):
        super().__init__(shape, dtype)
        self._strides = tuple(strides)

    def stride(self):
        return self._strides

    def is_contiguous(self):
        return False


def expect(g4, fn, status, fragment):
    with pytest.raises(g4.G4Error) as e:
        fn()
    assert fragment in str(e.value), str(e.value)
    assert e.value.status == status, str(e.value)


def pages(kind=np.int8, shape=(4, 16, 2, 128), scales=True, **kw):
    s = (shape[0], shape[2], shape[1])
    sc = [Fake(s, np.float32)] * 2 if kind == np.int8 and scales else [None, None]
    return gs.KVPages(Fake(shape, kind), Fake(shape, kind), *sc, **kw)


def chunk(seqs=2, tokens=6, max_q=4, max_kv=60, width=4):
    return gs.Chunk(Fake((seqs + 1,), np.int32), Fake((seqs,), np.int32), Fake((seqs, width), np.int32), tokens, max_q, max_kv)


def test_cache_and_chunk_refusals(g4):
    read = lambda p, c: gs.kv_read(p, c, Fake((c.tokens, p.kv_heads, p.head_dim), np.float32), None)
    expect(g4, lambda: pages(np.float32), 1, "pages are f16 or int8 codes")
    expect(g4, lambda: pages(scales=False), 1, "int8 pages need their scales")
    expect(g4, lambda: gs.KVPages(Fake((4, 16, 2, 128), np.float16), Fake((4, 16, 2, 64), np.float16)), 1, "of one 4-axis shape")
    expect(g4, lambda: gs.KVPages(Fake((4, 16, 2, 128), np.float16), Fake((4, 16, 2, 128), np.float16),
                                  Fake((4, 2, 16), np.float32)), 1, "f16 pages have no scales")
    expect(g4, lambda: gs.KVPages(*[Fake((4, 16, 2, 128), np.int8)] * 2, *[Fake((4, 16, 2), np.float32)] * 2), 1, "expected [4, 2, 16]")
    expect(g4, lambda: read(pages(shape=(4, 16, 2, 96)), chunk()), 5, "head_dim 96")
    expect(g4, lambda: read(pages(shape=(4, 24, 2, 128)), chunk()), 1, "page_size 24 is not a power of two")
    expect(g4, lambda: read(pages(shape=(4, 4, 2, 128)), chunk(max_kv=16)), 1, "page_size 4 is not a power of two from 8")
    expect(g4, lambda: read(pages(shape=(4, 8192, 2, 128)), chunk()), 1, "page_size 8192")
    expect(g4, lambda: read(pages(), chunk(max_kv=65)), 1, "4 table pages of 16 slots do not hold max_kv 65")
    expect(g4, lambda: read(pages(), chunk(max_q=0)), 1, "max_q 0")
    expect(g4, lambda: gs.Chunk(Fake((3,), np.int32), Fake((2,), np.int32), Fake((2, 4), np.int64), 6, 4, 60), 1, "int64")
    expect(g4, lambda: gs.Chunk(Fake((2,), np.int32), Fake((2,), np.int32), Fake((2, 4), np.int32), 6, 4, 60), 1, "q_start has shape")
    odd = pages()
    odd.c.k = 0x1008
    expect(g4, lambda: read(odd, chunk()), 1, "16-byte aligned")
    odd = pages()
    odd.c.slot_stride += 8
    expect(g4, lambda: read(odd, chunk()), 1, "multiples of 16 bytes")
    odd = pages()
    odd.c.head_stride = 64
    expect(g4, lambda: read(odd, chunk()), 1, "must hold a row")
    c = chunk()
    c.c.table_stride = 3
    expect(g4, lambda: read(pages(), c), 1, "table_stride 3 < 4")
    c = chunk()
    c.c.kv_len = None
    expect(g4, lambda: read(pages(), c), 1, "needs q_start, kv_len and page_table")


def test_read_refusals(g4):
    p, c = pages(), chunk()
    f = lambda *shape, dt=np.float32: Fake(shape, dt)
    expect(g4, lambda: gs.kv_read(p, c, None, None), 1, "kv-read needs")
    expect(g4, lambda: gs.kv_read(p, c, f(6, 2, 128, dt=np.int8), None), 1, "k_out cannot be int8")
    expect(g4, lambda: gs.kv_read(p, c, f(6, 2, 128), f(6, 2, 128, dt=np.float16)), 1, "of one type and layout")
    expect(g4, lambda: gs.kv_read(p, c, f(2, 3, 2, 128), None), 1, "holds 3 rows a sequence, max_q is 4")
    expect(g4, lambda: gs.kv_read(p, c, f(5, 2, 128), None), 1, "expected [6, 2, 128]")
    expect(g4, lambda: gs.kv_read(p, c, Fake((6, 2, 128), np.float32, 0x1004), None), 1, "16-byte aligned")
    L = g4.lib()
    expect(g4, lambda: g4._check(L.g4_kv_read(p.ref, c.ref, 0x1000, None, 0, 4 * 2 * 128 + 2, None)), 1, "seq_stride must hold")
    expect(g4, lambda: g4._check(L.g4_kv_read(p.ref, c.ref, None, None, 0, 0, None)), 1, "no output")
    expect(g4, lambda: g4._check(L.g4_kv_read(None, c.ref, 0x1000, None, 0, 0, None)), 1, "needs the pages and the chunk")


def test_prologue_refusals(g4):
    p, c = pages(), chunk()
    q, k = Fake((6, 4, 128), np.float32), Fake((6, 2, 128), np.float32)
    qo = Fake((6, 4, 128), np.float16)
    call = lambda q=q, k=k, v=k, qo=qo, **kw: gs.paged_prologue(p, c, q, k, v, qo, **kw)
    expect(g4, lambda: call(v=None), 1, "needs k and v together")
    expect(g4, lambda: call(qo=None), 1, "needs q and q_out together")
    expect(g4, lambda: call(q=None, k=None, v=None, qo=None), 1, "needs q, or k and v")
    expect(g4, lambda: call(k=Fake((6, 2, 128), np.float16), v=Fake((6, 2, 128), np.float16)), 1, "must be of one type")
    expect(g4, lambda: call(q=Fake((6, 4, 128), np.int32)), 1, "q cannot be int32")
    expect(g4, lambda: call(q=Strided((6, 4, 128), np.float32, (512, 130, 1))), 1, "heads must be packed")
    expect(g4, lambda: call(q=Strided((6, 4, 128), np.float32, (256, 128, 1))), 1, "its tokens apart")
    expect(g4, lambda: call(q_gain=Fake((64,), np.float32)), 1, "q_gain has shape")
    tab = Fake((59, 64), np.float32)
    expect(g4, lambda: call(cos=tab, sin=tab), 1, "the tables hold 59 positions, max_kv is 60")
    expect(g4, lambda: call(cos=tab), 1, "needs cos and sin together")
    L = g4.lib()
    raw = lambda xk=0, q=0x1000, k=0x1000, heads=4, qo=0x1000, qs=0: g4._check(L.g4_paged_prologue(
        p.ref, c.ref, xk, q, qs, 1.0, k, 0, 1.0, k, 0, 1.0, heads, None, None, None, None, 0, 1e-6, qo, None))
    expect(g4, lambda: raw(xk=3), 1, "rows are f32, f16 or int8 codes, got kind 3")
    expect(g4, lambda: raw(heads=0), 1, "q needs heads and q_out")
    expect(g4, lambda: raw(q=None), 1, "none of them stands alone")
    expect(g4, lambda: raw(qs=500), 1, "a row stride is shorter than the row")


def test_attention_refusals(g4):
    p, c = pages(), chunk()
    q = Fake((6, 4, 128), np.float16)
    ws = Fake((1 << 24,), np.uint8)
    call = lambda q=q, o=q, ws=ws, **kw: gs.attention_chunk(p, c, q, o, ws, **kw)
    expect(g4, lambda: call(q=Fake((6, 4, 128), np.float32)), 1, "q cannot be float32")
    expect(g4, lambda: call(q=Fake((6, 3, 128), np.float16), o=Fake((6, 3, 128), np.float16)), 1, "3 query heads do not divide over 2")
    expect(g4, lambda: call(o=Fake((6, 4, 64), np.float16)), 1, "out has shape")
    expect(g4, lambda: call(o=Fake((6, 4, 128), np.int8)), 1, "need the consumer's inScale")
    expect(g4, lambda: call(window=-1), 1, "window -1")
    expect(g4, lambda: call(ws=Fake((8,), np.uint8)), 1, "workspace 8 B <")
    expect(g4, lambda: call(q=Fake((6, 4, 128), np.float16, 0x1008)), 1, "16-byte aligned")
    expect(g4, lambda: call(q=Strided((6, 4, 128), np.float16, (516, 128, 1))), 1, "a multiple of 8")
    expect(g4, lambda: gs.attention_chunk_workspace_bytes(p, c, 3), 1, "no such call")
    expect(g4, lambda: g4._check(g4.lib().g4_attention_chunk(p.ref, c.ref, 0x1000, 0, 4, 1.0, 0, None, 0, 0x1000, 1, 0.0, None)), 1, "a workspace")
    expect(g4, lambda: g4._check(g4.lib().g4_attention_chunk(p.ref, c.ref, 0x1000, 0, 4, 1.0, 0, 0x1000, 1 << 24, 0x1000, 3, 0.0, None)), 1, "got kind 3")


def test_attention_limits(g4, monkeypatch):
    p, q, ws = pages(), Fake((6, 4, 128), np.float16), Fake((1 << 24,), np.uint8)
    call = lambda p=p, c=chunk(), **kw: gs.attention_chunk(p, c, q, q, ws, **kw)
    for scale in (float("inf"), float("nan"), 2.0 ** 127):
        expect(g4, lambda: call(scale=scale), 1, "below 2^127")
    wide = Strided((4, 16, 2, 128), np.float16, (1 << 31, 256, 128, 1))
    expect(g4, lambda: call(p=gs.KVPages(wide, wide)), 5, "2^31 or more elements apart")
    long = gs.Chunk(Fake((3,), np.int32), Fake((2,), np.int32), Fake((2, (1 << 26) + 1), np.int32), 6, 4, (1 << 30) + 1)
    expect(g4, lambda: call(c=long), 5, "over 2^30 positions")
    many = 1 << 23
    crowd = gs.Chunk(Fake((many + 1,), np.int32), Fake((many,), np.int32), Fake((many, 4), np.int32), many, 1, 60)
    big = Fake((many, 4, 128), np.float16)
    expect(g4, lambda: gs.attention_chunk(p, crowd, big, big, ws), 5, "blocks of query rows")
    expect(g4, lambda: gs.attention_chunk_workspace_bytes(p, crowd, 4), 1, "no such call")
    monkeypatch.setattr(gs, "_device", lambda: 1)
    for f in (call, lambda: gs.kv_read(p, chunk(), q, None), lambda: gs.paged_prologue(p, chunk(), q, None, None, q)):
        expect(g4, f, 1, "on another device than the current one")


def test_verify_refusals(g4):
    f = Fake
    base = dict(logits=f((5, 100), np.float32), draft_logits=f((3, 100), np.float32), draft_tokens=f((3,), np.int32),
                draft_start=f((3,), np.int32), u=f((3,), np.float32), u_next=f((2,), np.float32),
                tokens=f((2, 4), np.int32), accepted=f((2,), np.int32), logprobs=f((2, 4), np.float32),
                workspace=f((1 << 20,), np.uint8))

    def call(temperature=1.0, cap=0.0, **kw):
        gs.verify_drafts(*{**base, **kw}.values(), cap=cap, temperature=temperature)
    expect(g4, lambda: call(logits=f((4, 100), np.float32)), 1, "expected [5, 100]")
    expect(g4, lambda: call(draft_logits=f((3, 99), np.float32)), 1, "expected [3, 100]")
    expect(g4, lambda: call(draft_tokens=f((3,), np.int64)), 1, "int64")
    expect(g4, lambda: call(u=None), 1, "sampling needs the random numbers")
    expect(g4, lambda: call(u_next=None), 1, "sampling needs the random numbers")
    expect(g4, lambda: call(temperature=-1.0), 1, "temperature and cap")
    expect(g4, lambda: call(temperature=float("nan")), 1, "temperature and cap")
    expect(g4, lambda: call(cap=float("inf")), 1, "temperature and cap")
    expect(g4, lambda: call(tokens=f((2, 66), np.int32), logprobs=f((2, 66), np.float32)), 1, "max_drafts 65 (0 to 63)")
    expect(g4, lambda: call(workspace=f((16,), np.uint8)), 1, "workspace 16 B <")
    expect(g4, lambda: call(workspace=f((1 << 20,), np.uint8, 0x1008)), 1, "16-byte aligned")
    expect(g4, lambda: gs.verify_workspace_bytes(0, 1, 10), 1, "no such call")
    assert g4.lib().g4_verify_workspace_bytes(1, 1, 1 << 31) == 0


def test_host_tensors_are_refused(g4):
    torch = pytest.importorskip("torch")
    x = torch.zeros((4, 16, 2, 128), dtype=torch.float16)
    expect(g4, lambda: gs.KVPages(x, x), 1, "is not in device memory")
    expect(g4, lambda: gs.KVPages(x.double(), x.double()), 1, "no operand of this library is torch.float64")


def test_struct_layout(g4):
    """The ctypes structs are the header's, field by field."""
    assert ctypes.sizeof(gs.KVPagesStruct) == 4 * 8 + 5 * 4 + 4 + 3 * 8
    assert ctypes.sizeof(gs.ChunkStruct) == 4 * 4 + 3 * 8 + 8 + 8
    assert gs.ChunkStruct.table_stride.offset == 48 and gs.KVPagesStruct.page_stride.offset == 56
