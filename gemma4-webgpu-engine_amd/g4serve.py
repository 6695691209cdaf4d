"""Serving operators on a paged KV cache (include/g4serve.h): the plan of a chunk of new tokens, its
prologue with the quantising store, the read-back, attention of the chunk, low-rank adapters beside the
linears, draft verification, and sampling.

Operands are anything with a shape, a dtype and a device address: g4w8a8.DeviceBuffer, or a torch
tensor on the current device (torch imported before the library is loaded, by the first call into it,
so that both run on one HIP runtime). Types, shapes and layouts are checked here, values and
everything else by the library, which raises G4Error. Everything computes in the HIP library.

stream: a stream's handle (0: the default stream). None: torch's current stream where an operand is a
tensor, since what makes and reads tensors runs there, else the default stream.
"""
from __future__ import annotations

import ctypes
import os
import sys

import g4w8a8 as g4

_vp = ctypes.c_void_p
_KIND_NAMES = {"float32": g4.KIND_F32, "float16": g4.KIND_F16, "int8": g4.KIND_I8,
               "int32": g4.KIND_I32, "uint8": None}
_kinds = {}  # dtype object -> kind, filled as dtypes are met
_X_KINDS = (g4.KIND_F32, g4.KIND_F16, g4.KIND_I8)
_F32, _I32, _F16 = (g4.KIND_F32,), (g4.KIND_I32,), (g4.KIND_F16,)


def _kind(x):
    try:
        return _kinds[x.dtype]
    except KeyError:
        name = str(x.dtype).rpartition(".")[2]
        if name not in _KIND_NAMES:
            raise g4.G4Error(1, f"no operand of this library is {x.dtype}") from None
        return _kinds.setdefault(x.dtype, _KIND_NAMES[name])


def _device() -> int:
    """The current device, which torch tensors have to be on (asked once a call)."""
    torch = sys.modules.get("torch")
    if torch is None or not torch.cuda.is_initialized():
        return 0
    try:
        return torch._C._cuda_getDevice()
    except AttributeError:  # the same, a little slower
        return torch.cuda.current_device()


_one_runtime = None


def _check_runtime():
    """The library and torch share a HIP runtime only where torch's was loaded first: the library then
    finds it under its own runtime's name. Else the process has two, and neither's memory and streams
    are the other's."""
    global _one_runtime
    if _one_runtime is None:
        torch_lib = os.path.join(os.path.dirname(sys.modules["torch"].__file__), "lib", "libc10_hip.so")
        try:  # what each of the two calls
            ours, torchs = (ctypes.cast(x.hipGetDevice, _vp).value for x in (g4.lib(), ctypes.CDLL(torch_lib)))
            _one_runtime = ours == torchs
        except OSError:  # a torch of another layout: as many runtimes as files
            with open("/proc/self/maps") as f:
                _one_runtime = len({line.split()[-1] for line in f if "libamdhip64" in line}) == 1
    if not _one_runtime:
        raise g4.G4Error(1, "a torch tensor of another HIP runtime than this library's: import torch before the "
                            "first call into the library")


def _address(x, what, device):
    """The device address of a buffer or tensor. A host tensor, or one of another device than the
    current one, is refused: its address means nothing to a kernel launched here."""
    try:
        p = x.data_ptr()
    except AttributeError:
        if not x.ptr:
            raise g4.G4Error(1, f"{what} has no device memory") from None
        return x.ptr
    if x.get_device() != device:
        raise g4.G4Error(1, f"{what} is on another device than the current one" if x.is_cuda else
                         f"{what} is not in device memory")
    if not _one_runtime:
        _check_runtime()
    return p


def _stream(stream, device, *operands):
    """The handle to launch on."""
    torch = sys.modules.get("torch")
    if stream is not None or torch is None:
        return stream
    for x in operands:
        if hasattr(x, "data_ptr"):
            try:
                return torch._C._cuda_getCurrentRawStream(device)
            except AttributeError:  # the same, some microseconds slower
                return torch.cuda.current_stream(device).cuda_stream
    return None


def _call_device(pages, chunk) -> int:
    device = _device()
    if pages.device != device or chunk.device != device:
        raise g4.G4Error(1, "the pages or the chunk are on another device than the current one")
    return device


def _packed(x, what, kinds, shape, device):
    """The address of a contiguous operand of one of `kinds` and of `shape`. A call has up to 14 of them: what is in
    order is found so by five questions, and what is not is named by _checked."""
    try:
        if (x.get_device() == device and _one_runtime and _kinds[x.dtype] in kinds and x.shape == shape
                and x.is_contiguous()):
            return x.data_ptr()
    except (AttributeError, KeyError):  # a DeviceBuffer, or a type not met yet
        pass
    return _checked(x, what, kinds, shape, device)


def _checked(x, what, kinds, shape, device):
    if _kind(x) not in kinds:
        raise g4.G4Error(1, f"{what} cannot be {x.dtype}")
    if x.shape != shape:
        raise g4.G4Error(1, f"{what} has shape {list(x.shape)}, expected {list(shape)}")
    _need_contiguous(x, what)
    return _address(x, what, device)


def _need_contiguous(x, what):
    try:
        packed = x.is_contiguous()
    except AttributeError:  # a DeviceBuffer is
        packed = not hasattr(x, "stride")
    if not packed:
        raise g4.G4Error(1, f"{what} must be contiguous")


def _workspace(x, device):
    """(address, bytes) of a workspace. One that is not contiguous may hold fewer bytes than it counts."""
    try:
        if x.get_device() == device and _one_runtime and x.is_contiguous():
            return x.data_ptr(), x.nbytes
    except AttributeError:
        pass
    _need_contiguous(x, "the workspace")
    return _address(x, "workspace", device), x.nbytes


def _rows(x, what, kinds, heads, dim, tokens, device):
    """(address, kind, elements between tokens) of a [tokens][heads][dim] operand, whose tokens may
    lie apart (part of a wider projection's output)."""
    kind = _kind(x)
    if kind not in kinds:
        raise g4.G4Error(1, f"{what} cannot be {x.dtype}")
    if x.shape != (tokens, heads, dim):
        raise g4.G4Error(1, f"{what} has shape {list(x.shape)}, expected {[tokens, heads, dim]}")
    stride = heads * dim
    if hasattr(x, "stride"):
        st = x.stride()
        if st[2] != 1 or (heads > 1 and st[1] != dim) or (tokens > 1 and st[0] < stride):
            raise g4.G4Error(1, f"{what}: a token's heads must be packed, and its tokens apart")
        if tokens > 1:
            stride = st[0]
    return _address(x, what, device), kind, stride


class KVPagesStruct(ctypes.Structure):
    """include/g4serve.h g4_kv_pages."""
    _fields_ = [("k", _vp), ("v", _vp), ("k_scales", _vp), ("v_scales", _vp), ("kind", ctypes.c_int),
                ("num_pages", ctypes.c_int), ("page_size", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("page_stride", ctypes.c_int64),
                ("slot_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class ChunkStruct(ctypes.Structure):
    """include/g4serve.h g4_chunk."""
    _fields_ = [("seqs", ctypes.c_int), ("tokens", ctypes.c_int), ("max_q", ctypes.c_int),
                ("max_kv", ctypes.c_int), ("q_start", _vp), ("kv_len", _vp), ("page_table", _vp),
                ("table_pages", ctypes.c_int), ("table_stride", ctypes.c_int64)]


class KVPages:
    """One layer's page pools: k and v [pages][page_size][kv_heads][head_dim] (heads_first: [pages]
    [kv_heads][page_size][head_dim]), f16, or int8 codes with k_scales / v_scales f32 [pages][kv_heads]
    [page_size]. The pools may be strided views of a larger tensor (the last axis packed, k and v
    alike). Keeps its buffers alive."""

    def __init__(self, k, v, k_scales=None, v_scales=None, heads_first=False):
        kind = _kind(k)
        if kind not in (g4.KIND_F16, g4.KIND_I8) or _kind(v) != kind:
            raise g4.G4Error(1, f"pages are f16 or int8 codes, k and v alike; got {k.dtype} and {v.dtype}")
        if len(k.shape) != 4 or tuple(k.shape) != tuple(v.shape):
            raise g4.G4Error(1, f"pages need k and v of one 4-axis shape, got {list(k.shape)} and {list(v.shape)}")
        pages, a, b, dim = (int(n) for n in k.shape)
        slots, heads = (b, a) if heads_first else (a, b)
        strides = [a * b * dim, b * dim, dim]
        if hasattr(k, "stride"):
            if k.stride() != v.stride() or k.stride()[3] != 1:
                raise g4.G4Error(1, "pages: k and v need the same strides, and packed rows")
            strides = list(k.stride()[:3])
        # the stride of an axis of one element says nothing (torch keeps any number there)
        strides = [n if size > 1 else a * b * dim for n, size in zip(strides, (pages, a, b))]
        page_stride, slot, head = strides[0], *(reversed(strides[1:]) if heads_first else strides[1:])
        self.buffers = (k, v, k_scales, v_scales)
        self.kind, self.kv_heads, self.head_dim, self.page_size = kind, heads, dim, slots
        s = [None, None]
        device = self.device = _device()
        if kind == g4.KIND_I8:
            if k_scales is None or v_scales is None:
                raise g4.G4Error(1, "int8 pages need their scales")
            s = [_packed(x, "page scales", _F32, (pages, heads, slots), device) for x in (k_scales, v_scales)]
        elif k_scales is not None or v_scales is not None:
            raise g4.G4Error(1, "f16 pages have no scales")
        self.c = KVPagesStruct(_address(k, "k pages", device), _address(v, "v pages", device), s[0], s[1], kind,
                               pages, slots, heads, dim, page_stride, slot, head)
        self.ref = ctypes.byref(self.c)


class Chunk:
    """The new tokens of a batch: q_start int32 [seqs + 1], kv_len int32 [seqs], page_table int32
    [seqs][pages of a sequence], on the device (read when the kernels run). tokens: rows of the chunk;
    max_q, max_kv: the most rows and positions that a sequence has. Keeps its buffers alive."""

    def __init__(self, q_start, kv_len, page_table, tokens, max_q, max_kv):
        device = self.device = _device()
        at, seqs, width, stride = _table(page_table, device)
        self.buffers = (q_start, kv_len, page_table)
        self.seqs, self.tokens, self.max_q, self.max_kv = seqs, int(tokens), int(max_q), int(max_kv)
        self.c = ChunkStruct(seqs, self.tokens, self.max_q, self.max_kv,
                             _packed(q_start, "q_start", _I32, (seqs + 1,), device),
                             _packed(kv_len, "kv_len", _I32, (seqs,), device), at, width, stride)
        self.ref = ctypes.byref(self.c)


def paged_prologue(pages, chunk, q, k, v, q_out, q_gain=None, k_gain=None, cos=None, sin=None, eps=1e-6,
                   x_scale=1.0, q_scale=None, k_scale=None, v_scale=None, stream=None):
    """g4_paged_prologue: q / k norm and RoPE of a chunk, q out as f16, k and v stored in the cache.
    q [tokens][heads][head_dim], k and v [tokens][kv_heads][head_dim], of one type (f32, f16, or int8
    codes times q_scale / k_scale / v_scale, each x_scale where not given); their tokens may lie apart.
    q and q_out None: only the store; k and v None: only the queries."""
    d, t, device = pages.head_dim, chunk.tokens, _call_device(pages, chunk)
    kind, heads = None, 0
    qa = ka = va = (None, None, 0)
    qo = None
    if (k is None) != (v is None):
        raise g4.G4Error(1, "paged-prologue needs k and v together")
    if (q is None) != (q_out is None):
        raise g4.G4Error(1, "paged-prologue needs q and q_out together")
    if q is not None:
        heads = int(q.shape[1])
        qa = _rows(q, "q", _X_KINDS, heads, d, t, device)
        qo = _packed(q_out, "q_out", _F16, (t, heads, d), device)
        kind = qa[1]
    if k is not None:
        ka = _rows(k, "k", _X_KINDS, pages.kv_heads, d, t, device)
        va = _rows(v, "v", _X_KINDS, pages.kv_heads, d, t, device)
        if va[1] != ka[1] or kind not in (None, ka[1]):
            raise g4.G4Error(1, "paged-prologue: q, k and v must be of one type")
        kind = ka[1]
    qg = None if q_gain is None else _packed(q_gain, "q_gain", _F32, (d,), device)
    kg = None if k_gain is None else _packed(k_gain, "k_gain", _F32, (d,), device)
    tab_c, tab_s, positions = None, None, 0
    if cos is not None or sin is not None:
        if cos is None or sin is None:
            raise g4.G4Error(1, "paged-prologue needs cos and sin together")
        positions = int(cos.shape[0])
        tab_c = _packed(cos, "cos", _F32, (positions, d // 2), device)
        tab_s = _packed(sin, "sin", _F32, (positions, d // 2), device)
    st = g4.lib().g4_paged_prologue(
        pages.ref, chunk.ref, g4.KIND_F32 if kind is None else kind, qa[0], qa[2],
        x_scale if q_scale is None else q_scale, ka[0], ka[2], x_scale if k_scale is None else k_scale, va[0], va[2],
        x_scale if v_scale is None else v_scale, heads, qg, kg, tab_c, tab_s, positions, eps, qo,
        _stream(stream, device, *pages.buffers, *chunk.buffers, q, k, v, q_out, q_gain, k_gain, cos, sin))
    if st:
        g4._check(st)


def kv_read(pages, chunk, k_out, v_out, stream=None):
    """g4_kv_read: the chunk's rows back from the cache, f32 or f16, to [tokens][kv_heads][head_dim],
    or to [seqs][rows][kv_heads][head_dim] with rows >= max_q (row i of a sequence at [s][i]; the rest
    is left as it was). k_out or v_out may be None."""
    device, kinds, at = _call_device(pages, chunk), [], []
    for x, what in ((k_out, "k_out"), (v_out, "v_out")):
        if x is None:
            at.append(None)
            continue
        if len(x.shape) == 4:
            rows = int(x.shape[1])
            if rows < min(chunk.max_q, chunk.tokens):
                raise g4.G4Error(1, f"{what} holds {rows} rows a sequence, max_q is {chunk.max_q}")
            want = (chunk.seqs, rows, pages.kv_heads, pages.head_dim)
        else:
            rows, want = 0, (chunk.tokens, pages.kv_heads, pages.head_dim)
        at.append(_packed(x, what, (g4.KIND_F32, g4.KIND_F16), want, device))
        kinds.append((_kind(x), rows * pages.kv_heads * pages.head_dim))
    if not kinds or kinds[0] != kinds[-1]:
        raise g4.G4Error(1, "kv-read needs k_out and v_out of one type and layout, or one of them")
    st = g4.lib().g4_kv_read(pages.ref, chunk.ref, at[0], at[1], kinds[0][0], kinds[0][1],
                            _stream(stream, device, *pages.buffers, *chunk.buffers, k_out, v_out))
    if st:
        g4._check(st)


def attention_chunk_workspace_bytes(pages, chunk, heads, window=0) -> int:
    n = g4.lib().g4_attention_chunk_workspace_bytes(pages.ref, chunk.ref, heads, window)
    if not n:
        raise g4.G4Error(1, f"attention-chunk: no such call ({heads} heads on {pages.kv_heads}, window {window})")
    return n


def attention_chunk(pages, chunk, q, out, workspace, scale=1.0, window=0, in_scale=0.0, stream=None):
    """g4_attention_chunk: causal attention of the chunk's rows over the cache. q f16 [tokens][heads]
    [head_dim] (tokens may lie apart); out f16, f32, or int8 codes on in_scale, packed."""
    heads, device = int(q.shape[1]), _call_device(pages, chunk)
    qp, _, stride = _rows(q, "q", _F16, heads, pages.head_dim, chunk.tokens, device)
    op = _packed(out, "out", _X_KINDS, (chunk.tokens, heads, pages.head_dim), device)
    st = g4.lib().g4_attention_chunk(pages.ref, chunk.ref, qp, stride, heads, scale, window,
                                     *_workspace(workspace, device), op, _kind(out), in_scale,
                                     _stream(stream, device, *pages.buffers, *chunk.buffers, q, out, workspace))
    if st:
        g4._check(st)


def verify_workspace_bytes(seqs, drafts, vocab) -> int:
    n = g4.lib().g4_verify_workspace_bytes(seqs, drafts, vocab)
    if not n:
        raise g4.G4Error(1, f"verify-drafts: no such call ({seqs} sequences, {drafts} drafts, vocabulary {vocab})")
    return n


def verify_drafts(logits, draft_logits, draft_tokens, draft_start, u, u_next, tokens, accepted, logprobs,
                  workspace, cap=0.0, temperature=1.0, stream=None):
    """g4_verify_drafts. logits f32 [drafts + seqs][vocab] (each sequence's drafts and one more row),
    draft_logits f32 [drafts][vocab] or None, draft_tokens int32 [drafts], draft_start int32 [seqs + 1],
    u f32 [drafts] and u_next f32 [seqs] in [0, 1) (None when greedy); tokens int32 and logprobs f32 (or
    None) [seqs][max_drafts + 1] and accepted int32 [seqs] out."""
    device = _device()
    seqs, drafts = int(draft_start.shape[0]) - 1, int(draft_tokens.shape[0])
    vocab, width = int(logits.shape[1]), int(tokens.shape[1])
    st = g4.lib().g4_verify_drafts(
        _packed(logits, "logits", _F32, (drafts + seqs, vocab), device),
        None if draft_logits is None else _packed(draft_logits, "draft_logits", _F32, (drafts, vocab), device),
        _packed(draft_tokens, "draft_tokens", _I32, (drafts,), device),
        _packed(draft_start, "draft_start", _I32, (seqs + 1,), device), seqs, drafts, width - 1, vocab, cap, temperature,
        None if u is None else _packed(u, "u", _F32, (drafts,), device),
        None if u_next is None else _packed(u_next, "u_next", _F32, (seqs,), device),
        *_workspace(workspace, device), _packed(tokens, "tokens", _I32, (seqs, width), device),
        _packed(accepted, "accepted", _I32, (seqs,), device),
        None if logprobs is None else _packed(logprobs, "logprobs", _F32, (seqs, width), device),
        _stream(stream, device, logits, draft_logits, draft_tokens, draft_start, u, u_next, tokens, accepted, logprobs,
                workspace))
    if st:
        g4._check(st)


class FreePagesStruct(ctypes.Structure):
    """include/g4serve.h g4_free_pages."""
    _fields_ = [("pages", _vp), ("count", _vp), ("capacity", ctypes.c_int), ("num_pages", ctypes.c_int),
                ("page_size", ctypes.c_int)]


class AdaptersStruct(ctypes.Structure):
    """include/g4serve.h g4_adapters."""
    _fields_ = [("a", _vp), ("b", _vp), ("scales", _vp), ("ranks", _vp), ("count", ctypes.c_int),
                ("max_rank", ctypes.c_int), ("k", ctypes.c_int), ("n", ctypes.c_int), ("a_stride", ctypes.c_int64),
                ("b_stride", ctypes.c_int64)]


def _need_device(x, device, what):
    if x.device != device:
        raise g4.G4Error(1, f"{what} are on another device than the current one")


def _optional(x, what, kinds, shape, device):
    return None if x is None else _packed(x, what, kinds, shape, device)


def _table(page_table, device):
    """(address, sequences, pages, elements between rows) of a page table."""
    try:
        if (page_table.get_device() == device and _one_runtime and page_table.dim() == 2 and page_table.is_contiguous()
                and _kinds[page_table.dtype] == g4.KIND_I32):
            seqs, width = page_table.shape
            return page_table.data_ptr(), seqs, width, width
    except (AttributeError, KeyError):
        pass
    if len(page_table.shape) != 2:
        raise g4.G4Error(1, f"page_table has shape {list(page_table.shape)}, expected [seqs][pages]")
    seqs, width = (int(n) for n in page_table.shape)
    stride = width
    if hasattr(page_table, "stride"):
        st = page_table.stride()
        if (width > 1 and st[1] != 1) or (seqs > 1 and st[0] < width):
            raise g4.G4Error(1, "page_table rows must be packed")
        stride = st[0] if seqs > 1 else width
    if _kind(page_table) != g4.KIND_I32:
        raise g4.G4Error(1, f"page_table cannot be {page_table.dtype}")
    return _address(page_table, "page_table", device), seqs, width, stride


class FreePages:
    """The pages that no sequence holds: pages int32 [capacity], of which the first count (int32 [1]) are
    free. A plan or a release reads them and writes the count it leaves elsewhere: make one FreePages for each of
    two count buffers, on the same pages, and take them in turn. Keeps its buffers alive."""

    def __init__(self, pages, count, num_pages, page_size):
        device = self.device = _device()
        self.buffers = (pages, count)
        capacity = int(pages.shape[0])
        self.c = FreePagesStruct(_packed(pages, "free pages", _I32, (capacity,), device),
                                 _packed(count, "count", _I32, (1,), device), capacity, int(num_pages), int(page_size))
        self.ref = ctypes.byref(self.c)


def plan_chunk(free, cached, rows, page_table, q_start, kv_len, free_left, served, tokens, max_q, max_kv, held=None,
               held_out=None, seq_adapter=None, row_pos=None, row_slot=None, row_adapter=None, last_row=None,
               stream=None):
    """g4_plan_chunk: the arrays of a Chunk (q_start [seqs + 1], kv_len [seqs], new entries of page_table) from
    each request's cached positions and rows (int32 [seqs]), the free list's new count (free_left [1]), the number of
    sequences served ([1]), and optionally held_out and last_row [seqs], row_pos, row_slot and row_adapter [tokens];
    all int32."""
    device = _device()
    _need_device(free, device, "the free pages")
    at, seqs, width, stride = _table(page_table, device)
    each, row, one = (seqs,), (tokens,), (1,)
    st = g4.lib().g4_plan_chunk(
        free.ref,
        cached if cached is None else _packed(cached, "cached", _I32, each, device),
        rows if rows is None else _packed(rows, "rows", _I32, each, device),
        held if held is None else _packed(held, "held", _I32, each, device),
        seq_adapter if seq_adapter is None else _packed(seq_adapter, "seq_adapter", _I32, each, device),
        seqs, tokens, max_q, max_kv, at, width, stride,
        _packed(q_start, "q_start", _I32, (seqs + 1,), device), _packed(kv_len, "kv_len", _I32, each, device),
        held_out if held_out is None else _packed(held_out, "held_out", _I32, each, device),
        _packed(free_left, "free_left", _I32, one, device), _packed(served, "served", _I32, one, device),
        row_pos if row_pos is None else _packed(row_pos, "row_pos", _I32, row, device),
        row_slot if row_slot is None else _packed(row_slot, "row_slot", _I32, row, device),
        row_adapter if row_adapter is None else _packed(row_adapter, "row_adapter", _I32, row, device),
        last_row if last_row is None else _packed(last_row, "last_row", _I32, each, device),
        _stream(stream, device, page_table, q_start, kv_len, free_left, served, cached, rows, held, seq_adapter, held_out,
                row_pos, row_slot, row_adapter, last_row, *free.buffers))
    if st:
        g4._check(st)


def release_pages(free, page_table, first, last, count_out, stream=None):
    """g4_release_pages: entries first[s] .. last[s] - 1 (int32 [seqs]) of every sequence's row of page_table back to the
    free pages, but for absent ones; count_out int32 [1] is the new count."""
    device = _device()
    _need_device(free, device, "the free pages")
    at, seqs, width, stride = _table(page_table, device)
    st = g4.lib().g4_release_pages(
        free.ref, at, width, stride, _packed(first, "first", _I32, (seqs,), device), _packed(last, "last", _I32, (seqs,), device),
        seqs, _packed(count_out, "count_out", _I32, (1,), device),
        _stream(stream, device, *free.buffers, page_table, first, last, count_out))
    if st:
        g4._check(st)


class Adapters:
    """Low-rank adapters of one linear: a f16 [count][max_rank][k] and b f16 [count][n][max_rank] (adapters may lie
    apart, each packed), scales f32 [count] (1 where not given), ranks int32 [count] (max_rank). Keeps its buffers alive."""

    def __init__(self, a, b, scales=None, ranks=None):
        if len(a.shape) != 3 or len(b.shape) != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise g4.G4Error(1, f"adapters need a [count][max_rank][k] and b [count][n][max_rank], got {list(a.shape)} and "
                                f"{list(b.shape)}")
        device = self.device = _device()
        count, rank, k = (int(n) for n in a.shape)
        n = int(b.shape[1])
        self.buffers, self.count, self.k, self.n = (a, b, scales, ranks), count, k, n
        at = []
        for x, what, rows, width in ((a, "a", rank, k), (b, "b", n, rank)):
            if _kind(x) != g4.KIND_F16:
                raise g4.G4Error(1, f"{what} cannot be {x.dtype}")
            stride = rows * width
            if hasattr(x, "stride"):
                st = x.stride()
                if (width > 1 and st[2] != 1) or (rows > 1 and st[1] != width) or (count > 1 and st[0] < stride):
                    raise g4.G4Error(1, f"{what}: an adapter must be packed, and adapters apart")
                stride = st[0] if count > 1 else stride
            at.append((_address(x, what, device), stride))
        self.c = AdaptersStruct(at[0][0], at[1][0], _optional(scales, "scales", _F32, (count,), device),
                                _optional(ranks, "ranks", _I32, (count,), device), count, rank, k, n, at[0][1], at[1][1])
        self.ref = ctypes.byref(self.c)


def adapter_groups_bytes(tokens, adapters) -> int:
    n = g4.lib().g4_adapter_groups_bytes(tokens, adapters)
    if not n:
        raise g4.G4Error(1, f"adapter-groups: no such call ({tokens} tokens, {adapters} adapters)")
    return n


def adapter_groups(row_adapter, groups, adapters, stream=None):
    """g4_adapter_groups: the rows of a batch by adapter, for every adapter_linear of a step. row_adapter int32
    [tokens] (-1: none, -2: no row), groups adapter_groups_bytes(tokens, adapters) bytes."""
    device = _device()
    tokens = int(row_adapter.shape[0])
    st = g4.lib().g4_adapter_groups(_packed(row_adapter, "row_adapter", _I32, (tokens,), device), tokens, adapters,
                                    *_workspace(groups, device), _stream(stream, device, row_adapter, groups))
    if st:
        g4._check(st)


def adapter_workspace_bytes(adapters, tokens) -> int:
    n = g4.lib().g4_adapter_workspace_bytes(adapters.ref, tokens)
    if not n:
        raise g4.G4Error(1, f"adapter-linear: no such call ({tokens} tokens, adapters {list(adapters.buffers[0].shape)} and "
                            f"{list(adapters.buffers[1].shape)})")
    return n


def _matrix(x, what, tokens, width, device):
    """(address, kind, elements between rows) of [tokens][width], whose rows may lie apart."""
    try:
        if (x.get_device() == device and _one_runtime and x.shape == (tokens, width) and x.is_contiguous()
                and _kinds[x.dtype] in _X_KINDS):
            return x.data_ptr(), _kinds[x.dtype], width
    except (AttributeError, KeyError):
        pass
    kind = _kind(x)
    if kind not in _X_KINDS:
        raise g4.G4Error(1, f"{what} cannot be {x.dtype}")
    if x.shape != (tokens, width):
        raise g4.G4Error(1, f"{what} has shape {list(x.shape)}, expected {[tokens, width]}")
    stride = width
    if hasattr(x, "stride"):
        st = x.stride()
        if (width > 1 and st[1] != 1) or (tokens > 1 and st[0] < width):
            raise g4.G4Error(1, f"{what}: rows must be packed, and apart")
        stride = st[0] if tokens > 1 else width
    return _address(x, what, device), kind, stride


def adapter_linear(adapters, groups, x, base, out, workspace, x_scale=1.0, base_scale=1.0, out_scale=0.0, stream=None):
    """g4_adapter_linear: out = base + scale * (x A^T) B^T with each row's adapter. x [tokens][k] and base (or None)
    [tokens][n]: f32, f16 or int8 codes on x_scale / base_scale; out f32, f16, or int8 codes on out_scale; out may be
    base, not x. groups: of adapter_groups, for as many tokens."""
    device = _device()
    _need_device(adapters, device, "the adapters")
    tokens = int(x.shape[0])
    xa = _matrix(x, "x", tokens, adapters.k, device)
    ba = (None, g4.KIND_F32, 0) if base is None else _matrix(base, "base", tokens, adapters.n, device)
    oa = _matrix(out, "out", tokens, adapters.n, device)
    st = g4.lib().g4_adapter_linear(adapters.ref, *_workspace(groups, device), tokens, *xa, x_scale, *ba, base_scale, *oa,
                                    out_scale, *_workspace(workspace, device),
                                    _stream(stream, device, *adapters.buffers, groups, x, base, out, workspace))
    if st:
        g4._check(st)


def sample_workspace_bytes(rows, vocab) -> int:
    n = g4.lib().g4_sample_workspace_bytes(rows, vocab)
    if not n:
        raise g4.G4Error(1, f"sample-tokens: no such call ({rows} rows, vocabulary {vocab})")
    return n


def sample_tokens(logits, u, tokens, logprobs, workspace, row_index=None, temperature=None, top_k=None, top_p=None,
                  min_p=None, cap=0.0, stream=None):
    """g4_sample_tokens. logits f32 [rows of logits][vocab] (rows may lie apart), u f32 [rows] in [0, 1), tokens int32 and
    logprobs f32 (or None) [rows] out; optional: row_index and top_k int32, temperature, top_p and min_p f32 [rows]."""
    device = _device()
    if len(logits.shape) != 2:
        raise g4.G4Error(1, f"logits has shape {list(logits.shape)}, expected [rows][vocab]")
    logit_rows, vocab, rows = int(logits.shape[0]), int(logits.shape[1]), int(u.shape[0])
    at, kind, stride = _matrix(logits, "logits", logit_rows, vocab, device)
    if kind != g4.KIND_F32:
        raise g4.G4Error(1, f"logits cannot be {logits.dtype}")
    given = [_optional(x, what, kinds, (rows,), device) for x, what, kinds in (
        (row_index, "row_index", _I32), (temperature, "temperature", _F32), (top_k, "top_k", _I32), (top_p, "top_p", _F32),
        (min_p, "min_p", _F32))]
    st = g4.lib().g4_sample_tokens(
        at, logit_rows, stride, given[0], rows, vocab, cap, *given[1:], _packed(u, "u", _F32, (rows,), device),
        *_workspace(workspace, device), _packed(tokens, "tokens", _I32, (rows,), device),
        _optional(logprobs, "logprobs", _F32, (rows,), device),
        _stream(stream, device, logits, u, tokens, logprobs, workspace, row_index, temperature, top_k, top_p, min_p))
    if st:
        g4._check(st)
