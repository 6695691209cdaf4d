"""Batches for the serving operators' tests: a paged cache built on the host, its descriptors on the
device, and plain 64-bit forms of the operators."""
import numpy as np

import g4serve as gs
import g4w8a8 as g4


class View:
    """A window into a device buffer: the last axes packed, the leading ones `strides` elements apart."""

    def __init__(self, base, offset, shape, strides, dtype):
        self.base, self.shape, self.dtype = base, tuple(shape), np.dtype(dtype)
        self._strides = tuple(strides)
        self.ptr = base.ptr + offset * self.dtype.itemsize

    def stride(self):
        return self._strides


def dev(a):
    return g4.DeviceBuffer.from_array(a)


def quantise(x):
    """Codes and scales of f32 rows, by the definition in 64 bits (a zero row: scale 0)."""
    amax = np.abs(x).max(-1)
    scale = (amax / np.float32(127)).astype(np.float32)
    safe = np.where(amax == 0, 1, amax).astype(np.float64)
    codes = np.rint(127.0 * x.astype(np.float64) / safe[..., None]).astype(np.int8)
    return codes, scale


class Batch:
    """lens: (rows, positions) of each sequence. Rows of K and V are random; slots that no sequence
    uses hold NaN (f16) or large codes with NaN scales (int8). absent: (sequence, page) pairs left out."""

    def __init__(self, lens, kv_heads=1, dim=256, page=16, kind="i8", seed=0, absent=(), spare=2,
                 tail_rows=0, max_q=None, max_kv=None, extra_pages=0):
        r = np.random.default_rng(seed)
        self.lens, self.kind, self.dim, self.page, self.kv_heads = list(lens), kind, dim, page, kv_heads
        self.absent = set(absent)
        ms, kvs = [m for m, _ in lens], [kv for _, kv in lens]
        self.start = np.concatenate([[0], np.cumsum(ms)]).astype(np.int32)
        self.tokens = int(self.start[-1]) + tail_rows
        self.max_q = max(1, max(ms)) if max_q is None else max_q
        self.max_kv = max(1, max(kvs)) if max_kv is None else max_kv
        need = [-(-kv // page) for kv in kvs]
        width = -(-self.max_kv // page) + extra_pages
        self.pages_n = sum(need) + spare
        order = r.permutation(self.pages_n)
        self.table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (self.pages_n, page, kv_heads, dim)
        self.k32, self.v32 = (r.standard_normal(shape).astype(np.float32) for _ in range(2))
        used = np.zeros((self.pages_n, page), bool)
        for s, kv in enumerate(kvs):
            for p in range(kv):
                used[self.table[s, p // page], p % page] = True
        if kind == "f16":
            self.k, self.v = self.k32.astype(np.float16), self.v32.astype(np.float16)
            self.k[~used] = self.v[~used] = np.nan
            self.ks = self.vs = None
        else:
            (self.k, ks), (self.v, vs) = quantise(self.k32), quantise(self.v32)
            self.k[~used] = self.v[~used] = 127
            ks[~used] = vs[~used] = np.nan
            self.ks, self.vs = (np.ascontiguousarray(x.transpose(0, 2, 1)) for x in (ks, vs))
        for s, p in self.absent:  # the page exists, but the sequence has let go of it
            self.table[s, p] = -1 if (s + p) % 2 else self.pages_n + 7
        self.rng = r

    def upload(self):
        self.dk, self.dv = dev(self.k), dev(self.v)
        self.dks, self.dvs = (None, None) if self.ks is None else (dev(self.ks), dev(self.vs))
        self.pages = gs.KVPages(self.dk, self.dv, self.dks, self.dvs)
        return self.describe()

    def describe(self):
        self.chunk = gs.Chunk(dev(self.start), dev(np.array([kv for _, kv in self.lens], np.int32)),
                              dev(self.table), self.tokens, self.max_q, self.max_kv)
        return self

    def held(self, pool, scales, s):
        """Sequence s's rows in 64 bits [positions][kv_heads][dim], and which of them are present."""
        kv = self.lens[s][1]
        p = np.arange(kv)
        page = self.table[s, p // self.page]
        there = (page >= 0) & (page < self.pages_n)
        page = np.where(there, page, 0)
        x = pool[page, p % self.page].astype(np.float64)
        if scales is not None:
            x = x * scales.astype(np.float64)[page, :, p % self.page][..., None]
        return x, there

    def workspace(self, heads, window):
        return g4.DeviceBuffer(gs.attention_chunk_workspace_bytes(self.pages, self.chunk, heads, window))


def attention(b, q, scale, window):
    """(out, bound) in 64 bits [tokens][heads][dim]; bound: how far a kernel that adds in f32, rounds the
    softmax weights to f16 and the output not at all may be off.

    With |s~ - s| <= ds the weights are off by a factor within e^(2 ds) (numerator and sum), and by 2^-11
    of their own from the rounding to f16; one under 2^-14 of the row's largest loses up to 2^-25 of that.
    A weight is relative to a running maximum whose factor exp(m - m') is applied once more in f32. Sums
    of n terms in f32 lose (n + 8) 2^-24 of the sum of magnitudes. ds is the f32 dot product's (dim + 4)
    2^-24 of its magnitudes, and exp's few 2^-24; with an int8 cache an element of q may be off by half a step
    of 2^-15 of the row's largest (32512 steps) too, so a score by that times the sum of |k|."""
    heads = q.shape[1]
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    group = heads // b.kv_heads
    for s, (m, kv) in enumerate(b.lens):
        k, there = b.held(b.k, b.ks, s)
        v, _ = b.held(b.v, b.vs, s)
        pos = kv - m + np.arange(m)
        j = np.arange(kv)
        seen = there & (j <= pos[:, None])
        if window:
            seen &= j > pos[:, None] - window
        for h in range(heads):
            kk, vv = (np.where(there[:, None], x[:, h // group], 0) for x in (k, v))
            qq = q[b.start[s]:b.start[s + 1], h].astype(np.float64)
            sc = np.where(seen, qq @ kk.T * scale, -np.inf)
            mag = np.where(seen, np.abs(qq) @ np.abs(kk).T * abs(scale), 0)
            if not kv:
                continue
            top = sc.max(1, keepdims=True)
            top = np.where(np.isfinite(top), top, 0)
            p = np.where(seen, np.exp(sc - top), 0)
            tot = p.sum(1, keepdims=True)
            tot = np.where(tot == 0, 1, tot)
            p = p / tot
            sl = np.s_[b.start[s]:b.start[s + 1], h]
            out[sl] = p @ vv
            ds = (mag.max(1, keepdims=True, initial=0) * (b.dim + 4) + 16) * 2.0 ** -24
            if b.kind == "i8":
                ds = ds + np.abs(qq).max(1, keepdims=True, initial=0) / 65024 * \
                    np.abs(kk).sum(1).max(initial=0) * abs(scale)
            n = seen.sum(1, keepdims=True)
            spread = p @ np.abs(vv)
            vmax = np.abs(vv).max(initial=0)
            bound[sl] = spread * (4 * ds + 2.0 ** -11 + 2 * (n + 8) * 2.0 ** -24) + n * 2.0 ** -25 * vmax / tot
    return out, bound


def to_kind(y, bound, kind):
    """The bound of an output of this type: half a step of it on top (f16: 2^-11, subnormals 2^-25)."""
    if kind == np.float16:
        return bound + np.maximum(np.abs(y) * 2.0 ** -11, 2.0 ** -25) * 1.01
    return bound + np.abs(y) * 2.0 ** -24
