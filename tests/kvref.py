"""Reference of the attention side in 64 bits (numpy): paged caches, norm and rotation, attention, and their GPU glue."""
import numpy as np

import oracle as O
from brimkern_amd.capi import Context

f32, f64 = np.float32, np.float64


def quantize(fmt, x):
    """Planes of f32 vectors [..., D], each plane with the leading shape kept."""
    x = np.ascontiguousarray(x, f32)
    lead, D = x.shape[:-1], x.shape[-1]
    if x.size == 0:
        shapes = [(D, np.int8)] if fmt == "q8" else [(D // 2, np.uint8)]
        return [np.zeros(lead + (n,), t) for n, t in shapes + [(D // 32, np.uint16)] * (1 if fmt == "q8" else 2)]
    planes = O.quantize_q8(x.ravel()) if fmt == "q8" else O.quantize_q4(x.ravel())
    return [np.asarray(p).reshape(lead + (-1,)) for p in planes]


def values(fmt, planes):
    """The f64 values of planes [..., D]."""
    h = [p.view(np.uint16).view(np.float16).astype(f64) for p in planes[1:]]
    if fmt == "q8":
        q = planes[0].view(np.int8).astype(f64)
        return q * np.repeat(h[0], 32, -1)
    c = planes[0].view(np.uint8)
    q = np.stack((c & 15, c >> 4), -1).reshape(c.shape[:-1] + (-1,)).astype(f64)
    return q * np.repeat(h[0], 32, -1) + np.repeat(h[1], 32, -1)


class Paged:
    """A cache of `pages` pages, its pages given out in a shuffled order; planes on the host."""

    def __init__(self, fmt, KV, D, P, pages, seed=0, fill=None):
        self.fmt, self.KV, self.D, self.P, self.pages = fmt, KV, D, P, pages
        rng = np.random.default_rng(seed)
        self.free = list(rng.permutation(pages))
        self.planes = {}
        for n in "kv":
            code = rng.integers(0, 256, (pages, KV, P, D if fmt == "q8" else D // 2), np.uint8)
            half = [np.full((pages, KV, P, D // 32), 0x7E00 if fill is None else fill, np.uint16)      # NaN: never written
                    for _ in range(1 if fmt == "q8" else 2)]
            self.planes[n] = [code.view(np.int8) if fmt == "q8" else code, *half]

    def take(self, tokens):
        """Page ids for `tokens` tokens."""
        return [self.free.pop() for _ in range(-(-tokens // self.P))]

    def put(self, ids, k, v):
        """Tokens [T, KV, D] (f32) into the pages `ids`, from slot 0."""
        for n, x in (("k", k), ("v", v)):
            q = quantize(self.fmt, x)
            for t in range(len(x)):
                for dst, src in zip(self.planes[n], q):
                    dst[ids[t // self.P], :, t % self.P] = src[t]

    def get(self, n, ids, tokens):
        """f64 values [tokens, KV, D] of the first tokens of the pages `ids`."""
        if not tokens:
            return np.zeros((0, self.KV, self.D))
        ids = np.asarray(ids)
        t = np.arange(tokens)
        return values(self.fmt, [p[ids[t // self.P], :, t % self.P] for p in self.planes[n]])


def rope_angles(pos, freq):
    return np.asarray(pos, f64)[:, None] * np.asarray(freq, f32).astype(f64)


def norm_rope(x, w, eps, one_plus, pos, freq, interleaved):
    """[T, heads, D] f32 -> f32: norm (w not None), rotation (freq not None), in 64 bits, rounded once."""
    y = np.asarray(x, f32).astype(f64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + f64(f32(eps))) * (np.asarray(w, f32).astype(f64) + (1 if one_plus else 0))
    if freq is not None:
        a = rope_angles(pos, freq)[:, None]
        half = a.shape[-1]
        i = np.arange(half)
        p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        u, v = y[..., p], y[..., q]
        y = y.copy()
        y[..., p], y[..., q] = u * np.cos(a) - v * np.sin(a), v * np.cos(a) + u * np.sin(a)
    return y.astype(f32)


def attention(q, k, v, scale, window=0, softcap=0.0, exists=None):
    """One sequence in f64: q [n, H, D] its last n rows, k and v [L, KV, D]; `exists` [L]: tokens that are there."""
    q = np.asarray(q, f64)
    n, H, D = q.shape
    L, KV = k.shape[:2]
    if L == 0:
        return np.zeros((n, H, D))
    j = np.arange(L)
    pos = L - n + np.arange(n)
    seen = j[None] <= pos[:, None]
    if window:
        seen &= j[None] > pos[:, None] - window
    if exists is not None:
        seen &= exists[None]
    some = seen.any(0)
    out = np.zeros((n, H, D))
    kk, vv = np.where(some[:, None, None], k, 0), np.where(some[:, None, None], v, 0)
    for h in range(H):
        g = h // (H // KV)
        x = (q[:, h] @ kk[:, g].T) * f64(f32(scale))
        if softcap:
            x = softcap * np.tanh(x / softcap)
        x = np.where(seen, x, -np.inf)
        top = np.where(seen.any(1), x.max(1, initial=-np.inf), 0.0)
        e = np.where(seen, np.exp(x - top[:, None]), 0.0)
        s = e.sum(1)
        out[:, h] = (e @ vv[:, g]) / np.where(s == 0, 1, s)[:, None]
    return out


class Dev:
    """Uploads for one test, freed at its end."""

    def __init__(self, ctx: Context):
        self.ctx, self.bufs = ctx, []

    def up(self, a):
        b = self.ctx.upload(np.ascontiguousarray(a))
        self.bufs.append(b)
        return b

    def room(self, *shape):
        """An f32 buffer of NaN."""
        return self.up(np.full(shape, np.nan, f32))

    def down(self, b, *shape):
        return self.ctx.download(b, f32, int(np.prod(shape))).reshape(shape)

    def i32(self, v):
        return self.up(np.asarray(v, np.int32).ravel())

    def cache(self, c: Paged):
        self.pk, self.pv = [self.up(p) for p in c.planes["k"]], [self.up(p) for p in c.planes["v"]]
        return self.ctx.kv_cache(c.fmt, c.KV, c.D, c.P, c.pages, self.pk, self.pv)

    def planes(self, c: Paged):
        """The device's planes, into the host cache's arrays (a copy)."""
        out = {}
        for n, bufs in (("k", self.pk), ("v", self.pv)):
            out[n] = [self.ctx.download(b, p.dtype, p.size).reshape(p.shape) for b, p in zip(bufs, c.planes[n])]
        return out

    def batch(self, rows, lens, tables, cols=None, row_off=True, prefix=None, max_len=None, total=None):
        """rows, lens, tables (page id lists) per sequence; prefix: (page ids, tokens)."""
        cols = max([len(t) for t in tables] + [1]) if cols is None else cols
        tab = np.full((len(rows), cols), -1, np.int32)
        for b, t in enumerate(tables):
            tab[b, :len(t)] = t[:cols]
        off = np.concatenate(([0], np.cumsum(rows))).astype(np.int32)
        return self.ctx.kv_batch(seqs=len(rows), rows=int(off[-1]) if total is None else total, kv_len=self.i32(lens), table=self.i32(tab),
                                 table_cols=cols, max_len=max(lens) if max_len is None else max_len,
                                 row_off=self.i32(off) if row_off else None, max_rows=max(rows),
                                 prefix_len=prefix[1] if prefix else 0, prefix_table=self.i32(prefix[0]) if prefix else None)

    def free(self):
        for b in self.bufs:
            self.ctx.free(b)
        self.bufs.clear()
