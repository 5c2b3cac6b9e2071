"""Attention over the quantized cache (brik_attention) against a 64-bit softmax over the same planes.

Tolerance. Every product of the kernels is exact or off by at most 2^-22 of its operands (two halves), sums are f32. A score
is a sum of D products with partial sums of at most X = max |x| / scale: sqrt(D) roundings' worth of 2^-24 X, taken
twice for the split operand and the group sums; on scores up to about 10 and D up to 256 that is 2 * 16 * 6e-8 * 10 =
2e-5 absolute in the worst row and a third of it in the rms. It enters every weight with its own sign, so a row's
relative error (2-norm over the row's outputs) stays below 1e-5; the sums over keys add sqrt(keys) * 2^-24. NORM is twice
that. Rows with large scores, where one key takes all, are held to the same bound times max |x| / 10."""
import numpy as np
import pytest

import kvref as R
from brimkern_amd import synth
from brimkern_amd.capi import (BrikError, BRIK_EALIGN, BRIK_EINVAL, BRIK_OPT_ATTN_ROWS, BRIK_OPT_ATTN_SPLITS, Context)

pytestmark = pytest.mark.gpu
f32 = np.float32
NORM = 2e-5


@pytest.fixture()
def dev(ctx):
    d = R.Dev(ctx)
    yield d
    d.free()


class Case:
    """A batch over a filled cache, its device handles and the reference's answer."""

    def __init__(self, dev, fmt, H, KV, D, P, rows, lens, prefix=0, seed=0, window=0, softcap=0.0, kscale=1.0, vscale=1.0,
                 qscale=1.0, bad=(), row_off=True, scale=None, behind=0, slack=0, fill=None):
        rng = np.random.default_rng(1000 + seed)
        self.dev, self.H, self.KV, self.D, self.rows, self.lens = dev, H, KV, D, rows, lens
        self.scale = 1 / np.sqrt(D) if scale is None else scale
        self.window, self.softcap, self.prefix = window, softcap, prefix
        own = [n - prefix for n in lens]
        pages = sum(-(-max(n, 0) // P) for n in own) + -(-prefix // P) + 2
        self.c = c = R.Paged(fmt, KV, D, P, pages, seed=seed, fill=fill)

        def vec(n, s):
            return (rng.standard_normal((n, KV, D)) * np.exp(0.4 * rng.standard_normal((KV, D))) * s).astype(f32)
        self.pre = c.take(prefix)
        c.put(self.pre, vec(prefix, kscale), vec(prefix, vscale))
        self.tables = []
        for n in own:
            ids = c.take(max(n, 0))
            c.put(ids, vec(max(n, 0), kscale), vec(max(n, 0), vscale))
            self.tables.append(ids)
        self.shown = [list(t) for t in self.tables]
        for b, col, page in bad:
            self.shown[b][col] = page
        self.T = sum(rows)
        self.q = (rng.standard_normal((self.T + behind, H, D)) * qscale).astype(f32)
        self.cache = dev.cache(c)
        self.batch = dev.batch(rows, lens, self.shown, row_off=row_off, prefix=(self.pre, prefix) if prefix else None,
                               total=self.T + behind, max_len=max(lens + [1]) + slack)
        self.out = dev.room(self.T + behind, H, D)
        self.args = dev.ctx.attn_args(q=dev.up(self.q), out=self.out, heads=H, scale=self.scale, window=window, softcap=softcap)

    def run(self):
        self.dev.ctx.attention(self.cache, self.batch, self.args)
        return self.dev.down(self.out, *self.q.shape)

    def want(self, q=None, lens=None):
        q, at, out = self.q if q is None else q, 0, []
        for b, n in enumerate(self.rows):
            L = (self.lens if lens is None else lens)[b]
            own = max(L - self.prefix, 0)
            k, v = (np.concatenate((self.c.get(w, self.pre, min(self.prefix, L)), self.c.get(w, self.tables[b], own))) for w in "kv")
            there = np.ones(len(k), bool)
            for p in range(own):
                there[self.prefix + p if self.prefix else p] = 0 <= self.shown[b][p // self.c.P] < self.c.pages
            out.append(R.attention(q[at:at + n], k, v, self.scale, self.window, self.softcap, there))
            at += n
        return np.concatenate(out) if out else np.zeros((0, self.H, self.D))

    def check(self, tol=NORM):
        got, want = self.run(), self.want()
        close(got[:self.T], want, tol)
        assert np.isnan(got[self.T:]).all()                       # rows behind the last sequence: as they were
        return got


def close(got, want, tol=NORM):
    assert np.isfinite(got).all()
    n = np.sqrt((want ** 2).sum(-1))
    off = np.sqrt(((got - want) ** 2).sum(-1))
    assert (got[n == 0] == 0).all()
    rel = off / np.where(n == 0, 1, n)
    assert rel.max(initial=0) <= tol, (rel.max(), np.unravel_index(rel.argmax(), rel.shape))


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("H,KV,D,P", [(32, 8, 128, 64), (14, 2, 64, 16), (3, 3, 96, 32), (8, 1, 256, 128), (10, 2, 192, 16), (20, 1, 128, 256)])
def test_decode_lengths(dev, fmt, H, KV, D, P):
    """One row a sequence, lengths around the tiles' and pages' ends, among them none."""
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 300]
    Case(dev, fmt, H, KV, D, P, [1] * len(lens), lens, seed=D + H, row_off=False).check()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("H,KV,D,P,rows,lens", [
    (4, 2, 128, 16, [70], [70]),
    (32, 8, 128, 64, [3, 0, 1, 130], [500, 7, 1, 131]),
    (14, 2, 64, 32, [33, 64, 65], [33, 200, 65]),
    (2, 1, 256, 128, [129], [300]),
    (6, 2, 96, 16, [5, 20], [3, 19]),             # fewer tokens than rows: the first rows lie before the sequence
    (5, 5, 192, 64, [17, 16], [17, 1000]),
    (8, 8, 64, 64, [1, 257], [40, 513]),
    (24, 1, 128, 32, [6, 40, 11], [64, 95, 33]),
])
def test_many_rows(dev, fmt, H, KV, D, P, rows, lens):
    Case(dev, fmt, H, KV, D, P, rows, lens, seed=len(rows) + D, behind=2).check()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (17, 0.0), (64, 5.0), (100, 0.0), (0, 1.5), (1000, 50.0)])
def test_window_and_softcap(dev, fmt, window, softcap):
    Case(dev, fmt, 8, 2, 128, 32, [90, 1, 1, 40], [90, 333, 16, 200], window=window, softcap=softcap, seed=window, qscale=2.0).check()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("prefix", [1, 15, 16, 33, 200, 515])
@pytest.mark.parametrize("rows,own,window", [([1] * 7, [1, 2, 16, 17, 40, 65, 5], 0), ([3, 1, 20], [3, 50, 33], 0), ([1, 2, 5], [9, 30, 100], 48)])
def test_shared_prefix(dev, fmt, prefix, rows, own, window):
    Case(dev, fmt, 12, 3, 64, 16, rows, [prefix + n for n in own], prefix=prefix, window=window, seed=prefix).check()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_shared_prefix_rows_inside_it(dev, fmt):
    """Sequences that end inside the prefix see only its first tokens."""
    Case(dev, fmt, 4, 2, 128, 32, [1, 3, 2, 40], [100, 40, 1, 130], prefix=100, seed=5).check()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_prefix_gives_what_the_same_tokens_give_as_own(dev, fmt):
    """The prefix as its own pages of every sequence: the same answer within rounding."""
    a = Case(dev, fmt, 8, 2, 128, 16, [1, 2, 1], [150, 140, 131], prefix=130, seed=8)
    shared = a.run()
    tables = [list(a.pre) for _ in range(3)]
    c = a.c
    # the prefix ends inside a page: copy its last page and append the own tokens behind it
    for b, L in enumerate(a.lens):
        ids = c.take(0)
        need = -(-L // c.P) - len(a.pre)
        extra = [c.free.pop() if c.free else None for _ in range(need + 1)]
        if None in extra:
            break
        for n in "kv":
            for p in c.planes[n]:
                p[extra[0]] = p[a.pre[-1]]
                for t in range(L - 130):
                    at = 130 + t
                    col = at // c.P - (len(a.pre) - 1)
                    p[extra[col], :, at % c.P] = p[a.tables[b][t // c.P], :, t % c.P]
        one = dev.batch([a.rows[b]], [L], [tables[b][:-1] + extra])
        out = dev.room(a.rows[b], 8, 128)
        first = sum(a.rows[:b])
        dev.ctx.attention(dev.cache(c), one, dev.ctx.attn_args(q=dev.up(a.q[first:first + a.rows[b]]), out=out, heads=8, scale=a.scale))
        close(dev.down(out, a.rows[b], 8, 128), shared[first:first + a.rows[b]].astype(np.float64), 2 * NORM)
        break


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_pages_out_of_range_do_not_exist(dev, fmt):
    Case(dev, fmt, 4, 1, 64, 16, [1, 1, 40, 1], [100, 100, 90, 16], bad=[(0, 2, -1), (1, 0, 99), (1, 6, 1 << 30), (2, 1, -(1 << 31)), (3, 0, -1)],
         seed=3).check()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_max_len_and_table_end(dev, fmt):
    """Tokens past max_len or past the table are not attended to; a bound above the lengths changes nothing."""
    a = Case(dev, fmt, 4, 2, 64, 16, [1, 30], [90, 60], seed=1, slack=5000)
    whole = a.check()
    a.batch.max_len = 64
    got = a.run()
    short = R.attention(a.q[:1], a.c.get("k", a.tables[0], 64), a.c.get("v", a.tables[0], 64), a.scale)
    close(got[:1], short)
    assert np.abs(got[1:] - whole[1:]).max() <= 1e-5 * np.abs(whole).max()
    a.batch.max_len = 90
    b = dev.batch([1], [90], [a.tables[0]], cols=3)
    dev.ctx.attention(a.cache, b, a.args)
    close(dev.down(a.out, *a.q.shape)[:1], R.attention(a.q[:1], a.c.get("k", a.tables[0], 48), a.c.get("v", a.tables[0], 48), a.scale))


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_nan_and_infinity_stay_where_they_are(dev, fmt):
    """Scales of NaN and infinity in tokens a row does not see (slots never written are NaN in every test), a NaN row of q
    among others, and a token of infinity that its later rows do see."""
    a = Case(dev, fmt, 8, 2, 64, 16, [40, 1], [40, 50], seed=2)
    a.q[7, 3] = np.nan
    a.q[9, 5, 2] = np.inf
    dev.ctx.h2d(a.args.q, a.q)
    for n, p in (("k", dev.pk), ("v", dev.pv)):
        for plane, host in list(zip(p, a.c.planes[n]))[1:]:
            host[a.tables[0][30 // 16], :, 30 % 16] = 0x7C00          # token 30 of the first sequence
            dev.ctx.h2d(plane, host)
    got = a.run()
    q = a.q.copy()
    q[7, 3] = q[9, 5] = 0
    want = R.attention(q[:30], a.c.get("k", a.tables[0], 30), a.c.get("v", a.tables[0], 30), a.scale)
    clean = np.ones((30, 8), bool)
    clean[7, 3] = clean[9, 5] = False
    close(got[:30][clean], want[clean])
    assert np.isnan(got[7, 3]).all() and np.isnan(got[9, 5]).all()
    assert not np.isfinite(got[30:40]).all(-1).any()
    close(got[40:], R.attention(a.q[40:], a.c.get("k", a.tables[1], 50), a.c.get("v", a.tables[1], 50), a.scale))


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("kscale,vscale,qscale", [(1e-3, 1e-3, 1e3), (30.0, 3e3, 0.03), (1e3, 1.0, 1e-6), (1.0, 1e-2, 1e5)])
def test_magnitudes(dev, fmt, kscale, vscale, qscale):
    """Small and large keys, values and queries: the halves' range does not show. scale undoes what q and k do to the scores."""
    Case(dev, fmt, 8, 2, 128, 32, [1, 20], [300, 100], kscale=kscale, vscale=vscale, qscale=qscale, seed=4,
         scale=1 / np.sqrt(128) / (kscale * qscale)).check()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_peaked_scores(dev, fmt):
    """Scores of up to some hundreds, where one key takes all: no overflow, the error grows with the scores."""
    a = Case(dev, fmt, 8, 2, 128, 32, [1, 20], [300, 100], qscale=60.0, seed=6)
    a.check(NORM * 60)


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_values_of_very_different_size(dev, fmt):
    """Values whose scales differ by 2^20 from token to token: the large ones, far down in the softmax, still count."""
    a = Case(dev, fmt, 4, 1, 64, 16, [1, 3], [200, 90], seed=7)
    rng = np.random.default_rng(5)
    for ids, n in zip(a.tables, a.lens):
        v = (rng.standard_normal((n, 1, 64)) * 2.0 ** rng.integers(-10, 10, (n, 1, 1))).astype(f32)
        a.c.put(ids, a.c.get("k", ids, n).astype(f32), v)
    a.cache = dev.cache(a.c)
    a.check()


def test_negative_scales(dev):
    """Planes need not come from the encoder: a negative q8 scale is a value like another."""
    a = Case(dev, "q8", 4, 1, 64, 16, [1, 9], [77, 50], seed=9)
    for n in "kv":
        s = a.c.planes[n][1]
        s[...] = np.where((s & 0x7FFF) < 0x7C00, s ^ (np.arange(s.size).reshape(s.shape) % 3 == 0) * np.uint16(0x8000), s)
    a.cache = dev.cache(a.c)
    a.check()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_strides(dev, fmt):
    """q inside a packed q | k | v row, out inside a wider row: what lies between stays."""
    a = Case(dev, fmt, 4, 2, 64, 16, [5, 1], [30, 17], seed=11)
    wide = np.full((6, 4 * 64 + 12), np.nan, f32)
    wide[:, :256] = a.q.reshape(6, -1)
    ob = dev.room(6, 300)
    dev.ctx.attention(a.cache, a.batch, dev.ctx.attn_args(q=dev.up(wide), out=ob, heads=4, scale=a.scale, q_stride=268, out_stride=300))
    got = dev.down(ob, 6, 300)
    close(got[:, :256].reshape(6, 4, 64), a.want())
    assert np.isnan(got[:, 256:]).all()


@pytest.fixture(params=[(16, 1), (16, 5), (128, 0), (128, 1), (128, 3), (256, 1), (256, 7)], ids=lambda p: f"rows{p[0]}-splits{p[1]}")
def forced(request, ctx):
    """The kernels by tile rows, their keys whole or split, whatever the sizes would choose."""
    ctx.set_option(BRIK_OPT_ATTN_ROWS, request.param[0])
    ctx.set_option(BRIK_OPT_ATTN_SPLITS, request.param[1])
    yield request.param
    ctx.set_option(BRIK_OPT_ATTN_ROWS, 0)
    ctx.set_option(BRIK_OPT_ATTN_SPLITS, 0)


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("H,KV,D,P,rows,lens,more", [
    (8, 2, 128, 16, [70, 1, 0, 33], [70, 300, 5, 161], {}),
    (14, 2, 64, 64, [40, 3], [333, 2], dict(window=50)),
    (6, 3, 96, 32, [150, 20], [150, 90], dict(softcap=3.0, qscale=2.0)),
    (4, 1, 192, 128, [65], [200], dict(behind=3)),
    (10, 2, 256, 16, [30, 31], [97, 64], dict(window=17, softcap=20.0)),
    (12, 3, 64, 16, [1, 2, 40], [203, 230, 240], dict(prefix=200)),
    (8, 8, 128, 32, [20, 1], [90, 80], dict(prefix=77, window=60)),
    (4, 2, 128, 16, [5, 50], [40, 300], dict(bad=[(0, 1, -1), (1, 3, 1 << 20)])),
    (8, 2, 128, 32, [1, 60], [300, 100], dict(kscale=30.0, vscale=3e3, qscale=0.03, scale=0.1)),
    (8, 2, 64, 32, [33], [100], dict(scale=-0.2)),
])
def test_every_kernel(dev, forced, fmt, H, KV, D, P, rows, lens, more):
    c = Case(dev, fmt, H, KV, D, P, rows, lens, seed=D + H, **more)
    c.check()
    assert dev.ctx.last_kernel() == {16: "attn_few", 128: "attn_tile4", 256: "attn_tile4" if D > 128 else "attn_tile8"}[forced[0]]


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_every_kernel_on_hard_values(dev, forced, fmt, D):
    """Values of very different size, rows of NaN, tokens with scales that are not finite: seen by later rows only."""
    a = Case(dev, fmt, 4, 1, D, 16, [90, 3], [90, 64], seed=7)
    rng = np.random.default_rng(5)
    for ids, n in zip(a.tables, a.lens):
        v = (rng.standard_normal((n, 1, D)) * 2.0 ** rng.integers(-9, 10, (n, 1, 1))).astype(f32)
        a.c.put(ids, a.c.get("k", ids, n).astype(f32), v)
    a.cache = dev.cache(a.c)
    a.check()
    a.q[40, 2] = np.nan
    dev.ctx.h2d(a.args.q, a.q)
    want = a.want(np.nan_to_num(a.q))
    for n, p, t, g, bits in (("v", dev.pv, 60, 1, 0x7C00), ("v", dev.pv, 75, 0, 0xFE00)):
        a.c.planes[n][1][a.tables[0][t // 16], 0, t % 16, g] = bits
        dev.ctx.h2d(p[1], a.c.planes[n][1])
    got = a.run()
    assert np.isnan(got[40, 2]).all()
    ok = np.ones(got.shape[:2], bool)
    ok[40, 2] = False
    ok[60:90] = False
    close(got[ok], want[ok])
    assert not np.isfinite(got[60:90, :, 32:64]).any() and not np.isfinite(got[75:90, :, :32]).any()
    assert np.isfinite(got[60:75, :, :32]).all() and np.isfinite(got[60:90, :, 64:]).all()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("D,KV,H", [(64, 1, 4), (128, 2, 8), (96, 4, 4)])
def test_shared_out_keys(dev, fmt, D, KV, H):
    """Decoding of many sequences, one long: blocks end one sequence and begin the next, in the middle of 64 sequences and past
    them; sequences without keys, without rows, with fewer keys than a block takes."""
    rng = np.random.default_rng(D)
    lens = [int(x) for x in rng.integers(0, 120, 90)]
    lens[3], lens[50], lens[64], lens[66], lens[70], lens[89] = 1500, 0, 0, 700, 33, 0
    rows = [1] * 90
    rows[10] = rows[63] = rows[80] = 0
    rows[20] = 3
    lens[20] = 2
    Case(dev, fmt, H, KV, D, 32, rows, lens, seed=2).check()
    Case(dev, fmt, H, KV, D, 16, [1, 1, 1], [1100, 1, 2000], seed=3, window=700).check()


@pytest.mark.parametrize("D,lens", [(64, [2500, 700, 2180, 31]), (192, [3100]), (96, [1290, 1025])])
def test_joins_of_many_parts(dev, D, lens):
    """Every number of parts: weights come from other lanes of the wave that joins them."""
    a = Case(dev, "q8", 2, 1, D, 64, [1] * len(lens), lens, seed=4)
    a.check()
    for splits in (2, 3, 16, 17, 31, 33, 64, 65, 80):
        dev.ctx.set_option(BRIK_OPT_ATTN_SPLITS, splits)
        try:
            a.check()
        finally:
            dev.ctx.set_option(BRIK_OPT_ATTN_SPLITS, 0)


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("B,L", [(1, 5000), (3, 20000)])
def test_long(dev, fmt, B, L):
    """Long sequences: the keys are split over blocks and the pieces joined."""
    rng = np.random.default_rng(L)
    KV, D, P, H = 2, 128, 64, 8
    lens = [L - 777 * b for b in range(B)]
    pages = [-(-n // P) for n in lens]
    ids = rng.permutation(sum(pages) + 1)
    c = R.Paged(fmt, KV, D, P, sum(pages) + 1, seed=1, fill=0x2400)           # random codes, scale 2^-6, min 2^-6
    at = np.concatenate(([0], np.cumsum(pages)))
    tables = [list(ids[at[b]:at[b + 1]]) for b in range(B)]
    q = rng.standard_normal((B, H, D)).astype(f32)
    out = dev.room(B, H, D)
    dev.ctx.attention(dev.cache(c), dev.batch([1] * B, lens, tables, row_off=False),
                      dev.ctx.attn_args(q=dev.up(q), out=out, heads=H, scale=0.1 if fmt == "q8" else 0.5))
    for b in range(B):
        want = R.attention(q[b:b + 1], c.get("k", tables[b], lens[b]), c.get("v", tables[b], lens[b]), 0.1 if fmt == "q8" else 0.5)
        close(dev.down(out, B, H, D)[b:b + 1], want)


def test_many_sequences(dev):
    """More sequences than a wave has lanes, some without rows."""
    rows = [(b * 7) % 3 for b in range(150)]
    lens = [max(r, 1 + (b * 13) % 40) for b, r in enumerate(rows)]
    Case(dev, "q8", 2, 1, 64, 16, rows, lens, seed=1).check()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_cache_past_32_bit_offsets(dev, fmt):
    """Planes of over 4 GiB: tokens on the last pages are written, read back and attended to."""
    KV, D, P = 8, 128, 256
    slab = KV * P * (D if fmt == "q8" else D // 2)
    pages = (1 << 32) // slab + 8
    dev.ctx.sync()
    k, v = [[dev.ctx.alloc(pages * slab)] + [dev.ctx.alloc(pages * KV * P * D // 16) for _ in range(1 if fmt == "q8" else 2)] for _ in "kv"]
    dev.bufs += k + v
    rng = np.random.default_rng(1)
    n, rows = 300, (rng.standard_normal((2, 300, KV, D))).astype(f32)
    cache = dev.ctx.kv_cache(fmt, KV, D, P, pages, k, v)
    batch = dev.batch([n], [n], [[pages - 1, pages - 5]])
    dev.ctx.kv_write(cache, batch, dev.ctx.qkv_rows(head_dim=D, kv_heads=KV, k=dev.up(rows[0]), v=dev.up(rows[1])))
    ko, vo = dev.room(n, KV, D), dev.room(n, KV, D)
    dev.ctx.kv_read(cache, batch, ko, vo)
    want = [R.values(fmt, R.quantize(fmt, x)) for x in rows]
    assert np.array_equal(dev.down(ko, n, KV, D), want[0].astype(f32)) and np.array_equal(dev.down(vo, n, KV, D), want[1].astype(f32))
    q = rng.standard_normal((n, 16, D)).astype(f32)
    for m in (1, n):
        out = dev.room(m, 16, D)
        dev.ctx.attention(cache, dev.batch([m], [n], [[pages - 1, pages - 5]]),
                          dev.ctx.attn_args(q=dev.up(q[n - m:]), out=out, heads=16, scale=D ** -0.5))
        close(dev.down(out, m, 16, D), R.attention(q[n - m:], want[0], want[1], D ** -0.5))


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_same_call_twice_gives_the_same_bits(dev, fmt):
    a = Case(dev, fmt, 32, 8, 128, 64, [1] * 3 + [50], [900, 1, 400, 333], prefix=0, seed=13)
    first = a.run()
    Case(dev, fmt, 4, 2, 64, 16, [9], [100], seed=14).run()
    assert np.array_equal(first.view(np.uint32), a.run().view(np.uint32))


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_recorded_decode_steps(dev, fmt):
    """A recorded step of a growing batch: norm, rotation, write and attention replayed with new lengths, new q / k / v and the
    program's own eager calls between the replays, each replay against the eager result and the reference."""
    rng = np.random.default_rng(30)
    ctx, H, KV, D, P, B, cap = dev.ctx, 8, 2, 128, 16, 3, 200
    c = R.Paged(fmt, KV, D, P, 3 * 13 + 1, seed=4)
    tables = [c.take(cap) for _ in range(B)]
    lens = [5, 60, 113]
    for ids, n in zip(tables, lens):
        c.put(ids, rng.standard_normal((n, KV, D)).astype(f32), rng.standard_normal((n, KV, D)).astype(f32))
    cache = dev.cache(c)
    freq = (1e4 ** -(np.arange(0, D, 2) / D)).astype(f32)
    wq, wk = rng.standard_normal(D).astype(f32), rng.standard_normal(D).astype(f32)
    batch = dev.batch([1] * B, lens, tables, row_off=False, max_len=cap)
    qb, kb, vb, qr, out = dev.room(B, H, D), dev.room(B, KV, D), dev.room(B, KV, D), dev.room(B, H, D), dev.room(B, H, D)
    rows = ctx.qkv_rows(head_dim=D, heads=H, kv_heads=KV, q=qb, k=kb, v=vb, q_out=qr, q_norm=dev.up(wq), k_norm=dev.up(wk),
                        inv_freq=dev.up(freq), rot_dim=D)
    args = ctx.attn_args(q=qr, out=out, heads=H, scale=D ** -0.5)

    def step():
        ctx.kv_write(cache, batch, rows)
        ctx.attention(cache, batch, args)

    def feed(lens):
        q, k, v = (rng.standard_normal((B, n, D)).astype(f32) for n in (H, KV, KV))
        ctx.h2d(qb, q), ctx.h2d(kb, k), ctx.h2d(vb, v), ctx.h2d(batch.kv_len, np.asarray(lens, np.int32))
        for b, ids in enumerate(tables):
            t = lens[b] - 1
            kq = R.norm_rope(k[b:b + 1], wk, 1e-6, False, [t], freq, False)
            for n, x in (("k", kq), ("v", v[b:b + 1])):
                for dst, src in zip(c.planes[n], R.quantize(fmt, x)):
                    dst[ids[t // P], :, t % P] = src[0]
        return q

    def want(q, lens):
        qq = np.concatenate([R.norm_rope(q[b:b + 1], wq, 1e-6, False, [lens[b] - 1], freq, False) for b in range(B)])
        return np.concatenate([R.attention(qq[b:b + 1], c.get("k", ids, lens[b]), c.get("v", ids, lens[b]), D ** -0.5)
                               for b, ids in enumerate(tables)])

    q = feed(lens)
    step()
    close(dev.down(out, B, H, D), want(q, lens))
    ctx.graph_begin()
    step()
    graph = ctx.graph_end()
    try:
        for i in range(4):
            lens = [n + 1 for n in lens]
            q = feed(lens)
            graph.launch()
            got = dev.down(out, B, H, D)
            close(got, want(q, lens))
            ctx.h2d(out, np.full((B, H, D), np.nan, f32))
            step()                                     # the same step eagerly: writes the same bytes, gives the same bits
            assert np.array_equal(dev.down(out, B, H, D), got)
    finally:
        graph.destroy()


def test_two_graphs_share_the_workspace(dev):
    """Two recorded calls that both split their keys, replayed in turn, and an older graph refused once the workspace moved."""
    a = Case(dev, "q8", 8, 2, 128, 64, [1, 1], [1500, 900], seed=21)
    b = Case(dev, "q4", 8, 2, 128, 64, [1, 1], [1200, 1100], seed=22)
    ea, eb = a.run(), b.run()
    graphs = []
    for x in (a, b):
        dev.ctx.graph_begin()
        dev.ctx.attention(x.cache, x.batch, x.args)
        graphs.append(dev.ctx.graph_end())
    try:
        for _ in range(3):
            for g, x, e in zip(graphs, (a, b), (ea, eb)):
                dev.ctx.h2d(x.out, np.full_like(e, np.nan))
                g.launch()
                assert np.array_equal(dev.down(x.out, *e.shape), e)
    finally:
        for g in graphs:
            g.destroy()


def test_two_contexts_at_once(dev):
    """Two contexts (two streams) over one cache, calls in flight together, each with its own workspace."""
    a = Case(dev, "q8", 32, 8, 128, 64, [1] * 4, [2000, 1500, 900, 3], seed=23)
    eager = a.run()
    other = Context(0)
    try:
        d2 = R.Dev(other)
        outs = [d2.room(*eager.shape) for _ in range(4)]
        dev.ctx.sync()
        for o in outs:
            dev.ctx.attention(a.cache, a.batch, a.args)
            args = other.attn_args(q=a.args.q, out=o, heads=32, scale=a.scale)
            other.attention(a.cache, a.batch, args)
        for o in outs:
            assert np.array_equal(d2.down(o, *eager.shape), eager)
        assert np.array_equal(dev.down(a.out, *eager.shape), eager)
    finally:
        other.close()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_decoder_layer_around_it(dev, fmt):
    """The attention half of a decoder layer as a program runs it: the q / k / v plan, the write, attention, the wo plan with its
    residual; prefill by 37 rows, then three decoded tokens through the plans, against 64 bits on the values the plans gave."""
    ctx, d, H, KV, D, P, n = dev.ctx, 256, 4, 2, 64, 16, 37
    rng = np.random.default_rng(40)
    from helpers import Gpu
    g = Gpu(ctx)

    def weight(seed, N, K):
        t = synth.q4_tensor(seed, N, K)
        return g.planes("q4", t), t
    import oracle as O
    (pq, tq), (pk, tk), (pv, tv), (po, to) = (weight(50 + i, N, K) for i, (N, K) in enumerate([(H * D, d), (KV * D, d), (KV * D, d), (d, H * D)]))
    freq, wn = (1e4 ** -(np.arange(0, D, 2) / D)).astype(f32), rng.standard_normal(d).astype(f32)
    wq, wk = rng.standard_normal(D).astype(f32), rng.standard_normal(D).astype(f32)
    c = R.Paged(fmt, KV, D, P, 8, seed=6)
    ids = c.take(64)
    cache, fb, wqb, wkb = dev.cache(c), dev.up(freq), dev.up(wq), dev.up(wk)

    def attend(qb, kb, vb, m, L, out):
        batch = dev.batch([m], [L], [ids])
        qo = dev.room(m, H, D)
        ctx.kv_write(cache, batch, ctx.qkv_rows(head_dim=D, heads=H, kv_heads=KV, q=qb, k=kb, v=vb, q_out=qo, q_norm=wqb, k_norm=wkb,
                                                inv_freq=fb, rot_dim=D))
        ctx.attention(cache, batch, ctx.attn_args(q=qo, out=out, heads=H, scale=D ** -0.5))
        q, k, v = dev.down(qb, m, H, D), dev.down(kb, m, KV, D), dev.down(vb, m, KV, D)
        pos = np.arange(L - m, L)
        kr = R.norm_rope(k, wk, 1e-6, False, pos, freq, False)
        for name, x in (("k", kr), ("v", v)):
            for dst, src in zip(c.planes[name], R.quantize(fmt, x)):
                for i, p in enumerate(pos):
                    dst[ids[p // P], :, p % P] = src[i]
        want = R.attention(R.norm_rope(q, wq, 1e-6, False, pos, freq, False), c.get("k", ids, L), c.get("v", ids, L), D ** -0.5)
        close(dev.down(out, m, H, D), want)

    x = dev.up(synth.normal(60, n * d).reshape(n, d))
    q, k, v, a, y = dev.room(n, H * D), dev.room(n, KV * D), dev.room(n, KV * D), dev.room(n, H * D), dev.room(n, d)
    ctx.matmul_t_q4(x, *pq, q, n, d, H * D)
    ctx.matmul_t_q4(x, *pk, k, n, d, KV * D)
    ctx.matmul_t_q4(x, *pv, v, n, d, KV * D)
    attend(q, k, v, n, n, a)
    ctx.matmul_t_q4(a, *po, y, n, H * D, d)
    r = O.matmul_t_q4(dev.down(a, n, H * D), to["nib"], to["sc"], to["mn"], n, H * D, d)
    assert np.abs(dev.down(y, n, d) - r).max() <= 1e-3 * np.abs(r).max()
    h = dev.up(synth.normal(61, d))
    norm = dict(norm_w=dev.up(wn), eps=1e-6)
    job = lambda p, src, dst, K, N, **f: dict(x=src, p0=p[0], sc=p[1], mn=p[2], y=dst, K=K, N=N, **f)  # noqa: E731
    qkv = ctx.gemv_plan("q4", [job(pq, h, q, d, H * D, **norm), job(pk, h, k, d, KV * D, **norm), job(pv, h, v, d, KV * D, **norm)])
    wo = ctx.gemv_plan("q4", [job(po, a, h, H * D, d, res=h)])
    try:
        for t in range(3):
            before = dev.down(h, d)
            qkv.run()
            attend(q, k, v, 1, n + 1 + t, a)
            wo.run()
            r = before + O.matmul_t_q4(dev.down(a, n, H * D)[:1], to["nib"], to["sc"], to["mn"], 1, H * D, d).ravel()
            assert np.abs(dev.down(h, d) - r).max() <= 1e-5 * np.abs(r).max()
    finally:
        qkv.destroy(), wo.destroy(), g.free()


def test_refusals(dev):
    a = Case(dev, "q8", 4, 2, 64, 16, [2], [9], seed=31)
    ctx = dev.ctx

    def refused(code, cache=None, batch=None, **change):
        args = ctx.attn_args(**{**dict(q=a.args.q, out=a.out, heads=4, scale=1.0), **change})
        with pytest.raises(BrikError) as e:
            ctx.attention(cache or a.cache, batch or a.batch, args)
        assert e.value.code == code

    for change in (dict(heads=3), dict(heads=0), dict(window=-1), dict(scale=float("inf")), dict(scale=float("nan")), dict(softcap=-1.0),
                   dict(softcap=float("inf")), dict(q=None), dict(out=None), dict(q_stride=128), dict(out_stride=258), dict(out=a.args.q),
                   dict(out=a.args.q + 64)):
        refused(BRIK_EINVAL, **change)
    refused(BRIK_EALIGN, q=a.args.q + 4)
    refused(BRIK_EALIGN, out=a.out.offset(8))
    for D in (32, 160, 224):
        cc = dev.cache(R.Paged("q8", 2, D, 16, 1))
        refused(BRIK_EINVAL, cache=cc)
    wrong = dev.batch([2], [9], [a.tables[0]])
    wrong.row_off, wrong.rows, wrong.seqs = None, 5, 2
    refused(BRIK_EINVAL, batch=wrong)
    wrong = dev.batch([2], [9], [a.tables[0]])
    wrong.prefix_len = 3
    refused(BRIK_EINVAL, batch=wrong)


def test_option_refusals(ctx):
    for option, values in ((BRIK_OPT_ATTN_ROWS, (-1, 1, 32, 64, 512)), (BRIK_OPT_ATTN_SPLITS, (-1, 257))):
        for value in values:
            with pytest.raises(BrikError) as e:
                ctx.set_option(option, value)
            assert e.value.code == BRIK_EINVAL


@pytest.mark.parametrize("fmt,B", [("q8", 700), ("q4", 1030)])
def test_many_sequences_behind_a_prefix(dev, fmt, B):
    """So many rows share the prefix that it goes to tiles of 128 rows and more, the sequences' own keys to tiles of 16, in one
    call: shared out where there are up to 1024 sequences and one is long."""
    rng = np.random.default_rng(B)
    own = [int(x) for x in rng.integers(1, 20, B)]
    own[5], own[B - 1] = 1100, 40
    c = Case(dev, fmt, 32, 8, 64, 16, [1] * B, [45 + n for n in own], prefix=45, seed=B)
    c.check()
    assert dev.ctx.last_kernel() == "attn_few"


@pytest.mark.parametrize("fmt,D,window", [("q8", 64, 1100), ("q4", 256, 0), ("q4", 128, 1030)])
def test_shared_out_keys_behind_a_window(dev, fmt, D, window):
    rng = np.random.default_rng(D)
    lens = [int(x) for x in rng.integers(1, 2500, 40)]
    lens[0], lens[7], lens[39] = 2500, 1, 0
    rows = [1] * 40
    rows[39] = 0
    Case(dev, fmt, 8, 8, D, 16, rows, lens, seed=D, window=window, behind=2).check()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("H,KV,D,rows,lens", [(8, 2, 128, [300], [1500]), (6, 2, 64, [256] * 4, [256] * 4), (4, 1, 96, [130, 1, 64], [900, 700, 64]),
                                              (2, 2, 256, [200], [2000]), (16, 1, 192, [40, 50], [600, 1000])])
def test_prompts_by_the_choice_of_the_call(dev, fmt, H, KV, D, rows, lens):
    """Rows and splits as the sizes choose them, eager and again in other batches on the same workspace."""
    a = Case(dev, fmt, H, KV, D, 32, rows, lens, seed=1)
    a.check()
    b = Case(dev, fmt, H, KV, D, 32, [1] * len(rows), lens, seed=2)
    b.check()
    a = Case(dev, fmt, H, KV, D, 32, rows, lens, seed=1)
    a.check()
