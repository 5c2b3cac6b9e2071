"""Head norms and rotation (brik_qk_norm_rope), the cache's writes (brik_kv_write) and reads (brik_kv_read) against 64-bit
references. Norm and rotation are computed in 64 bits and rounded once, so results may differ from the reference's by one
rounding of a value that lies within 2^-40 of a tie: at most one unit in the last place of f32, and equal in all but
one in ten thousand values. Written bytes must equal the encoders' on the same f32 values."""
import numpy as np
import pytest

import kvref as R
from brimkern_amd.capi import BrikError, BRIK_EALIGN, BRIK_EINVAL

pytestmark = pytest.mark.gpu
f32 = np.float32


@pytest.fixture()
def dev(ctx):
    d = R.Dev(ctx)
    yield d
    d.free()


def rows_of(rng, T, heads, D):
    return (rng.standard_normal((T, heads, D)) * np.exp(0.5 * rng.standard_normal(D))).astype(f32)


def freqs(rot):
    return (1e4 ** -(np.arange(0, rot, 2) / rot)).astype(f32)


def near(got, want):
    """One unit in the last place at most, and that rarely."""
    off = np.abs(got.astype(np.float64) - want.astype(np.float64)) / np.spacing(np.maximum(np.abs(want), f32(1e-30))).astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.where(np.isnan(off), 0, off)
    assert off.max() <= 1.0 and (off > 0).mean() <= 1e-4, (off.max(), (off > 0).mean())


@pytest.mark.parametrize("T,H,KV,D,rot,norm,one_plus,inter", [
    (1, 32, 8, 128, 128, True, False, False),
    (1, 14, 2, 64, 64, False, False, False),
    (5, 3, 1, 96, 48, True, True, False),
    (7, 4, 4, 256, 256, True, False, True),
    (3, 2, 1, 32, 8, True, False, True),
    (130, 5, 5, 160, 152, True, True, True),
    (65, 9, 3, 192, 192, True, False, False),
    (2, 1, 1, 224, 0, True, False, False),
    (4, 6, 2, 128, 64, False, False, False),
])
def test_norm_rope(dev, T, H, KV, D, rot, norm, one_plus, inter):
    rng = np.random.default_rng(T * D + H)
    q, k = rows_of(rng, T, H, D), rows_of(rng, T, KV, D)
    wq, wk = (rng.standard_normal(D).astype(f32) for _ in range(2))
    pos = rng.integers(0, 1 << 20, T).astype(np.int32)
    freq = freqs(rot) if rot else None
    qo, ko = dev.room(T, H, D), dev.room(T, KV, D)
    rows = dev.ctx.qkv_rows(head_dim=D, heads=H, kv_heads=KV, q=dev.up(q), k=dev.up(k), q_out=qo, k_out=ko,
                            q_norm=dev.up(wq) if norm else None, k_norm=dev.up(wk) if norm else None, eps=1e-5, one_plus=one_plus,
                            inv_freq=dev.up(freq) if rot else None, rot_dim=rot, positions=dev.i32(pos), interleaved=inter)
    dev.ctx.qk_norm_rope(dev.ctx.kv_batch(seqs=1, rows=T), rows)
    for got, x, w, h in ((qo, q, wq, H), (ko, k, wk, KV)):
        near(dev.down(got, T, h, D), R.norm_rope(x, w if norm else None, 1e-5, one_plus, pos, freq, inter))


def test_norm_rope_values_at_the_edges(dev):
    """Zero rows, tiny and huge rows (their squares leave f32), a NaN and an infinity that stay in their head, negative and far
    positions."""
    rng = np.random.default_rng(3)
    T, H, D = 8, 3, 64
    q = rows_of(rng, T, H, D)
    q[0, 0] = 0
    q[1] *= f32(1e-30)
    q[2] *= f32(1e30)
    q[3, 1, 5] = np.nan
    q[4, 2, 63] = np.inf
    pos = np.array([0, 1, -1, 7, 9, -(1 << 30), (1 << 31) - 1, 1 << 30], np.int32)
    w = rng.standard_normal(D).astype(f32)
    qo = dev.room(T, H, D)
    rows = dev.ctx.qkv_rows(head_dim=D, heads=H, q=dev.up(q), q_out=qo, q_norm=dev.up(w), eps=0.0 + 1e-6, inv_freq=dev.up(freqs(D)),
                            rot_dim=D, positions=dev.i32(pos))
    dev.ctx.qk_norm_rope(dev.ctx.kv_batch(seqs=1, rows=T), rows)
    with np.errstate(all="ignore"):
        want = R.norm_rope(q, w, 1e-6, False, pos, freqs(D), False)
    got = dev.down(qo, T, H, D)
    assert np.isnan(got[4, 2]).any() and np.isfinite(got[4, :2]).all() and np.isfinite(got[3, 0]).all()
    ok = np.ones((T, H), bool)
    ok[4, 2] = False
    near(got[ok], want[ok])


def test_norm_rope_in_place_with_strides_and_batch_positions(dev):
    """One packed q | k | v row as a fused projection leaves it, normed in place; positions from ragged lengths; a row behind
    the last sequence stays as it is."""
    rng = np.random.default_rng(4)
    H, KV, D, rows, lens = 4, 2, 96, [3, 0, 5], [9, 4, 5]
    T, width = 9, (4 + 2 * 2) * 96 + 8
    x = rng.standard_normal((T, width)).astype(f32)
    w = rng.standard_normal(D).astype(f32)
    buf = dev.up(x)
    a = dev.ctx.qkv_rows(head_dim=D, heads=H, kv_heads=KV, q=buf, k=buf.offset(4 * H * D), q_out=buf, k_out=buf.offset(4 * H * D),
                         q_stride=width, k_stride=width, q_out_stride=width, k_out_stride=width, q_norm=dev.up(w),
                         inv_freq=dev.up(freqs(D)), rot_dim=D)
    dev.ctx.qk_norm_rope(dev.batch(rows, lens, [[], [], []], total=T), a)
    got = dev.down(buf, T, width)
    pos = [6, 7, 8, 0, 1, 2, 3, 4]
    want = x.copy()
    want[:8, :H * D] = R.norm_rope(x[:8, :H * D].reshape(8, H, D), w, 1e-6, False, pos, freqs(D), False).reshape(8, -1)
    want[:8, H * D:(H + KV) * D] = R.norm_rope(x[:8, H * D:(H + KV) * D].reshape(8, KV, D), None, 0, False, pos, freqs(D), False).reshape(8, -1)
    near(got, want)
    assert np.array_equal(got[8], x[8]) and np.array_equal(got[:, (H + KV) * D:], x[:, (H + KV) * D:])


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("D,KV,P,rows,lens", [
    (128, 8, 64, [1] * 5, [1, 64, 65, 130, 7]),
    (64, 2, 16, [37, 1, 0, 20], [40, 33, 3, 20]),
    (96, 1, 32, [70], [101]),
    (256, 3, 256, [2, 2], [2, 259]),
    (32, 5, 16, [9], [9]),
    (192, 4, 128, [1], [1]),
    (160, 2, 64, [3], [66]),
])
def test_write_and_read_back(dev, fmt, D, KV, P, rows, lens):
    """Bytes equal the encoders'; every other byte of the cache stays; the read gives the planes' values."""
    rng = np.random.default_rng(D + KV + P)
    c = R.Paged(fmt, KV, D, P, sum(-(-n // P) for n in lens) + 2, seed=D)
    tables = [c.take(n) for n in lens]
    T = sum(rows)
    k, v = rows_of(rng, T, KV, D), rows_of(rng, T, KV, D)
    cache, batch = dev.cache(c), dev.batch(rows, lens, tables)
    dev.ctx.kv_write(cache, batch, dev.ctx.qkv_rows(head_dim=D, kv_heads=KV, k=dev.up(k), v=dev.up(v)))
    got = dev.planes(c)
    at = 0
    for n, L, ids in zip(rows, lens, tables):
        for name, x in (("k", k), ("v", v)):
            q = R.quantize(fmt, x[at:at + n])
            for i, p in enumerate(range(L - n, L)):
                for dst, src in zip(c.planes[name], q):
                    dst[ids[p // P], :, p % P] = src[i]
        at += n
    for name in "kv":
        for a, b in zip(got[name], c.planes[name]):
            assert np.array_equal(a, b), name
    ko, vo = dev.room(T, KV, D), dev.room(T, KV, D)
    dev.ctx.kv_read(cache, batch, ko, None)
    dev.ctx.kv_read(cache, batch, None, vo)
    at = 0
    for n, L, ids in zip(rows, lens, tables):
        for name, o in (("k", ko), ("v", vo)):
            want = c.get(name, ids, L)[L - n:].astype(f32)
            assert np.array_equal(dev.down(o, T, KV, D)[at:at + n], want), name
        at += n


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_written_bytes_on_hard_values(dev, fmt):
    """NaN, infinities, zeros of both signs, ties, subnormal and huge values: the bytes of brik_quantize_* on the same rows."""
    rng = np.random.default_rng(9)
    D, KV, P, T = 64, 2, 16, 24
    x = (rng.standard_normal((T, KV, D)) * rng.choice([1e-6, 1e-3, 1, 40], (T, 1, 1))).astype(f32)
    f = x.reshape(-1)
    f[5] = np.nan
    f[32:64] = np.nan
    f[64:96] = 0
    f[64], f[80] = -0.0, -0.0
    f[96:128] = np.abs(f[96:128])
    f[100], f[101], f[110] = 0.0, -0.0, -0.0
    f[130], f[140] = np.inf, -np.inf
    f[160:192] = np.round(f[160:192] * 4) / 4
    f[192:224] = (np.arange(32) - 15.5) * 0.0625
    f[224:256] = 1e-30
    f[256:288] = 3e38
    f[288:320] = -np.inf
    f[320:352] = np.abs(f[320:352])
    f[330], f[340] = -0.0, 0.0
    f[352:384] = np.arange(32) * 0.5 - 8
    f[384:416] = np.arange(32) - 127.5 + 96
    c = R.Paged(fmt, KV, D, P, 3, seed=1)
    ids = c.take(T)
    cache, batch, src = dev.cache(c), dev.batch([T], [T], [ids]), dev.up(x)
    dev.ctx.kv_write(cache, batch, dev.ctx.qkv_rows(head_dim=D, kv_heads=KV, k=src, v=src))
    n = x.size
    planes = [dev.up(np.zeros(n if fmt == "q8" else n // 2, np.uint8))] + [dev.up(np.zeros(n // 32, np.uint16)) for _ in range(1 if fmt == "q8" else 2)]
    dev.ctx.quantize(fmt, src, planes, n)
    want = [dev.ctx.download(b, np.uint8 if i == 0 else np.uint16, n // 32 if i else n if fmt == "q8" else n // 2).reshape(T, KV, -1)
            for i, b in enumerate(planes)]
    got = dev.planes(c)
    t = np.arange(T)
    for name in "kv":
        for g, w in zip(got[name], want):
            g = g[np.asarray(ids)[t // P], :, t % P]
            assert np.array_equal(g.view(w.dtype), w), (name, np.argwhere(g.view(w.dtype) != w)[:5])


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_fused_write_gives_the_bytes_of_the_separate_calls(dev, fmt):
    rng = np.random.default_rng(12)
    H, KV, D, P, rows, lens = 8, 2, 128, 32, [1, 3, 40], [77, 3, 100]
    T = sum(rows)
    q, k, v = rows_of(rng, T, H, D), rows_of(rng, T, KV, D), rows_of(rng, T, KV, D)
    wq, wk, freq = dev.up(rng.standard_normal(D).astype(f32)), dev.up(rng.standard_normal(D).astype(f32)), dev.up(freqs(D))
    c = R.Paged(fmt, KV, D, P, 12, seed=2)
    tables = [c.take(n) for n in lens]
    batch = dev.batch(rows, lens, tables)
    how = dict(head_dim=D, heads=H, kv_heads=KV, q_norm=wq, k_norm=wk, inv_freq=freq, rot_dim=D)
    qb, kb, vb = dev.up(q), dev.up(k), dev.up(v)
    q1, k1, q2, k2 = dev.room(T, H, D), dev.room(T, KV, D), dev.room(T, H, D), dev.room(T, KV, D)
    one = dev.cache(c)
    dev.ctx.kv_write(one, batch, dev.ctx.qkv_rows(q=qb, k=kb, v=vb, q_out=q1, k_out=k1, **how))
    fused = dev.planes(c)
    two = dev.cache(c)
    dev.ctx.qk_norm_rope(batch, dev.ctx.qkv_rows(q=qb, k=kb, q_out=q2, k_out=k2, **how))
    dev.ctx.kv_write(two, batch, dev.ctx.qkv_rows(head_dim=D, kv_heads=KV, k=k2, v=vb))
    apart = dev.planes(c)
    assert np.array_equal(dev.down(q1, T, H, D), dev.down(q2, T, H, D)) and np.array_equal(dev.down(k1, T, KV, D), dev.down(k2, T, KV, D))
    for n in "kv":
        for a, b in zip(fused[n], apart[n]):
            assert np.array_equal(a, b), n


def test_prefix_and_tokens_that_do_not_exist(dev):
    """Writes skip prefix tokens, pages out of range, tokens past the table and past max_len; reads give the prefix's
    values and zeros for what does not exist."""
    rng = np.random.default_rng(20)
    KV, D, P, fmt = 2, 64, 16, "q8"
    c = R.Paged(fmt, KV, D, P, 10, seed=3)
    pre = c.take(20)
    c.put(pre, rows_of(rng, 20, KV, D), rows_of(rng, 20, KV, D))
    a, b = c.take(40), c.take(40)
    bad = list(b)
    bad[1] = 10                                             # one past the last page
    rows, lens = [22, 40], [20 + 2, 20 + 40]
    T = sum(rows)
    k, v = rows_of(rng, T, KV, D), rows_of(rng, T, KV, D)
    cache = dev.cache(c)
    batch = dev.batch(rows, lens, [a, bad], cols=3, prefix=(pre, 20), max_len=58)
    dev.ctx.kv_write(cache, batch, dev.ctx.qkv_rows(head_dim=D, kv_heads=KV, k=dev.up(k), v=dev.up(v)))
    for name, x in (("k", k), ("v", v)):
        q = R.quantize(fmt, x)
        for ids, first, n, L in ((a, 0, 22, 22), (bad, 22, 40, 60)):
            for i in range(n):
                p = L - n + i - 20
                if p < 0 or ids[p // P] == 10 or p + 20 >= 58:
                    continue
                for dst, src in zip(c.planes[name], q):
                    dst[ids[p // P], :, p % P] = src[first + i]
    got = dev.planes(c)
    for n in "kv":
        for x, y in zip(got[n], c.planes[n]):
            assert np.array_equal(x, y), n
    ko, vo = dev.room(T, KV, D), dev.room(T, KV, D)
    dev.ctx.kv_read(cache, batch, ko, vo)
    pk, r = c.get("k", pre, 20).astype(f32), dev.down(ko, T, KV, D)
    assert np.array_equal(r[:20], pk) and np.array_equal(r[20:22], c.get("k", a, 2).astype(f32))
    want = np.zeros((40, KV, D), f32)
    for i in range(40):
        if bad[i // P] != 10 and i + 20 < 58:
            want[i] = values_at(c, "k", bad[i // P], i % P)
    assert np.array_equal(r[22:], want)


def values_at(c, n, page, slot):
    return R.values(c.fmt, [p[page, :, slot] for p in c.planes[n]]).astype(f32)


def test_sizes_of_nothing(dev):
    """No rows, no q and k: nothing is touched; rows of sequences without any."""
    c = R.Paged("q8", 1, 32, 16, 1)
    cache, x = dev.cache(c), dev.up(np.ones((1, 1, 32), f32))
    empty = dev.ctx.kv_batch(seqs=0, rows=0)
    dev.ctx.kv_write(cache, empty, dev.ctx.qkv_rows(head_dim=32, kv_heads=1, k=x, v=x))
    dev.ctx.kv_read(cache, empty, x, x)
    dev.ctx.qk_norm_rope(empty, dev.ctx.qkv_rows(head_dim=32, heads=1, q=x, q_out=x))
    dev.ctx.qk_norm_rope(dev.ctx.kv_batch(seqs=1, rows=1), dev.ctx.qkv_rows(head_dim=32))
    assert np.array_equal(dev.planes(c)["k"][0], c.planes["k"][0])


def test_refusals(dev):
    c = R.Paged("q4", 2, 64, 16, 2)
    x, out = dev.up(np.zeros((3, 2, 64), f32)), dev.room(3, 2, 64)
    ctx = dev.ctx

    def refused(code, call, *a):
        with pytest.raises(BrikError) as e:
            call(*a)
        assert e.value.code == code

    cache, batch = dev.cache(c), dev.batch([3], [3], [c.take(3)])
    rows = dict(head_dim=64, kv_heads=2, k=x, v=x)
    ctx.kv_write(cache, batch, ctx.qkv_rows(**rows))
    for change in (dict(head_dim=96), dict(head_dim=40), dict(kv_heads=1), dict(k=None), dict(v=None), dict(k_stride=64), dict(k_stride=130),
                   dict(eps=-1.0), dict(eps=float("nan")), dict(inv_freq=x, rot_dim=12), dict(inv_freq=x, rot_dim=72), dict(q=x),
                   dict(k_out=x, k_stride=132)):
        refused(BRIK_EINVAL, ctx.kv_write, cache, batch, ctx.qkv_rows(**{**rows, **change}))
    refused(BRIK_EALIGN, ctx.kv_write, cache, batch, ctx.qkv_rows(**{**rows, "k": x.offset(4)}))
    for field, value in (("fmt", 3), ("page", 24), ("page", 8), ("pages", 0), ("heads", 0), ("head_dim", 16), ("reserved", 1), ("v_mins", None)):
        wrong = dev.cache(c)
        setattr(wrong, field, value)
        refused(BRIK_EINVAL, ctx.kv_read, wrong, batch, out, out)
    for field, value in (("seqs", 0), ("rows", -1), ("kv_len", None), ("table", None), ("max_len", -1)):
        wrong = dev.batch([3], [3], [[0]])
        setattr(wrong, field, value)
        refused(BRIK_EINVAL, ctx.kv_read, cache, wrong, out, out)
    refused(BRIK_EALIGN, ctx.kv_read, cache, batch, out.offset(4), None)
    refused(BRIK_EINVAL, ctx.qk_norm_rope, batch, ctx.qkv_rows(head_dim=64, heads=2, q=x))


def test_rows_behind_the_last_sequence_with_positions_of_their_own(dev):
    """A padded batch: with given positions, or without rotation, the lengths are not looked at, and still those rows stay."""
    rng = np.random.default_rng(8)
    H, D, T = 2, 64, 9
    q, w, pos = rows_of(rng, T, H, D), rng.standard_normal(D).astype(f32), np.arange(T, dtype=np.int32) * 3
    for rot in (D, 0):
        out = dev.room(T, H, D)
        rows = dev.ctx.qkv_rows(head_dim=D, heads=H, q=dev.up(q), q_out=out, q_norm=dev.up(w), inv_freq=dev.up(freqs(D)) if rot else None,
                                rot_dim=rot, positions=dev.i32(pos) if rot else None)
        dev.ctx.qk_norm_rope(dev.ctx.kv_batch(seqs=2, rows=T, row_off=dev.i32(np.array([0, 4, 6]))), rows)
        got = dev.down(out, T, H, D)
        near(got[:6], R.norm_rope(q[:6], w, 1e-6, False, pos[:6], freqs(D) if rot else None, False))
        assert np.isnan(got[6:]).all()
