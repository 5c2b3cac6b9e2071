"""Steps over a part of a larger batch: row_off begins above 0 and ends below the rows there are. The rows before and behind
belong to no sequence: nothing is written into the cache for them, and what their outputs hold stays. The rows between are
compared with a 64-bit reference at the tolerances of test_gpu_attention.py and test_gpu_kv_rows.py."""
import numpy as np
import pytest

import kvref as R
from brimkern_amd.capi import BRIK_OPT_ATTN_ROWS, BRIK_OPT_ATTN_SPLITS
from test_gpu_attention import Case, close
from test_gpu_kv_rows import freqs, near

pytestmark = pytest.mark.gpu
f32 = np.float32


@pytest.fixture()
def dev(ctx):
    d = R.Dev(ctx)
    yield d
    d.free()
    ctx.set_option(BRIK_OPT_ATTN_ROWS, 0)
    ctx.set_option(BRIK_OPT_ATTN_SPLITS, 0)


def inside(dev, a, lead):
    """The case's rows moved up by `lead` within its buffers, which are long enough for that."""
    a.batch.row_off = dev.i32(lead + np.concatenate(([0], np.cumsum(a.rows)))).ptr
    dev.ctx.h2d(a.args.q, np.roll(a.q, lead, axis=0))
    dev.ctx.h2d(a.out, np.full(a.q.shape, np.nan, f32))


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("tile,splits", [(0, 0), (16, 1), (16, 3), (16, 20), (128, 1), (128, 3), (256, 1), (256, 5)])
@pytest.mark.parametrize("H,KV,D,rows,lens,prefix,lead", [
    (8, 2, 128, [1, 1, 1], [300, 90, 513], 0, 5),
    (4, 4, 64, [40, 0, 3], [200, 7, 90], 0, 70),
    (12, 3, 64, [1, 2, 5], [90, 140, 75], 70, 4),
])
def test_attention(dev, fmt, tile, splits, H, KV, D, rows, lens, prefix, lead):
    """Keys whole and split, few and many parts to join, with and without a prefix, by every kernel."""
    a = Case(dev, fmt, H, KV, D, 16, rows, lens, prefix=prefix, seed=lead, behind=lead + 3)
    dev.ctx.set_option(BRIK_OPT_ATTN_ROWS, tile)
    dev.ctx.set_option(BRIK_OPT_ATTN_SPLITS, splits)
    a.run()                                             # leaves its partial results in the workspace
    inside(dev, a, lead)
    got = a.run()
    close(got[lead:lead + a.T], a.want())
    assert np.isnan(got[:lead]).all() and np.isnan(got[lead + a.T:]).all()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("lens,prefix,lead", [([2500, 2100], 0, 1000), ([2400, 1, 1800, 700], 40, 3)])
def test_attention_with_shared_out_keys(dev, fmt, lens, prefix, lead):
    a = Case(dev, fmt, 32, 8, 128, 64, [1] * len(lens), [n + prefix for n in lens], prefix=prefix, seed=lead, behind=lead + 2)
    many = 12                                           # enough of them that their keys are shared out
    a.rows, a.lens = a.rows * many, a.lens * many
    a.T = len(a.rows)
    rng = np.random.default_rng(1)
    a.tables, a.shown = a.tables * many, a.shown * many
    a.q = rng.standard_normal((a.T + lead + 2, 32, 128)).astype(f32)
    a.batch = dev.batch(a.rows, a.lens, a.shown, prefix=(a.pre, prefix) if prefix else None, total=a.T + lead + 2)
    a.out = dev.room(*a.q.shape)
    a.args = dev.ctx.attn_args(q=dev.up(a.q), out=a.out, heads=32, scale=a.scale)
    inside(dev, a, lead)
    got = a.run()
    close(got[lead:lead + len(lens)], a.want()[:len(lens)])
    last = slice(a.T - len(lens), a.T)
    close(got[lead:][last], a.want()[last])
    assert np.isfinite(got[lead:lead + a.T]).all() and np.isnan(got[:lead]).all() and np.isnan(got[lead + a.T:]).all()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("rows,lens,lead,behind", [([1], [100], 4, 0), ([3, 0, 20], [40, 3, 33], 5, 2), ([2] * 70, [50] * 70, 66, 1)])
def test_write_and_read(dev, fmt, rows, lens, lead, behind):
    """The whole cache, and every row of q_out, k_out and of what is read back."""
    rng = np.random.default_rng(lead)
    H, KV, D, P, T = 4, 2, 64, 16, sum(rows)
    all_rows = lead + T + behind
    c = R.Paged(fmt, KV, D, P, sum(-(-n // P) for n in lens) + 2, seed=lead)
    tables = [c.take(n) for n in lens]
    q, k, v = (rng.standard_normal((all_rows, h, D)).astype(f32) for h in (H, KV, KV))
    wk, freq = rng.standard_normal(D).astype(f32), freqs(D)
    cache, batch = dev.cache(c), dev.batch(rows, lens, tables, total=all_rows)
    batch.row_off = dev.i32(lead + np.concatenate(([0], np.cumsum(rows)))).ptr
    qo, ko = dev.room(all_rows, H, D), dev.room(all_rows, KV, D)
    dev.ctx.kv_write(cache, batch, dev.ctx.qkv_rows(head_dim=D, heads=H, kv_heads=KV, q=dev.up(q), k=dev.up(k), v=dev.up(v), q_out=qo,
                                                    k_out=ko, k_norm=dev.up(wk), inv_freq=dev.up(freq), rot_dim=D))
    pos = np.concatenate([np.arange(L - n, L) for n, L in zip(rows, lens)])
    mine = slice(lead, lead + T)
    kr = R.norm_rope(k[mine], wk, 1e-6, False, pos, freq, False)
    got_q, got_k = dev.down(qo, all_rows, H, D), dev.down(ko, all_rows, KV, D)
    near(got_q[mine], R.norm_rope(q[mine], None, 0, False, pos, freq, False))
    near(got_k[mine], kr)
    for x in (got_q, got_k):
        assert np.isnan(x[:lead]).all() and np.isnan(x[lead + T:]).all()
    at = 0
    for n, L, ids in zip(rows, lens, tables):
        for name, x in (("k", got_k[mine]), ("v", v[mine])):
            planes = R.quantize(fmt, x[at:at + n])
            for i, p in enumerate(range(L - n, L)):
                for dst, src in zip(c.planes[name], planes):
                    dst[ids[p // P], :, p % P] = src[i]
        at += n
    there = dev.planes(c)
    for name in "kv":
        for plane, want in zip(there[name], c.planes[name]):
            assert np.array_equal(plane, want)
    kb, vb = dev.room(all_rows, KV, D), dev.room(all_rows, KV, D)
    dev.ctx.kv_read(cache, batch, kb, vb)
    for name, buf in (("k", kb), ("v", vb)):
        got = dev.down(buf, all_rows, KV, D)
        want = np.concatenate([c.get(name, ids, L)[L - n:] for n, L, ids in zip(rows, lens, tables)])
        assert np.array_equal(got[mine], want.astype(f32)) and np.isnan(got[:lead]).all() and np.isnan(got[lead + T:]).all()


@pytest.mark.parametrize("given", [False, True])
def test_norm_rope(dev, given):
    """Positions of the batch, and given ones."""
    rng = np.random.default_rng(9)
    rows, lens, lead, behind, H, D = [2, 0, 3], [9, 4, 5], 3, 2, 3, 96
    T = sum(rows)
    q = rng.standard_normal((lead + T + behind, H, D)).astype(f32)
    w, qo = rng.standard_normal(D).astype(f32), dev.room(lead + T + behind, H, D)
    batch = dev.batch(rows, lens, [[], [], []], total=lead + T + behind)
    batch.row_off = dev.i32(lead + np.concatenate(([0], np.cumsum(rows)))).ptr
    pos = rng.integers(0, 1 << 20, lead + T + behind) if given else np.concatenate((np.zeros(lead, int), [7, 8, 2, 3, 4], np.zeros(behind, int)))
    dev.ctx.qk_norm_rope(batch, dev.ctx.qkv_rows(head_dim=D, heads=H, q=dev.up(q), q_out=qo, q_norm=dev.up(w), inv_freq=dev.up(freqs(D)),
                                                 rot_dim=D, positions=dev.i32(pos) if given else None))
    got = dev.down(qo, lead + T + behind, H, D)
    mine = slice(lead, lead + T)
    near(got[mine], R.norm_rope(q[mine], w, 1e-6, False, pos[mine], freqs(D), False))
    assert np.isnan(got[:lead]).all() and np.isnan(got[lead + T:]).all()
