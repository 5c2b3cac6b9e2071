"""Scores up to the stated 2^22, of which one leads: the largest takes all, and the output is its token's values, with no overflow
of what lies between.

The queries are chosen so that the largest score leads by more than 2^-9 of its size, 2^13 times the error of a score (2^-22 of the
largest product's operands); from 2^15 on the other weights are then exp(-2^6) or less. What is left is the output's own rounding:
the value in halves (2^-22) times weights that cancel (a quotient of equal sums, 2^-23): 2^-20 in all."""
import numpy as np
import pytest

import kvref as R
from brimkern_amd.capi import BRIK_OPT_ATTN_ROWS, BRIK_OPT_ATTN_SPLITS
from test_gpu_attention import Case

pytestmark = pytest.mark.gpu
f32 = np.float32


@pytest.fixture()
def dev(ctx):
    d = R.Dev(ctx)
    yield d
    d.free()
    ctx.set_option(BRIK_OPT_ATTN_ROWS, 0)
    ctx.set_option(BRIK_OPT_ATTN_SPLITS, 0)


def leads(q, k):
    """Whether the largest score of every row and head leads by 2^-9 of the largest size."""
    x = np.einsum("thd,jhd->thj", q.astype(np.float64), np.repeat(k, q.shape[1] // k.shape[1], 1))
    t = np.sort(np.where(np.arange(len(k)) <= len(k) - len(q) + np.arange(len(q))[:, None, None], x, -np.inf), -1)
    return ((t[..., -1] - t[..., -2]) > 2.0**-9 * np.abs(x).max(-1)).all()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("tile,splits", [(16, 1), (16, 3), (128, 1), (128, 2), (256, 1), (256, 3)])
@pytest.mark.parametrize("size", [2.0**15, 2.0**17, 2.0**19])
@pytest.mark.parametrize("vscale", [1.0, 300.0])
def test_largest_takes_all(dev, fmt, tile, splits, size, vscale):
    n, L, D = 20, 150, 64
    a = Case(dev, fmt, 4, 2, D, 32, [n], [L], seed=3, vscale=vscale)
    rng, k = np.random.default_rng(11), a.c.get("k", a.tables[0], L)
    for t in range(n):                                   # queries that lead, row by row
        for _ in range(200):
            a.q[t] = rng.standard_normal((4, D))
            if leads(a.q[t:t + 1], k[:L - n + t + 1]):
                break
        else:
            raise AssertionError("no such query")
    a.q = (a.q * size).astype(f32)
    assert np.abs(np.einsum("thd,jhd->thj", a.q.astype(np.float64), np.repeat(k, 2, 1))).max() * a.scale < 2.0**22
    dev.ctx.h2d(a.args.q, a.q)
    dev.ctx.set_option(BRIK_OPT_ATTN_ROWS, tile)
    dev.ctx.set_option(BRIK_OPT_ATTN_SPLITS, splits)
    got, want = a.run(), a.want()
    assert np.isfinite(got).all()
    off = np.abs(got - want).max(-1) / np.abs(want).max(-1)
    assert off.max() <= 2.0**-20, off.max()
