"""Sequences with more rows than max_rows: only what lies past max_rows is not said, the rows before hold what they hold in any
other call (a recorded step reads row_off when it is replayed, so a sequence may have grown since)."""
import numpy as np
import pytest

import kvref as R
from brimkern_amd.capi import BRIK_OPT_ATTN_ROWS, BRIK_OPT_ATTN_SPLITS
from test_gpu_attention import Case, close

pytestmark = pytest.mark.gpu


@pytest.fixture()
def dev(ctx):
    d = R.Dev(ctx)
    yield d
    d.free()
    ctx.set_option(BRIK_OPT_ATTN_ROWS, 0)
    ctx.set_option(BRIK_OPT_ATTN_SPLITS, 0)


def check(dev, a, most):
    a.batch.max_rows = most
    dev.ctx.h2d(a.out, np.full(a.q.shape, np.nan, np.float32))
    got, want, at = a.run(), a.want(), 0
    for n in a.rows:
        close(got[at:at + min(n, most)], want[at:at + min(n, most)])
        at += n


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("tile,splits", [(0, 0), (16, 1), (16, 3), (16, 20), (128, 1), (128, 3), (256, 1), (256, 5)])
@pytest.mark.parametrize("H,KV,D,rows,lens,most", [
    (2, 2, 64, [20, 3, 50], [20, 30, 300], 16),
    (8, 2, 128, [20, 1, 0, 33], [70, 300, 5, 161], 4),
    (4, 1, 64, [300, 2, 150], [320, 2, 200], 70),
    (2, 2, 128, [600, 130], [600, 700], 256),
])
def test_first_rows(dev, fmt, tile, splits, H, KV, D, rows, lens, most):
    a = Case(dev, fmt, H, KV, D, 16, rows, lens, seed=most)
    dev.ctx.set_option(BRIK_OPT_ATTN_ROWS, tile)
    dev.ctx.set_option(BRIK_OPT_ATTN_SPLITS, splits)
    check(dev, a, most)


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_first_rows_behind_a_prefix(dev, fmt):
    a = Case(dev, fmt, 4, 2, 64, 16, [30, 2, 90], [200, 140, 180], prefix=80, seed=3)
    check(dev, a, 20)


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_first_rows_of_shared_out_keys(dev, fmt):
    lens = [2000 - 100 * b for b in range(14)]
    a = Case(dev, fmt, 16, 16, 64, 32, [3 + 2 * b for b in range(14)], lens, seed=5)
    check(dev, a, 8)
