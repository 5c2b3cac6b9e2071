"""A token that a row sees and whose value scale is not finite: its group of the output is not finite, however the keys are split
and however far the token lies below the row's largest score."""
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


def spoil(dev, a, b, token, peak, group, bits):
    """The token's value scale of the group replaced; a token `peak` whose keys follow q, with a score of many thousands."""
    host, P = a.c.planes, a.c.P
    page, slot = a.tables[b][peak // P], peak % P
    host["k"][0][page, :, slot] = 127 * np.sign(a.q[sum(a.rows[:b]), ::a.H // a.KV]).astype(np.int8)
    host["k"][1][page, :, slot] = np.float16(200.0).view(np.uint16)
    host["v"][1][a.tables[b][token // P], :, token % P, group] = bits
    a.cache = dev.cache(a.c)


@pytest.mark.parametrize("bits", [0x7C00, 0xFE00])
@pytest.mark.parametrize("tile,splits", [(16, 1), (16, 3), (16, 12), (16, 40), (128, 1), (128, 4), (128, 30)])
def test_by_splits(dev, tile, splits, bits):
    """The far token in the first split, and in the last."""
    n = 3 if tile == 16 else 40
    for token, peak in ((5, 5000 - n), (5000 - n - 3, 8)):
        a = Case(dev, "q8", 2, 2, 64, 64, [n], [5000], seed=1)
        spoil(dev, a, 0, token, peak, 1, bits)
        dev.ctx.set_option(BRIK_OPT_ATTN_ROWS, tile)
        dev.ctx.set_option(BRIK_OPT_ATTN_SPLITS, splits)
        got = a.run()
        assert not np.isfinite(got[0, :, 32:]).any() and np.isfinite(got[0, :, :32]).all()


@pytest.mark.parametrize("bits", [0x7C00, 0xFE00])
def test_shared_out(dev, bits):
    lens = [3000] + [1500] * 13
    a = Case(dev, "q8", 16, 16, 64, 64, [1] * 14, lens, seed=2)
    clean = a.check()
    for token, peak in ((5, 2990), (2990, 5)):
        a = Case(dev, "q8", 16, 16, 64, 64, [1] * 14, lens, seed=2)
        spoil(dev, a, 0, token, peak, 1, bits)
        got = a.run()
        assert not np.isfinite(got[0, :, 32:]).any() and np.isfinite(got[0, :, :32]).all()
        assert np.array_equal(got[1:], clean[1:])
