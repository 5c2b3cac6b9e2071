"""q and out side by side in the rows of one buffer, as a step's workspace may have them: they do not overlap, and nothing between
them changes."""
import numpy as np
import pytest

import kvref as R
from brimkern_amd.capi import BrikError, BRIK_EINVAL
from test_gpu_attention import Case, close

pytestmark = pytest.mark.gpu


@pytest.fixture()
def dev(ctx):
    d = R.Dev(ctx)
    yield d
    d.free()


@pytest.mark.parametrize("rows,lens", [([1, 1], [900, 40]), ([50], [90])])
def test_q_and_out_in_one_buffer(dev, rows, lens):
    a = Case(dev, "q8", 4, 2, 64, 16, rows, lens, seed=3)
    rng, width = np.random.default_rng(1), 4 * 64 + 24 + 4 * 64 + 8
    wide = rng.standard_normal((a.T, width)).astype(np.float32)
    wide[:, :256] = a.q.reshape(a.T, -1)
    buf = dev.up(wide)
    dev.ctx.attention(a.cache, a.batch, dev.ctx.attn_args(q=buf, out=buf.offset(4 * 280), heads=4, scale=a.scale, q_stride=width, out_stride=width))
    got = dev.down(buf, a.T, width)
    close(got[:, 280:536].reshape(a.T, 4, 64), a.want())
    assert np.array_equal(got[:, :280], wide[:, :280]) and np.array_equal(got[:, 536:], wide[:, 536:])
    with pytest.raises(BrikError) as e:
        dev.ctx.attention(a.cache, a.batch, dev.ctx.attn_args(q=buf, out=buf.offset(4 * 252), heads=4, scale=a.scale, q_stride=width, out_stride=width))
    assert e.value.code == BRIK_EINVAL
