"""The added values of an 8-bit product are a rounding of their own, whatever kernel and splits are picked: y is, bit for bit, the f32
sum times w_scales, times x_scales, plus res, each rounded."""
import numpy as np
import pytest

from brimkern_amd.capi import BRIK_OPT_I8_KERNEL, BRIK_OPT_I8_SPLITS
from test_gpu_i8 import KERNELS, operands, run_product
from test_gpu_moe import dev        # noqa: F401

pytestmark = pytest.mark.gpu


def by_steps(x, xs, w, ws, res):
    sums = np.rint(x.astype(np.float64) @ w.astype(np.float64).T)            # exact: below 2^53
    return (sums.astype(np.float32) * ws[None]) * xs[:, None] + res


@pytest.mark.parametrize("kernel", range(KERNELS + 1))
@pytest.mark.parametrize("splits", [0, 3])
def test_added_values(dev, kernel, splits):
    """res of the product's size, so that the sum cancels in part: a product that is not rounded first shows in most values."""
    ctx = dev.ctx
    try:
        for M, K, N in ((1, 32, 1), (70, 1120, 45), (300, 96, 290), (33, 4128, 17), (130, 2592, 300), (1, 4096, 513)):
            rng = np.random.default_rng(K + N)
            ops = operands(rng, M, K, N)
            res = (rng.standard_normal((M, N)) * 5000 * np.sqrt(K) * 2.0 ** -10).astype(np.float32)
            ctx.set_option(BRIK_OPT_I8_KERNEL, kernel)
            ctx.set_option(BRIK_OPT_I8_SPLITS, splits)
            for in_place in (False, True):
                assert (run_product(dev, *ops, res=res, in_place=in_place) == by_steps(*ops, res)).all()
    finally:
        ctx.set_option(BRIK_OPT_I8_KERNEL, 0)
        ctx.set_option(BRIK_OPT_I8_SPLITS, 0)
