"""Routing weights within the bound that include/brik.h gives: (2.3 d + 44) 2^-24 of the weight and 2^-125 of scale, d how far the logit
lies below the largest that counts."""
import numpy as np
import pytest

import moeref as R
from test_gpu_moe import HOW, dev, run_route        # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", range(4))
@pytest.mark.parametrize("T,E,k,spread", [(300, 16, 4, 1), (200, 64, 8, 12), (200, 256, 16, 30), (100, 256, 40, 60), (60, 1024, 64, 20), (60, 1000, 64, 100)])
def test_weights(dev, T, E, k, spread, how):
    rng = np.random.default_rng(E + spread)
    logits = (spread * rng.standard_normal((T, E)) + rng.uniform(-50, 50, (T, 1))).astype(np.float32)
    h = HOW[how]
    ids, w = run_route(dev, logits, k, sort=False, **h)
    want_ids, want = R.route(logits, k, **h)
    assert (ids == want_ids).all()
    l = np.take_along_axis(logits.astype(np.float64), ids, -1)
    d = l.max(-1, keepdims=True) - l                              # (the largest of a token is chosen)
    if h.get("sigmoid") and not h.get("renorm"):
        d = np.maximum(-l, 0)
    scale = h.get("scale", 1.0)
    assert (np.abs(w - want) <= (2.3 * d + 44) * R.HALF * np.abs(want) + 2.0 ** -125 * scale).all()
