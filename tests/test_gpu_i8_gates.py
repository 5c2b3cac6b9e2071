"""Gated rows quantized to 8 bits at gates and values where the f32 path could go wrong: subnormal gates, values next to a border
between two codes, rows that are read again from memory; codes and scales are those of 64 bits."""
import numpy as np
import pytest

import moeref as R
from test_gpu_moe import dev        # noqa: F401

pytestmark = pytest.mark.gpu
LENGTHS = [768, 4096, 9728, 16416]       # a row by a wave, by 256 and 1024 threads, and read again


def same(dev, gate, x):
    M, K = x.shape
    codes, scales = dev.full((M, K), 99, np.int8), dev.full(M, 99.0)
    dev.ctx.quantize_i8(dev.up(x), codes, scales, M, K, gate=dev.up(gate))
    want = R.quantize(R.act(gate) * x.astype(np.float64))
    assert (want[1] > 0).all()                                    # rows that are quantized, not cleared
    assert (dev.get(scales, M) == want[1]).all() and (dev.get(codes, (M, K), np.int8) == want[0]).all()


@pytest.mark.parametrize("K", LENGTHS)
@pytest.mark.parametrize("low,high,size", [(-149, -149, 1e12), (-149, -143, 1e12), (-149, -140, 1e38), (-149, -126, 1e37), (-135, -126, 1e9),
                                           (-127, -124, 1e9), (-126, -120, 1e9), (-126, -120, 1e37)])
def test_tiny_gates(dev, low, high, size, K):
    """Gates of +-2^low to 2^high: half of a subnormal one is no f32 value any more, though its product with x is an ordinary one."""
    rng = np.random.default_rng(K - low)
    gate = (rng.choice([-1, 1], (5, K)) * np.exp2(rng.uniform(low, high, (5, K)))).astype(np.float32)
    same(dev, gate, (rng.uniform(-1, 1, (5, K)) * size).astype(np.float32))


def test_one_tiny_gate_among_others(dev):
    """The largest value of a row, or one of its smaller ones, from a subnormal gate; gates of 0 beside."""
    rng = np.random.default_rng(1)
    gate, x = rng.standard_normal((4, 768)).astype(np.float32), (rng.standard_normal((4, 768)) * 1e-8).astype(np.float32)
    gate[:, ::3] = 0
    gate[:, 100], x[:, 100] = 11 * 2.0 ** -149, [3e38, 3e37, -3e38, 2e36]
    same(dev, gate, x)


@pytest.mark.parametrize("K", [16416, 19968])
def test_long_rows(dev, K):
    """Rows longer than registers hold, without a value that would send them to 64 bits."""
    rng = np.random.default_rng(K)
    same(dev, (3 * rng.standard_normal((3, K))).astype(np.float32), rng.standard_normal((3, K)).astype(np.float32))


@pytest.mark.parametrize("K", LENGTHS)
@pytest.mark.parametrize("low,high", [(-5, 5), (-63.99, -40), (-64.5, -63.5), (5, 80), (1e-30, 1e-3)])
def test_borders_with_gate(dev, low, high, K):
    """SiLU(gate) * x up to three steps of f32 from the middle of two codes, for gates of each part of the range."""
    rng = np.random.default_rng(int(K + 10 * low))
    gate = rng.uniform(low, high, (6, K)).astype(np.float32)
    if low == 1e-30:
        gate = np.exp(rng.uniform(np.log(low), np.log(high), (6, K))).astype(np.float32)
    a = R.act(gate)
    x = np.empty((6, K), np.float32)
    for m in range(6):
        top = np.exp(3 * rng.standard_normal()) * np.abs(a[m, 0])
        x[m, 0] = top / a[m, 0]
        s = float(np.float32(a[m, 0] * float(x[m, 0]) / 127))
        x[m] = s * (rng.integers(-126, 126, K) + 0.5) / a[m]
        x[m, 0] = top / a[m, 0]
        x[m, 1:] = (x[m, 1:].view(np.int32) + rng.integers(-3, 4, K - 1).astype(np.int32)).view(np.float32)
    assert np.isfinite(x).all()
    same(dev, gate, x)
