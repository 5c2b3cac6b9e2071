"""Products of 8-bit integers with more experts, rows or channels than one kernel's launch has blocks for: another kernel takes them
(tests/native/i8_fits.cpp on the host, one such call on the GPU)."""
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_plans(tmp_path):
    exe = str(tmp_path / "i8_fits")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    os.path.join(HERE, "native", "i8_fits.cpp"), "-o", exe], check=True)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.strip() == "ok", p.stdout + p.stderr


@pytest.mark.gpu
def test_one_row_of_many_experts(ctx):
    """65536 experts of 2048 channels: the kernel of few rows would need 2^23 blocks."""
    import moeref as R
    E, K, N, last = 65536, 32, 2048, 65533
    rng = np.random.default_rng(0)
    x, w = rng.integers(-128, 128, (1, K)).astype(np.int8), rng.integers(-128, 128, (N, K)).astype(np.int8)
    xs, ws = np.float32([0.75]), rng.uniform(0.5, 2, N).astype(np.float32)
    off = np.zeros(E + 1, np.int32)
    off[last + 1:] = 1
    bufs = [ctx.upload(x), ctx.upload(xs), ctx.upload(off), ctx.alloc(E * N * K), ctx.alloc(4 * E * N), ctx.upload(np.full(N, 7, np.float32))]
    try:
        xd, sd, od, wd, wsd, yd = bufs                           # (the other experts' weights do not matter)
        ctx.h2d(wd, w, last * N * K)
        ctx.h2d(wsd, ws, 4 * last * N)
        ctx.moe_matmul_t_i8(xd, sd, od, wd, wsd, yd, E, 1, K, N)
        want, bound = R.product(x, xs, w, ws)
        assert (np.abs(ctx.download(yd, np.float32, N).astype(np.float64) - want[0]) <= bound[0]).all()
    finally:
        for b in bufs:
            ctx.free(b)
