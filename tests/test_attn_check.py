"""The attention side's argument checks, and the look-up of tokens whose page ids are out of range, on the host: the same
functions that the entry points and the kernels call, compiled into a small driver (tests/native/attn_check.cpp)."""
import os
import subprocess

import numpy as np

import kvref as R

HERE = os.path.dirname(os.path.abspath(__file__))


def test_checks_and_token_lookup(tmp_path):
    exe = str(tmp_path / "attn_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    os.path.join(HERE, "native", "attn_check.cpp"), "-o", exe], check=True)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0 and p.stdout.strip() == "ok", p.stdout + p.stderr


def test_the_reference_itself():
    """kvref's attention against a direct sum over a few tokens, its rotation against complex products, its page look-up."""
    rng = np.random.default_rng(0)
    k, v, q = rng.standard_normal((5, 1, 32)), rng.standard_normal((5, 1, 32)), rng.standard_normal((2, 2, 32))
    out = R.attention(q, k, v, 0.5, window=3)
    for t, h in ((0, 0), (1, 1)):
        e = [np.exp(0.5 * q[t, h] @ k[j, 0]) for j in range(1 + t, 4 + t)]
        want = sum(w * v[j, 0] for w, j in zip(e, range(1 + t, 4 + t))) / sum(e)
        assert np.allclose(out[t, h], want, rtol=1e-6)
    assert (R.attention(q, k[:1], v[:1], 1.0)[0] == 0).all()
    x = rng.standard_normal((1, 1, 32)).astype(np.float32)
    freq = (0.1 ** np.arange(8)).astype(np.float32)
    got = R.norm_rope(x, None, 0, False, [11], freq, True)[0, 0]
    z = (x[0, 0, :16:2] + 1j * x[0, 0, 1:16:2].astype(np.float64)) * np.exp(1j * 11 * freq.astype(np.float64))
    assert np.allclose(got[:16:2], z.real, rtol=1e-5) and np.allclose(got[1:16:2], z.imag, rtol=1e-5) and (got[16:] == x[0, 0, 16:]).all()
    for fmt in ("q8", "q4"):
        c = R.Paged(fmt, 2, 64, 16, 4)
        ids = c.take(20)
        y = rng.standard_normal((20, 2, 64)).astype(np.float32)
        c.put(ids, y, y)
        step = 0.02 if fmt == "q8" else 0.25
        assert np.abs(c.get("k", ids, 20) - y).max() < step * np.abs(y).max()
