"""The argument checks and plans of the experts' and 8-bit products' entry points on the host: the same functions that the entry
points call, compiled into a small driver (tests/native/moe_check.cpp); and the reference forms that the GPU tests compare with."""
import os
import subprocess

import numpy as np

import moeref as R

HERE = os.path.dirname(os.path.abspath(__file__))


def test_checks_and_plans(tmp_path):
    exe = str(tmp_path / "moe_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    os.path.join(HERE, "native", "moe_check.cpp"), "-o", exe], check=True)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.strip() == "ok", p.stdout + p.stderr


def test_the_reference_itself():
    """moeref's routing by a loop over the experts, its gradient against differences, its codes by fractions."""
    from fractions import Fraction
    rng = np.random.default_rng(0)
    logits = rng.integers(-3, 4, (20, 7)) / 2.0
    logits[3, 2:] = -np.inf
    for sigmoid in (False, True):
        ids, w = R.route(logits, 3, sigmoid, renorm=True, scale=2.0)
        for t in range(20):
            s = 1 / (1 + np.exp(-logits[t])) if sigmoid else np.exp(logits[t]) / np.exp(logits[t]).sum()
            left, want = [e for e in range(7) if logits[t, e] > -np.inf], []
            while left and len(want) < 3:
                e = max(left, key=lambda e: (logits[t, e], -e))
                left.remove(e)
                want.append(e)
            assert ids[t].tolist() == want + [-1] * (3 - len(want))
            assert np.allclose(w[t, : len(want)], 2 * s[want] / s[want].sum(), rtol=1e-12) and (w[t, len(want):] == 0).all()
    row_off, src, slot = R.sort(np.array([[2, 0], [0, 9], [2, -1]]), 3)
    assert row_off.tolist() == [0, 2, 2, 4] and src.tolist() == [1, 2, 0, 4, -1, -1] and slot.tolist() == [[2, 0], [1, -1], [3, -1]]
    l, dw = rng.standard_normal((2, 6)), rng.standard_normal((2, 3))
    for sigmoid in (False, True):
        for renorm in (False, True):
            ids, _ = R.route(l, 3, sigmoid, renorm, 1.5)
            got, _ = R.route_grad(l, ids, dw, sigmoid, renorm, 1.5)
            def loss(x):
                s = np.take_along_axis(R.scores(x, sigmoid), ids, -1)
                return 1.5 * (dw * (s / s.sum(-1, keepdims=True) if renorm else s)).sum()
            for t in range(2):
                for e in range(6):
                    d = np.zeros_like(l)
                    d[t, e] = 1e-6
                    assert abs((loss(l + d) - loss(l - d)) / 2e-6 - got[t, e]) < 1e-8
    x = rng.standard_normal((3, 32)).astype(np.float32)
    codes, scales = R.quantize(x)
    for m in range(3):
        for i in range(32):
            q = Fraction(float(x[m, i])) / Fraction(float(scales[m])) + Fraction(1, 2)
            assert codes[m, i] == max(-127, min(127, q.numerator // q.denominator))
