"""The cache and attention methods of both hosts: brimkern_amd/js (over the addon) and brimkern_amd.engine."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")


@pytest.mark.skipif(NODE is None, reason="node not installed")
def test_addon_has_the_entry_points():
    r = subprocess.run([NODE, "-e", "const n = require('./brimkern_amd/js/brik.node'); console.log(['qkNormRope', 'kvWrite', 'kvRead', "
                        "'attention'].every(k => typeof n[k] === 'function'))"], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.stdout.strip() == "true", r.stderr


@pytest.mark.gpu
@pytest.mark.skipif(NODE is None, reason="node not installed")
def test_js_attention_on_gpu():
    r = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "engine_attention.js")], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
    res = json.loads(r.stdout.strip().splitlines()[-1])
    assert res["failed"] == 0 and res["checks"] >= 20


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["q8", "q4"])
def test_python_engine(dtype):
    """A prompt, then single tokens, through the engine: outputs are those of the tokens read back, in 64 bits."""
    from brimkern_amd.capi import BrikError
    from brimkern_amd.engine import Engine
    H, KV, D, P, n = 8, 2, 128, 32, 50
    rng = np.random.default_rng(3)
    eng = Engine(0)
    up = lambda a: eng.ctx.upload(np.ascontiguousarray(a))
    cache = eng.kv_cache(dtype, KV, D, P, 4)
    table, length, freq = up(np.array([2, 0, 3], np.int32)), up(np.array([n], np.int32)), up((1e4 ** (-np.arange(64) / 64)).astype(np.float32))
    kb, vb = eng.ctx.alloc(4 * 96 * KV * D), eng.ctx.alloc(4 * 96 * KV * D)
    for rows, total in ((n, n), (1, n + 1), (1, n + 2)):
        q, k, v = (rng.standard_normal((rows, h, D)).astype(np.float32) for h in (H, KV, KV))
        eng.ctx.h2d(length, np.array([total], np.int32))
        batch = eng.kv_batch(1, rows, length, table, 3, 96)
        qd = up(q)
        eng.kv_write(cache, batch, heads=H, q=qd, q_out=qd, k=up(k), v=up(v), inv_freq=freq, rot_dim=D)
        out = eng.attention(cache, batch, qd, H)
        eng.kv_read(cache, eng.kv_batch(1, total, length, table, 3, 96), kb, vb)
        read = lambda b, r, h: eng.ctx.download(b, np.float32, r * h * D).reshape(r, h, D).astype(np.float64)
        qr, kr, vr, got = read(qd, rows, H), read(kb, total, KV), read(vb, total, KV), read(out, rows, H)
        x = np.einsum("thd,jhd->htj", qr, np.repeat(kr, H // KV, 1)) / np.sqrt(D)
        x[:, np.arange(total)[None, :] > total - rows + np.arange(rows)[:, None]] = -np.inf
        p = np.exp(x - x.max(-1, keepdims=True))
        want = np.einsum("htj,jhd->thd", p / p.sum(-1, keepdims=True), np.repeat(vr, H // KV, 1))
        # parts of 22 bits in both products and f32 sums: 64 roundings of 2^-24
        assert np.linalg.norm(got - want) <= 64 * 2.0 ** -24 * np.linalg.norm(want)
    for bad in (lambda: eng.attention(cache, batch, qd, 3), lambda: eng.kv_cache("q3", 1, 64, 16, 1), lambda: eng.kv_cache("q8", 1, 8, 16, 1)):
        with pytest.raises(BrikError):
            bad()
    eng.free_kv_cache(cache)
    eng.close()
