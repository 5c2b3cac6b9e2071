"""The experts' and 8-bit products' methods of both hosts: brimkern_amd/js (over its second addon) and brimkern_amd.engine."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

import moeref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")
NAMES = ["moeRoute", "moeRouteGrad", "moeSort", "moeDispatch", "moeCombine", "moeCombineGrad", "quantizeI8", "matmulI8", "moeMatmulI8"]


@pytest.mark.skipif(NODE is None, reason="node not installed")
def test_addon_exports():
    r = subprocess.run([NODE, "-e", "console.log(JSON.stringify(Object.getOwnPropertyNames(require('./brimkern_amd/js/brik_experts.node'))))"],
                       cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert sorted(json.loads(r.stdout)) == sorted(NAMES)


@pytest.mark.skipif(NODE is None, reason="node not installed")
def test_arguments_are_checked_without_a_device():
    """A context that is none, missing arguments and things that are no pointers throw; nothing ends the process."""
    script = """
const n = require('./brimkern_amd/js/brik_experts.node'), said = [];
for (const f of [() => n.moeRoute(1, {}), () => n.moeRoute(), () => n.moeSort({}), () => n.quantizeI8(null, {}), () => n.matmulI8(undefined, 1, 2, 3, 4, 5, 6, 7, 8, 9),
                 () => n.moeMatmulI8()])
  try { f(); said.push('nothing'); } catch (e) { said.push(e.code); }
console.log(JSON.stringify(said));
"""
    r = subprocess.run([NODE, "-e", script], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert json.loads(r.stdout) == ["BRIK_EINVAL"] * 6


@pytest.mark.gpu
@pytest.mark.skipif(NODE is None, reason="node not installed")
def test_js_experts_on_gpu():
    r = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "engine_experts.js")], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
    res = json.loads(r.stdout.strip().splitlines()[-1])
    assert res["failed"] == 0 and res["checks"] >= 18


@pytest.mark.gpu
def test_python_engine():
    """A feed-forward layer of 8-bit products with its residual, and a routed one, through the engine's handles."""
    from brimkern_amd.capi import BrikError
    from brimkern_amd.engine import Engine
    T, H, F, E, k = 9, 128, 160, 6, 2
    rng = np.random.default_rng(2)
    eng = Engine(0)
    up = lambda a: eng.ctx.upload(np.ascontiguousarray(a, np.float32))
    get = lambda b, *shape, t=np.float32: eng.ctx.download(b, t, int(np.prod(shape))).reshape(shape)
    x, w1, w2 = rng.standard_normal((T, H)), rng.standard_normal((2 * F, H)), rng.standard_normal((H, F))
    xd = up(x)
    xq, a, b = eng.quantize_i8(xd, T, H), eng.quantize_i8(up(w1), 2 * F, H), eng.quantize_i8(up(w2), H, F)
    gu = eng.mm_i8(xq, a, T, H, 2 * F)
    hq = eng.quantize_i8(gu.offset(4 * F), T, F, x_stride=2 * F, gate=gu, gate_stride=2 * F)
    y = get(eng.mm_i8(hq, b, T, F, H, res=xd), T, H)
    (c0, s0), (c1, s1), (c2, s2) = (R.quantize(v.astype(np.float32)) for v in (x, w1, w2))
    g = get(gu, T, 2 * F)
    want, bound = R.product(c0, s0, c1, s1)
    assert (np.abs(g - want) <= bound).all()
    want, bound = R.product(*R.quantize(R.act(g[:, :F]) * g[:, F:]), c2, s2, res=x.astype(np.float32))
    assert (np.abs(y - want) <= bound).all()
    logits, we = rng.standard_normal((T, E)).astype(np.float32), rng.standard_normal((E, 64, H)).astype(np.float32)
    r = eng.moe_route(up(logits), T, E, k, renorm=True)
    ids, _ = R.route(logits, k, renorm=True)
    off, src, slot = R.sort(ids, E)
    assert (get(r["slot"], T, k, t=np.int32) == slot).all()
    wq, ys, out, xs = eng.quantize_i8(up(we), E * 64, H), eng.ctx.alloc(4 * T * k * 64), eng.ctx.alloc(4 * T * 64), eng.ctx.alloc(4 * T * k * H)
    eng.moe_mm_i8(xq, r["row_off"], wq, ys, E, T * k, H, 64, src=r["src"], k=k)
    eng.moe_combine(ys, r["slot"], r["weights"], out, T, k, 64)
    eng.moe_dispatch(xd, r["slot"], xs, T, k, H)
    assert (get(xs, T * k, H) == x.astype(np.float32)[src // k]).all()
    rows, wr = get(ys, T * k, 64).astype(np.float64), get(r["weights"], T, k).astype(np.float64)
    terms = wr[..., None] * rows[slot]
    assert (np.abs(get(out, T, 64) - terms.sum(1)) <= (k + 1) * R.HALF * np.abs(terms).sum(1)).all()
    for bad in (lambda: eng.mm(xd, a, 1, H, 32), lambda: eng.quantize_i8(xd, 1, 33), lambda: eng.quantize_i8(xd, -1, 32),
                lambda: eng.moe_route(xd, T, E, 7), lambda: eng.mm_i8(xq, a, T, 40, 4)):
        with pytest.raises(BrikError):
            bad()
    eng.free_routing(r)
    eng.close()
