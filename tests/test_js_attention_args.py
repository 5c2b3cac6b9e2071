"""How the Node facade fills in what a call leaves out, without a device: its methods over a stand-in for the addon."""
import json
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")
pytestmark = pytest.mark.skipif(NODE is None, reason="node not installed")

STUB = """
const { Engine } = require('./brimkern_amd/js');
const seen = [], freed = [];
let left = %d;
const engine = Object.create(Engine.prototype, {
  native: { value: { attention: (ctx, cache, batch, args) => seen.push(args) } }, ctx: { value: 1 },
  alloc: { value: function (n) {
    if (left-- <= 0) throw new Error('out of memory');
    const b = { bytes: n, destroy: function () { freed.push(n); }, view: function (o) { return { at: o }; } };
    return b;
  } } });
"""


def run(script, left=1000):
    r = subprocess.run([NODE, "-e", STUB % left + script], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    return json.loads(r.stdout)


def test_scale_left_out_in_every_way():
    """Absent, undefined and null are the default; 0 is 0."""
    got = run("""
const cache = { headDim: 64 }, batch = { rows: 2 }, out = {};
for (const a of [{}, { scale: undefined }, { scale: null }, { scale: 0 }, { scale: 0.5 }])
  engine.attention(cache, batch, Object.assign({ q: {}, out: out, heads: 4 }, a));
console.log(JSON.stringify(seen.map(a => a.scale)));
""")
    assert got == [0.125, 0.125, 0.125, 0, 0.5]


def test_second_allocation_of_a_cache_fails():
    got = run("""
let said = null;
try { engine.kvCache('q8', 2, 64, 16, 4); } catch (e) { said = e.message; }
console.log(JSON.stringify([said, freed]));
""", left=1)
    assert got[0] == "out of memory" and len(got[1]) == 1


def test_whole_surface_of_the_addon():
    """Every own property of the addon, whether its keys list it or not."""
    from test_js_host import EXPORTS
    r = subprocess.run([NODE, "-e", "console.log(JSON.stringify(Object.getOwnPropertyNames(require('./brimkern_amd/js/brik.node'))))"],
                       cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert sorted(json.loads(r.stdout)) == sorted(EXPORTS + ["qkNormRope", "kvWrite", "kvRead", "attention"])
