'use strict';
// The JavaScript host's cache and attention methods against plain loops in doubles on seeded inputs. Prints one JSON line;
// exit code 0 iff every check passed. Run by tests/test_js_attention.py.
const path = require('path');
const brik = require(path.join(__dirname, '..', '..', 'brimkern_amd', 'js'));

const results = [];
function check(name, ok, detail) {
  results.push({ name: name, ok: !!ok, detail: detail });
  if (!ok) console.error('FAIL ' + name + ' ' + JSON.stringify(detail));
}

// |y - r| / |r| over all values
function apart(y, r) {
  let num = 0, den = 0;
  for (let i = 0; i < r.length; i++) { num += (y[i] - r[i]) * (y[i] - r[i]); den += r[i] * r[i]; }
  return Math.sqrt(num / den);
}

function values(n, seed) {   // sums of uniform numbers, seeded
  let a = seed >>> 0;
  const next = function () {
    a = (Math.imul(a, 1664525) + 1013904223) >>> 0;
    return a / 4294967296 - 0.5;
  };
  return Float32Array.from({ length: n }, function () { return 2 * (next() + next() + next()); });
}

// heads of a row: normed by gain g, then pairs (i, i + D / 2) rotated by p * freq[i]
function normRope(x, rows, heads, D, g, eps, freq, pos) {
  const y = new Float64Array(x.length);
  for (let t = 0; t < rows; t++) {
    for (let h = 0; h < heads; h++) {
      const o = (t * heads + h) * D;
      let ss = 0;
      for (let i = 0; i < D; i++) ss += x[o + i] * x[o + i];
      const inv = 1 / Math.sqrt(ss / D + eps);
      for (let i = 0; i < D / 2; i++) {
        const c = Math.cos(pos[t] * freq[i]), s = Math.sin(pos[t] * freq[i]);
        const a = x[o + i] * inv * g[i], b = x[o + i + D / 2] * inv * g[i + D / 2];
        y[o + i] = a * c - b * s;
        y[o + i + D / 2] = b * c + a * s;
      }
    }
  }
  return y;
}

// one sequence: rows at positions len - rows ..., keys and values [len, KV, D]
function attend(q, k, v, rows, len, H, KV, D, scale, window) {
  const out = new Float64Array(rows * H * D);
  for (let t = 0; t < rows; t++) {
    const p = len - rows + t, from = window ? Math.max(0, p - window + 1) : 0;
    for (let h = 0; h < H; h++) {
      const g = Math.floor(h / (H / KV)), x = [];
      for (let j = from; j <= p; j++) {
        let s = 0;
        for (let i = 0; i < D; i++) s += q[(t * H + h) * D + i] * k[(j * KV + g) * D + i];
        x.push(s * scale);
      }
      const top = Math.max.apply(null, x);
      let sum = 0;
      x.forEach(function (s, j) {
        const w = Math.exp(s - top);
        sum += w;
        for (let i = 0; i < D; i++) out[(t * H + h) * D + i] += w * v[((from + j) * KV + g) * D + i];
      });
      for (let i = 0; i < D; i++) out[(t * H + h) * D + i] /= sum;
    }
  }
  return out;
}

async function run(engine, dtype) {
  const H = 6, KV = 2, D = 64, P = 16, lens = [37, 5], T = 42, eps = 1e-5;
  const dev = function (a) { return engine.uploadGpuRaw(a); };
  const cache = engine.kvCache(dtype, KV, D, P, 8);
  const x = { q: values(T * H * D, 1), k: values(T * KV * D, 2), v: values(T * KV * D, 3) };
  const g = values(D, 4).map(function (e) { return 1 + e / 4; }), freq = Float32Array.from({ length: D / 2 }, function (_, i) { return Math.pow(1e4, -2 * i / D); });
  const pos = Array.from({ length: T }, function (_, t) { return t < 37 ? t : t - 37; });
  const b = { q: dev(x.q), k: dev(x.k), v: dev(x.v), g: dev(g), f: dev(freq), off: dev(Int32Array.from([0, 37, 42])),
    len: dev(Int32Array.from(lens)), table: dev(Int32Array.from([6, 1, 3, 2, 0, 0])) };
  const batch = { seqs: 2, rows: T, rowOff: b.off, kvLen: b.len, table: b.table, tableCols: 3, maxLen: 40 };
  const rows = { heads: H, kvHeads: KV, headDim: D, q: b.q, k: b.k, v: b.v, qOut: b.q, qNorm: b.g, kNorm: b.g, eps: eps, invFreq: b.f, rotDim: D };
  engine.kvWrite(cache, batch, rows);
  const qr = await engine.readBackAsync(b.q, 4 * T * H * D);
  // one rounding to f32, half a step
  check(dtype + ': q normed and rotated', apart(qr, normRope(x.q, T, H, D, g, eps, freq, pos)) < 2 ** -24, {});
  const kb = engine.alloc(4 * T * KV * D), vb = engine.alloc(4 * T * KV * D);
  engine.kvRead(cache, batch, kb, vb);
  const k = await engine.readBackAsync(kb, 4 * T * KV * D), v = await engine.readBackAsync(vb, 4 * T * KV * D);
  // a value is at most half a step of its group off: q8 a 254th of the group's largest, q4 a 30th of its range
  const half = dtype === 'q8' ? 1 / 254 : 1 / 30, kw = normRope(x.k, T, KV, D, g, eps, freq, pos);
  const within = function (got, want) {
    for (let o = 0; o < want.length; o += 32) {
      const w = Array.from(want.slice(o, o + 32));
      const range = dtype === 'q8' ? Math.max.apply(null, w.map(Math.abs)) : Math.max.apply(null, w) - Math.min.apply(null, w);
      const top = Math.max.apply(null, w.map(Math.abs));
      // scale and min are rounded to halves: 15 (127) steps of 2^-11 of the scale and 2^-11 of the min
      if (!w.every(function (e, i) { return Math.abs(got[o + i] - e) <= range * half + 2 ** -11 * (range + 2 * top); })) return false;
    }
    return true;
  };
  check(dtype + ': keys within half a step', within(k, kw), {});
  check(dtype + ': values within half a step', within(v, x.v), {});
  for (const window of [0, 9]) {
    const out = engine.attention(cache, batch, { q: b.q, heads: H, window: window });
    const y = await engine.readBackAsync(out, 4 * T * H * D);
    const part = function (a, n, t0, t1) { return a.subarray(t0 * n, t1 * n); };
    let far = 0;
    [[0, 37], [37, 42]].forEach(function (r, s) {
      far = Math.max(far, apart(part(y, H * D, r[0], r[1]),
        attend(part(qr, H * D, r[0], r[1]), part(k, KV * D, r[0], r[1]), part(v, KV * D, r[0], r[1]), r[1] - r[0], lens[s], H, KV, D, 1 / 8, window)));
    });
    // halves' parts of 22 bits in both products and f32 sums of at most 64 terms: 64 roundings of 2^-24
    check(dtype + ': attention, window ' + window, far < 64 * 2 ** -24, { far: far });
    out.destroy();
  }
  // one more token of the first sequence, recorded: the replay reads the lengths anew
  const one = { seqs: 1, rows: 1, kvLen: b.len, table: b.table, tableCols: 3, maxLen: 40 };
  const nq = dev(values(H * D, 5)), nk = dev(values(KV * D, 6)), nv = dev(values(KV * D, 7)), no = engine.alloc(4 * H * D);
  const step = function () {
    engine.kvWrite(cache, one, { kvHeads: KV, headDim: D, k: nk, v: nv });
    engine.attention(cache, one, { q: nq, out: no, heads: H });
  };
  step();
  const graph = engine.record(step);
  for (const len of [38, 39, 38]) {
    engine.writeBuffer(b.len, Int32Array.from([len]));
    graph.launch();
    const y = await engine.readBackAsync(no, 4 * H * D);
    engine.kvRead(cache, Object.assign({}, batch, { seqs: 1, rows: len, rowOff: null, maxLen: 40 }), kb, vb);
    const kk = await engine.readBackAsync(kb, 4 * len * KV * D), vv = await engine.readBackAsync(vb, 4 * len * KV * D);
    const far = apart(y, attend(values(H * D, 5), kk, vv, 1, len, H, KV, D, 1 / 8, 0));
    check(dtype + ': recorded step of ' + len, far < 64 * 2 ** -24, { far: far });
  }
  graph.destroy();
  const refused = function (name, f, code) {
    let got = null;
    try { f(); } catch (e) { got = e.code; }
    check(dtype + ': ' + name, got === code, { code: got });
  };
  const live = engine.liveBuffers();
  refused('heads not shared evenly', function () { engine.attention(cache, batch, { q: b.q, heads: 5 }); }, 'BRIK_EINVAL');
  check(dtype + ': the output of a refused call is freed', engine.liveBuffers() === live, {});
  refused('no q and no k: nothing to do, no error', function () { engine.qkNormRope(batch, { heads: H, headDim: D, qOut: b.q }); }, null);
  refused('q without qOut', function () { engine.qkNormRope(batch, { heads: H, headDim: D, q: b.q }); }, 'BRIK_EINVAL');
  refused('a size that is no integer', function () { engine.attention(cache, batch, { q: b.q, heads: 6.5 }); }, 'BRIK_EINVAL');
  refused('a size past 32 bits', function () { engine.kvRead(cache, Object.assign({}, batch, { rows: 4294967297 }), kb, null); }, 'BRIK_EINVAL');
  refused('no cache', function () { engine.kvRead(null, batch, kb, null); }, 'BRIK_EINVAL');
  refused('q3', function () { engine.kvCache('q3', 1, 64, 16, 1); }, 'BRIK_EINVAL');
  Object.keys(b).forEach(function (n) { b[n].destroy(); });
  [kb, vb, nq, nk, nv, no].forEach(function (e) { e.destroy(); });
  cache.destroy();
}

async function main() {
  const engine = new brik.Engine(0);
  const before = engine.liveBuffers();
  await run(engine, 'q8');
  await run(engine, 'q4');
  check('all buffers freed', engine.liveBuffers() === before, { live: engine.liveBuffers() });
  const failed = results.filter(function (r) { return !r.ok; }).length;
  process.stdout.write(JSON.stringify({ checks: results.length, failed: failed }) + '\n');
  process.exit(failed === 0 ? 0 : 1);
}

main().catch(function (e) { console.error(e && e.stack ? e.stack : e); process.exit(2); });
