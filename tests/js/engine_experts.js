'use strict';
// The JavaScript host's experts and 8-bit products against plain loops in doubles on seeded inputs: routing, sorting, gate and up
// projections of quantized tokens, SwiGLU into 8 bits, down projections and back, gradients, refusals. Prints one JSON line; exit
// code 0 iff every check passed. Run by tests/test_js_experts.py.
const path = require('path');
const brik = require(path.join(__dirname, '..', '..', 'brimkern_amd', 'js'));

const results = [];
function check(name, ok, detail) {
  results.push({ name: name, ok: !!ok, detail: detail });
  if (!ok) console.error('FAIL ' + name + ' ' + JSON.stringify(detail));
}

function values(n, seed) {   // sums of uniform numbers, seeded
  let a = seed >>> 0;
  const next = function () {
    a = (Math.imul(a, 1664525) + 1013904223) >>> 0;
    return a / 4294967296 - 0.5;
  };
  return Float32Array.from({ length: n }, function () { return 2 * (next() + next() + next()); });
}

const HALF = Math.pow(2, -24);

function quantized(h, M, K) {   // codes and scales of rows of doubles
  const codes = new Int8Array(M * K), sc = new Float32Array(M);
  for (let m = 0; m < M; m++) {
    let top = 0;
    for (let i = 0; i < K; i++) top = Math.max(top, Math.abs(h[m * K + i]));
    sc[m] = top / 127;
    for (let i = 0; i < K; i++) codes[m * K + i] = sc[m] ? Math.max(-127, Math.min(127, Math.floor(h[m * K + i] / sc[m] + 0.5))) : 0;
  }
  return { codes: codes, sc: sc };
}

async function main() {
  const eng = new brik.Engine(0);
  const T = 37, E = 8, k = 2, H = 64, F = 96, n = T * k;
  const up = function (a) { return eng.uploadGpuRaw(a); };
  const ints = function (len) { return eng.alloc(4 * len); };
  const read = async function (b, Type, len) {
    return new Type((await eng.native.readbackAsync(eng.ctx, b.ptr, len * Type.BYTES_PER_ELEMENT)));
  };
  const logits = values(T * E, 1), x = values(T * H, 2), wgu = values(E * 2 * F * H, 3), wd = values(E * H * F, 4);
  const r = { logits: up(logits), tokens: T, experts: E, k: k, ids: ints(n), weights: ints(n), rowOff: ints(E + 1), src: ints(n), slot: ints(n),
    renorm: true };
  eng.moeRoute(r);
  const ids = await read(r.ids, Int32Array, n), w = await read(r.weights, Float32Array, n), off = await read(r.rowOff, Int32Array, E + 1);
  const src = await read(r.src, Int32Array, n), slot = await read(r.slot, Int32Array, n);
  let same = true, near = true;
  for (let t = 0; t < T; t++) {
    const order = Array.from({ length: E }, function (_, e) { return e; });
    order.sort(function (a, b) { return logits[t * E + b] - logits[t * E + a] || a - b; });
    let sum = 0;
    for (let j = 0; j < k; j++) sum += Math.exp(logits[t * E + order[j]]);
    for (let j = 0; j < k; j++) {
      same = same && ids[t * k + j] === order[j];
      // exponentials of differences up to 6, off by 8 half steps each, their sum and quotient
      near = near && Math.abs(w[t * k + j] * sum / Math.exp(logits[t * E + order[j]]) - 1) <= 24 * HALF;
    }
  }
  check('ids', same);
  check('weights', near);
  let row = 0, sorted = off[0] === 0;
  for (let e = 0; e < E; e++) {
    for (let a = 0; a < n; a++) {
      if (ids[a] !== e) continue;
      sorted = sorted && src[row] === a && slot[a] === row;
      row++;
    }
    sorted = sorted && off[e + 1] === row;
  }
  check('sorted', sorted);
  const off2 = ints(E + 1), src2 = ints(n), slot2 = ints(n);
  eng.moeSort(r.ids, off2, src2, slot2, T, k, E);
  check('sort alone', JSON.stringify(Array.from(await read(slot2, Int32Array, n))) === JSON.stringify(Array.from(slot)));

  const gu = eng.quantizeI8(up(wgu), E * 2 * F, H), dn = eng.quantizeI8(up(wd), E * H, F), xd = up(x), xq = eng.quantizeI8(xd, T, H);
  const wantX = quantized(x, T, H), wantG = quantized(wgu, E * 2 * F, H), wantD = quantized(wd, E * H, F);
  const gotX = await read(xq.i8, Int8Array, T * H);
  check('codes', gotX.every(function (c, i) { return c === wantX.codes[i]; }));
  const y = eng.alloc(4 * n * 2 * F), ys = eng.alloc(4 * n * H), out = eng.alloc(4 * T * H);
  eng.moeMatmulI8(xq, r.rowOff, gu, y, E, n, H, 2 * F, { src: r.src, k: k });
  const g = await read(y, Float32Array, n * 2 * F);
  const product = function (got, rows, N, K, xc, xs, xrow, wc, ws) {
    let ok = true;
    for (let e = 0; e < E; e++) {
      for (let m = off[e]; m < off[e + 1]; m++) {
        for (let c = 0; c < N; c++) {
          let s = 0;
          const xr = xrow(m) * K, wr = (e * N + c) * K;
          for (let i = 0; i < K; i++) s += xc[xr + i] * wc[wr + i];
          const want = s * ws[e * N + c] * xs[xrow(m)];
          ok = ok && Math.abs(got[m * N + c] - want) <= 3.01 * HALF * Math.abs(want);
        }
      }
    }
    return ok;
  };
  check('gate and up', product(g, n, 2 * F, H, wantX.codes, wantX.sc, function (m) { return Math.floor(src[m] / k); }, wantG.codes, wantG.sc));
  const hq = eng.quantizeI8({ ptr: y.ptr + BigInt(4 * F) }, n, F, { gate: y, xStride: 2 * F, gateStride: 2 * F });
  const h = new Float64Array(n * F);
  for (let m = 0; m < n; m++)
    for (let i = 0; i < F; i++) h[m * F + i] = g[m * 2 * F + i] / (1 + Math.exp(-g[m * 2 * F + i])) * g[m * 2 * F + F + i];
  const wantH = quantized(h, n, F), gotH = await read(hq.i8, Int8Array, n * F);
  check('codes of the gated rows', gotH.every(function (c, i) { return c === wantH.codes[i]; }));
  eng.moeMatmulI8(hq, r.rowOff, dn, ys, E, n, F, H);
  const d = await read(ys, Float32Array, n * H);
  check('down', product(d, n, H, F, wantH.codes, wantH.sc, function (m) { return m; }, wantD.codes, wantD.sc));
  eng.moeCombine(ys, r.slot, r.weights, xd, out, T, k, H);
  const o = await read(out, Float32Array, T * H);
  let back = true;
  for (let t = 0; t < T; t++) {
    for (let i = 0; i < H; i++) {
      let s = x[t * H + i], size = Math.abs(s);
      for (let j = 0; j < k; j++) {
        const v = w[t * k + j] * d[slot[t * k + j] * H + i];
        s += v;
        size += Math.abs(v);
      }
      back = back && Math.abs(o[t * H + i] - s) <= (k + 2) * HALF * size;
    }
  }
  check('back', back);
  const xs = eng.alloc(4 * n * H), dw = ints(n), dl = eng.alloc(4 * T * E);
  eng.moeDispatch(xd, r.slot, null, xs, T, k, H);
  const spread = await read(xs, Float32Array, n * H);
  check('there', spread.every(function (v, i) { return v === x[Math.floor(src[Math.floor(i / H)] / k) * H + i % H]; }));
  eng.moeCombineGrad(xd, ys, r.slot, r.weights, xs, dw, T, k, H);
  eng.moeRouteGrad(r, dw, dl);
  const gw = await read(dw, Float32Array, n), gl = await read(dl, Float32Array, T * E);
  let gradient = true;
  for (let t = 0; t < T; t++) {
    let mean = 0, size = 0;
    for (let j = 0; j < k; j++) {
      let s = 0, abs = 0;
      for (let i = 0; i < H; i++) {
        s += x[t * H + i] * d[slot[t * k + j] * H + i];
        abs += Math.abs(x[t * H + i] * d[slot[t * k + j] * H + i]);
      }
      gradient = gradient && Math.abs(gw[t * k + j] - s) <= 14 * HALF * abs;
      mean += w[t * k + j] * gw[t * k + j];
      size += w[t * k + j] * Math.abs(gw[t * k + j]);
    }
    for (let j = 0; j < k; j++) {
      const want = w[t * k + j] * (gw[t * k + j] - mean);
      gradient = gradient && Math.abs(gl[t * E + ids[t * k + j]] - want) <= 64 * HALF * w[t * k + j] * (Math.abs(gw[t * k + j]) + size);
    }
  }
  check('gradients', gradient);
  const dense = eng.mmI8(xq, { i8: gu.i8, isc: gu.isc }, T, H, 2 * F);
  const yd = await read(dense, Float32Array, T * 2 * F);
  let s0 = 0;
  for (let i = 0; i < H; i++) s0 += wantX.codes[i] * wantG.codes[i];
  check('dense', Math.abs(yd[0] - s0 * wantG.sc[0] * wantX.sc[0]) <= 3.01 * HALF * Math.abs(yd[0]) + 1e-30);
  const refused = function (name, f) {
    let code = null;
    try { f(); } catch (e) { code = e.code; }
    check('refuses ' + name, code === 'BRIK_EINVAL' || code === 'BRIK_EALIGN', code);
  };
  refused('k over experts', function () { eng.moeRoute(Object.assign({}, r, { k: 9 })); });
  refused('width', function () { eng.moeCombine(ys, r.slot, null, null, out, T, k, 6); });
  refused('K', function () { eng.quantizeI8(xd, 2, 33); });
  refused('negative rows', function () { eng.quantizeI8(xd, -1, 32); });
  refused('an 8-bit handle as a .brik weight', function () { eng.mm(xd, gu, 1, H, 32); });
  refused('null scales', function () { eng.mmI8(xq, { i8: gu.i8, isc: null }, T, H, 2 * F); });
  const failed = results.filter(function (c) { return !c.ok; }).length;
  console.log(JSON.stringify({ checks: results.length, failed: failed }));
  process.exit(failed ? 1 : 0);
}

main().catch(function (e) { console.error(e.stack); process.exit(2); });
