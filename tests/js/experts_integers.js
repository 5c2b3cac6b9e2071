'use strict';
// Sizes that are no 32-bit integers, at every place of every method of experts and 8-bit products: each is refused, and nothing is
// computed. Prints one JSON line: the calls that were taken. Run by tests/test_js_experts_args.py.
const path = require('path');
const brik = require(path.join(__dirname, '..', '..', 'brimkern_amd', 'js'));

const eng = new brik.Engine(0);
const b = eng.uploadGpuRaw(new Float32Array(1 << 14));
const h = { i8: b, isc: b };
// (every buffer holds 64 KiB, more than any of these calls reads or writes; ids, slots and offsets are 0)
const calls = {
  moeSort: [function (s) { eng.moeSort(b, b.view(16384), b.view(32768), b.view(49152), s[0], s[1], s[2]); }, [4, 2, 8]],
  moeDispatch: [function (s) { eng.moeDispatch(b, b.view(16384), null, b.view(32768), s[0], s[1], s[2]); }, [1, 1, 8]],
  moeCombine: [function (s) { eng.moeCombine(b, b.view(16384), null, null, b.view(32768), s[0], s[1], s[2]); }, [1, 1, 8]],
  moeCombineGrad: [function (s) { eng.moeCombineGrad(b, b.view(8192), b.view(16384), null, b.view(32768), b.view(49152), s[0], s[1], s[2]); }, [1, 1, 8]],
  quantizeI8: [function (s) { eng.quantizeI8(b, s[0], s[1], { out: { i8: b.view(16384), isc: b.view(32768) } }); }, [2, 64]],
  mmI8: [function (s) { eng.mmI8(h, h, s[0], s[1], s[2], { out: b.view(32768) }); }, [2, 64, 8]],
  moeMatmulI8: [function (s) { eng.moeMatmulI8(h, b.view(16384), h, b.view(32768), s[0], s[1], s[2], s[3], { src: b.view(49152), k: s[4], xRows: s[5] }); },
    [2, 4, 64, 8, 2, 2]],
  moeRoute: [function (s) { eng.moeRoute({ logits: b, ids: b.view(32768), weights: b.view(49152), tokens: s[0], experts: s[1], k: s[2] }); }, [4, 8, 2]],
};
const taken = [];
for (const name of Object.keys(calls)) {
  const run = calls[name][0], good = calls[name][1];
  run(good);
  for (let i = 0; i < good.length; i++) {
    for (const v of [good[i] + 0.5, good[i] + 4294967296, good[i] - 4294967296, NaN, Infinity, undefined, String(good[i])]) {
      if (name === 'moeRoute' && v === undefined) continue;                    // (a field that is left out is 0)
      if (name === 'moeMatmulI8' && i === 5 && v === undefined) continue;      // (rows / k)
      if (name === 'quantizeI8' && v === undefined) continue;                  // (refused by the facade, or a field left out)
      const s = good.slice();
      s[i] = v;
      try { run(s); taken.push(name + ' ' + i + ' ' + v); } catch (e) { if (e.code !== 'BRIK_EINVAL') taken.push(name + ' ' + i + ' ' + v + ' ' + e); }
    }
  }
}
eng.readGpu(b, 4).then(function () { console.log(JSON.stringify(taken)); });
