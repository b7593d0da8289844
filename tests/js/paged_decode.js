// Drives qkNormRope and the paged cache through the Node-API addon: a small decoding run against a model in plain
// doubles, gradients, eviction and the errors a caller sees.  Needs a GPU.
'use strict';
const path = require('path');
const native = require(path.join(__dirname, '..', '..', 'framework_amd', 'lib', 'mni_rocm.node'));

let passed = 0, failed = 0;
function assert(cond, msg) { if (cond) { passed++; } else { failed++; console.log('FAIL: ' + msg); } }
function assertClose(a, b, tol, msg) { assert(Math.abs(a - b) <= tol, msg + ' (got ' + a + ', want ' + b + ')'); }
function assertThrows(f, text, msg) {
  try { f(); } catch (e) { assert(e.message.includes(text), msg + ': ' + e.message); return; }
  assert(false, msg + ': nothing was thrown');
}
function lcg(seed) { let s = seed >>> 0; return () => { s = (Math.imul(s, 1664525) + 1013904223) >>> 0; return s / 4294967296; }; }
const rnd = lcg(11);
function rand(n) { const a = new Float32Array(n); for (let i = 0; i < n; i++) a[i] = 2 * rnd() - 1; return a; }
const tensor = (a, shape) => native.fromFloat32(a, shape);

const H = 2, GROUP = 2, D = 16, THETA = 10000, EPS = 1e-6;

// ---- norm and rotation ---------------------------------------------------------------------
function rotate(row, gain, position) {  // split halves, all dims
  let ss = 0;
  for (const x of row) ss += x * x;
  const r = 1 / Math.sqrt(ss / D + EPS), out = new Float64Array(D);
  for (let i = 0; i < D / 2; i++) {
    const a = position * Math.pow(THETA, -2 * i / D), lo = row[i] * r * gain[i], hi = row[i + D / 2] * r * gain[i + D / 2];
    out[i] = lo * Math.cos(a) - hi * Math.sin(a);
    out[i + D / 2] = hi * Math.cos(a) + lo * Math.sin(a);
  }
  return out;
}
const S = 3, q0 = rand(H * GROUP * S * D), k0 = rand(H * S * D), gq = rand(D), gk = rand(D);
const ids = [tensor(q0, [1, H * GROUP, S, D]), tensor(k0, [1, H, S, D]), tensor(gq, [D]), tensor(gk, [D])];
ids.forEach(i => native.setRequiresGrad(i, true));
const [qr, kr] = native.qkNormRope(ids[0], ids[1], ids[2], ids[3], null, 5, D, false, THETA, EPS);
const qv = native.toFloat32(qr), kv = native.toFloat32(kr);
// (D / 2 + 10) half steps of the two products, each at most the largest row norm times gain, sqrt(D) here
const TOL = 2 * (D / 2 + 10) * Math.pow(2, -24) * 2 * Math.sqrt(D);
for (let row = 0; row < H * GROUP * S; row++) {
  const want = rotate(q0.subarray(row * D, row * D + D), gq, 5 + row % S);
  for (let e = 0; e < D; e++) assertClose(qv[row * D + e], want[e], TOL, 'rotated query ' + row + ' ' + e);
}
native.backward(native.add(native.sumAll(qr), native.sumAll(kr)));
for (const [i, n] of [[0, q0.length], [1, k0.length], [2, D], [3, D]]) {
  const g = native.getGrad(ids[i]);
  assert(g != null && native.toFloat32(g).length === n && native.toFloat32(g).every(Number.isFinite), 'gradient of input ' + i);
}
// the gain's gradient against a difference of the sum of outputs (a quotient of doubles, off by 1e-9; the sum over S * H
// rows of values of order 1 in fp32: 1e-5 is a hundred of its steps)
const total = g => { let t = 0; for (let row = 0; row < H * S; row++) for (const x of rotate(k0.subarray(row * D, row * D + D), g, 5 + row % S)) t += x; return t; };
const gg = native.toFloat32(native.getGrad(ids[3]));
for (let e = 0; e < D; e += 5) {
  const up = Float64Array.from(gk), down = Float64Array.from(gk);
  up[e] += 1e-5; down[e] -= 1e-5;
  assertClose(gg[e], (total(up) - total(down)) / 2e-5, 1e-5, 'gain gradient ' + e);
}

// ---- paged cache ----------------------------------------------------------------------------
const cache = native.pagedCacheCreate(3, 32, 9, 4, H, D, false, true);
const a = native.pagedCacheAdd(cache), b = native.pagedCacheAdd(cache), held = { [a]: [], [b]: [] };
const k1 = rand(2 * H * 6 * D), v1 = rand(2 * H * 6 * D);
native.pagedCacheAppend(cache, [a, b], tensor(k1, [2, H, 6, D]), tensor(v1, [2, H, 6, D]), [6, 2]);
function take(seq, i, k, v, tokens, count) {
  for (let t = 0; t < count; t++) {
    const at = h => ((i * H + h) * tokens + t) * D;
    held[seq].push({ k: [0, 1].map(h => k.subarray(at(h), at(h) + D)), v: [0, 1].map(h => v.subarray(at(h), at(h) + D)) });
  }
}
take(a, 0, k1, v1, 6, 6); take(b, 1, k1, v1, 6, 2);
const k2 = rand(2 * H * D), v2 = rand(2 * H * D), q2 = rand(2 * H * GROUP * D);
native.pagedCacheAppend(cache, new Uint32Array([a, b]), tensor(k2, [2, H, 1, D]), tensor(v2, [2, H, 1, D]), null);
take(a, 0, k2, v2, 1, 1); take(b, 1, k2, v2, 1, 1);
assert(native.pagedCacheLen(cache, a) === 7 && native.pagedCacheSeen(cache, b) === 3, 'lengths');
assert(native.pagedCacheFreePages(cache) === 6, 'three pages are held');
const out = native.toFloat32(native.pagedCacheAttend(cache, [a, b], tensor(q2, [2, H * GROUP, 1, D]), 0.25, true));
[a, b].forEach((seq, i) => {
  for (let j = 0; j < H * GROUP; j++) {
    const q = q2.subarray((i * H * GROUP + j) * D, (i * H * GROUP + j + 1) * D), h = Math.floor(j / GROUP);
    const p = held[seq].map(r => { let s = 0; for (let e = 0; e < D; e++) s += q[e] * r.k[h][e]; return Math.exp(0.25 * s); });
    const sum = p.reduce((x, y) => x + y);
    for (let e = 0; e < D; e++) {
      const want = held[seq].reduce((x, r, t) => x + p[t] / sum * r.v[h][e], 0);
      assertClose(out[(i * H * GROUP + j) * D + e], want, 1e-5, 'attention ' + seq + ' ' + j + ' ' + e);  // values of order 1
    }
  }
});
const [w, pos] = native.pagedCacheTrack(cache, [a]);
const weights = native.toFloat32(w), positions = Array.from(native.intBufferToInt32(pos));
for (let h = 0; h < H; h++) {
  let sum = 0;
  for (let t = 0; t < 7; t++) sum += weights[h * 7 + t];
  assertClose(sum, GROUP, 1e-5, 'weights of key head ' + h);
}
assert(positions.join() === '0,1,2,3,4,5,6,0,1,2,3,4,5,6', 'positions');
const more = new Float32Array(H * 7); more[0] = more[7 + 3] = 9;
native.pagedCacheAddWeights(cache, [a], tensor(more, [1, H, 7]));
const c = native.pagedCacheFork(cache, a);
native.pagedCacheEvict(cache, [a], 3, 2);
const kept = native.toFloat32(native.pagedCacheRead(cache, a)[0]);
assert(kept.slice(0, D).every((x, e) => x === held[a][0].k[0][e]), 'the heaviest row of head 0 keeps its place');
const row3 = held[a][3].k[1];
assert([0, 1, 2].some(t => kept.slice((3 + t) * D, (4 + t) * D).every((x, e) => x === row3[e])), 'the heaviest row of head 1 stays');
assert(native.pagedCacheLen(cache, a) === 3 && native.pagedCacheLen(cache, c) === 7, 'a fork is not evicted with its parent');
native.pagedCacheTruncate(cache, [b, c], [1, 5]);
assert(native.pagedCacheLen(cache, b) === 1 && native.pagedCacheSeen(cache, c) === 5, 'truncated');
native.pagedCacheDrop(cache, c);

// ---- errors -----------------------------------------------------------------------------------
assertThrows(() => native.pagedCacheTruncate(cache, [a], [2]), 'cannot be cut to 2', 'evicted rows do not leave by truncation');
assertThrows(() => native.pagedCacheTruncate(cache, [a, b], [3]), 'as many lengths', 'one length for two sequences');
assertThrows(() => native.pagedCacheAppend(cache, [a, a], tensor(k2, [2, H, 1, D]), tensor(v2, [2, H, 1, D]), null), 'occurs twice', 'a sequence twice');
assertThrows(() => native.pagedCacheLen(cache, c), 'invalid paged cache sequence id', 'a dropped sequence');
assertThrows(() => native.pagedCacheAdd(77), 'invalid paged cache id', 'an unknown cache');
assertThrows(() => native.qkNormRope(ids[0], ids[1], ids[2], ids[3], null, 0, 3, false, THETA, EPS), 'must be even', 'odd rotary dims');
assertThrows(() => native.pagedCacheEvict(cache, a, 1, 0), 'an array of sequence ids', 'an id where a list is wanted');
native.pagedCacheFree(cache);
assertThrows(() => native.pagedCacheFreePages(cache), 'invalid paged cache id', 'a freed cache');

console.log(passed + ' passed, ' + failed + ' failed');
process.exit(failed ? 1 : 0);
