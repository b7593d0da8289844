// What qkNormRope and the paged cache's exports refuse before they call the library: ids, lengths and numbers that are none.
// No cache exists, so a value that got through would end in another error (or, for pagedCacheFree, in none).  No GPU needed.
'use strict';
const path = require('path');
const native = require(path.join(__dirname, '..', '..', 'framework_amd', 'lib', 'mni_rocm.node'));

let passed = 0, failed = 0;
function assertThrows(f, text, msg) {
  try { f(); } catch (e) {
    if (e.message.includes(text)) { passed++; } else { failed++; console.log('FAIL: ' + msg + ': ' + e.message); }
    return;
  }
  failed++;
  console.log('FAIL: ' + msg + ': nothing was thrown');
}
const notIds = [undefined, null, 'x', '1', {}, true, NaN, Infinity, -1, 0.5, 2 ** 32 - 1, 2 ** 32, 2 ** 53, 5n];
const notCounts = ['x', '1', {}, true, NaN, Infinity, 0.5, 2 ** 53, 5n];
const text = x => typeof x === 'bigint' ? x + 'n' : typeof x === 'object' ? JSON.stringify(x) : String(x);
const calls = {  // with a cache id c and a list of sequences s
  pagedCacheAppend: (c, s) => native.pagedCacheAppend(c, s, 0, 0, null),
  pagedCacheTruncate: (c, s) => native.pagedCacheTruncate(c, s, s instanceof Object && 'length' in s ? Array.from(s, () => 0) : [0]),
  pagedCacheAttend: (c, s) => native.pagedCacheAttend(c, s, 0, 1, false),
  pagedCacheAddWeights: (c, s) => native.pagedCacheAddWeights(c, s, 0),
  pagedCacheEvict: (c, s) => native.pagedCacheEvict(c, s, 4, 0),
  pagedCacheTrack: (c, s) => native.pagedCacheTrack(c, s),
};
for (const [name, f] of Object.entries(calls)) {
  for (const x of notIds) {
    assertThrows(() => f(77, [x]), 'every id must be', name + ' of [' + text(x) + ']');
    assertThrows(() => f(77, [0, x]), 'every id must be', name + ' of [0, ' + text(x) + ']');
    assertThrows(() => f(x, [0]), 'an id, a whole number', name + ' of the cache ' + text(x));
  }
  for (const x of [NaN, -1, 0.5, 2 ** 32]) assertThrows(() => f(77, new Float64Array([0, x])), 'every id must be', name + ' of doubles, ' + x);
  assertThrows(() => f(77, new Int32Array([0, -1])), 'every id must be', name + ' of integers, -1');
  for (const x of [undefined, null, 3, 'ab', {}, new Float32Array(1), new Uint8Array(1), new BigInt64Array(1)])
    assertThrows(() => f(77, x), 'an array of sequence ids is wanted', name + ' of no list');
  for (const s of [[], [0], new Uint32Array([0, 4]), new Int32Array([3]), new Float64Array([1, 2])])
    assertThrows(() => f(77, s), 'invalid paged cache id: 77', name + ' of a proper list');
}
for (const x of notCounts.concat([undefined, null])) {
  assertThrows(() => native.pagedCacheAppend(77, [0], 0, 0, [x]), 'every length must be', 'a count of ' + text(x));
  assertThrows(() => native.pagedCacheTruncate(77, [0], [x]), 'every length must be', 'a length of ' + text(x));
  assertThrows(() => native.pagedCacheEvict(77, [0], x, 0), 'a whole number is wanted', 'a budget of ' + text(x));
  assertThrows(() => native.pagedCacheCreate(1, 16, 1, x, 1, 8, false, false), 'a whole number is wanted', 'a page of ' + text(x));
}
for (const x of notCounts) assertThrows(() => native.pagedCacheEvict(77, [0], 4, x), 'a whole number is wanted', 'recent tokens of ' + text(x));
for (const x of notIds) {
  for (const name of ['pagedCacheFree', 'pagedCacheFreePages', 'pagedCacheAdd']) assertThrows(() => native[name](x), 'an id, a whole number', name + ' of ' + text(x));
  for (const name of ['pagedCacheFork', 'pagedCacheDrop', 'pagedCacheLen', 'pagedCacheSeen', 'pagedCacheRead']) {
    assertThrows(() => native[name](77, x), 'an id, a whole number', name + ' of the sequence ' + text(x));
    assertThrows(() => native[name](x, 0), 'an id, a whole number', name + ' of the cache ' + text(x));
  }
  assertThrows(() => native.pagedCacheAppend(77, [0], x, 0, null), 'an id, a whole number', 'keys ' + text(x));
  assertThrows(() => native.pagedCacheAppend(77, [0], 0, x, null), 'an id, a whole number', 'values ' + text(x));
  assertThrows(() => native.pagedCacheAttend(77, [0], x, 1, false), 'an id, a whole number', 'queries ' + text(x));
  assertThrows(() => native.qkNormRope(0, x, 0, 0, null, 0, 8, false, 1e4, 1e-6), 'an id, a whole number', 'rotated keys ' + text(x));
  if (x != null) assertThrows(() => native.qkNormRope(0, 0, 0, 0, x, 0, 8, false, 1e4, 1e-6), 'an id, a whole number', 'positions ' + text(x));
}
for (const x of notCounts) assertThrows(() => native.qkNormRope(0, 0, 0, 0, null, x, 8, false, 1e4, 1e-6), 'a whole number is wanted', 'an offset of ' + text(x));
for (const x of ['x', undefined, null, {}]) {
  assertThrows(() => native.qkNormRope(0, 0, 0, 0, null, 0, x, false, 1e4, 1e-6), 'a whole number is wanted', 'rotary dims ' + text(x));
  assertThrows(() => native.qkNormRope(0, 0, 0, 0, null, 0, 8, false, x, 1e-6), 'theta must be a number', 'theta ' + text(x));
  assertThrows(() => native.qkNormRope(0, 0, 0, 0, null, 0, 8, false, 1e4, x), 'eps must be a number', 'eps ' + text(x));
  assertThrows(() => native.pagedCacheAttend(77, [0], 0, x, false), 'the scale must be a number', 'scale ' + text(x));
}
native.pagedCacheFree(77);  // an id of no cache: nothing to do
console.log(passed + ' passed, ' + failed + ' failed');
process.exit(failed ? 1 : 0);
