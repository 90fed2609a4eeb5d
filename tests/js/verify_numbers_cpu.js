// Counts in the descriptors of the verification dispatches are whole numbers of 32 bits; anything else is refused, not cut.
'use strict'
const assert = require('assert')
const path = require('path')
const addon = require(path.join(__dirname, '..', '..', 'zero-tvm_amd', 'js', 'ztvm_napi.node'))
const cache = { format: 0, kv_heads: 2, head_dim: 64, page_size: 16, head_page_stride: 1024, v_page_offset: 2048, kv_page_stride: 4096,
  pages_capacity: 16384n, pages: 0x10000n }
const read = { tokens: 1, out_stride: 128, k_out: 0x1000n, slots: 0x2000n, cache }
const call = (change) => () => addon.kvRead(null, Object.assign({}, read, change))
for (const fine of [0, 1, 7]) assert.throws(call({ tokens: fine }), /null context/)
assert.throws(call({ out_stride: 4294967295 }), /null context/)
for (const bad of [-1, 4294967296, 4294967297, 1.5, NaN, Infinity, -Infinity]) {
  assert.throws(call({ tokens: bad }), /'tokens' must be a whole number/)
  assert.throws(call({ cache: Object.assign({}, cache, { page_size: bad }) }), /'page_size' must be a whole number/)
}
for (const bad of ['1', true, null, {}]) assert.throws(call({ tokens: bad }), /'tokens' must be a number/)
for (const fine of [0x4000n, 0x4000]) assert.throws(call({ k_out: fine }), /null context/)
for (const bad of [-1n, -2n, 1n << 64n, -2, 1.5, NaN, Infinity, 2 ** 53]) {
  assert.throws(call({ k_out: bad }), /'k_out' must be an address/)
  assert.throws(call({ cache: Object.assign({}, cache, { pages_capacity: bad }) }), /'pages_capacity' must be an address or a count/)
}
console.log('js verify number checks ok')
