// The verification dispatches through the addon without a device: descriptors are checked before the context is looked at.
'use strict'
const assert = require('assert')
const path = require('path')
const z = require(path.join(__dirname, '..', '..', 'zero-tvm_amd', 'js', 'index.js'))
const addon = require(path.join(__dirname, '..', '..', 'zero-tvm_amd', 'js', 'ztvm_napi.node'))
const cache = { format: z.KV.F16, kv_heads: 2, head_dim: 64, page_size: 16, head_page_stride: 1024, v_page_offset: 2048, kv_page_stride: 4096,
  pages_capacity: 16384n, pages: 0x10000n }
const with_ = (a, b) => Object.assign({}, a, b)
const says = (fn, desc, pattern) => assert.throws(() => addon[fn](null, desc), pattern)
const rope = { tokens: 3, heads: 4, rotary_dim: 64, qkv_stride: 512, q_stride: 256, attn_factor: 1, qkv: 0x100000n, q_out: 0x200000n,
  frequencies: 0x3000n, positions: 0x4000n, slots: 0x5000n, cache }
says('ropeAppend', rope, /null context/)
says('ropeAppend', with_(rope, { rotary_dim: 63 }), /rotary_dim/)
says('ropeAppend', with_(rope, { cache: with_(cache, { pages_capacity: 0n }) }), /capacities/)
says('ropeAppend', with_(rope, { heads: 'four' }), /must be a number/)
const read = { tokens: 1, out_stride: 128, k_out: 0x1000n, slots: 0x2000n, cache }
says('kvRead', read, /null context/)
says('kvRead', with_(read, { out_stride: 5 }), /out_stride/)
const attention = { tokens: 5, sequences: 2, heads: 4, max_query: 3, max_kv: 100, q_stride: 256, out_stride: 256, page_table_stride: 7,
  mask_words: 1, scale: 0.125, q: 0x100000n, out: 0x200000n, query_start: 0x4000n, kv_length: 0x5000n, page_table: 0x6000n, tree_mask: 0x7000n, cache }
says('attention', attention, /null context/)
says('attention', with_(attention, { scale: NaN }), /scale/)
says('attention', with_(attention, { max_kv: 1000 }), /page_table_stride/)
const score = { rows: 1, vocab: 10, row_stride: 10, inv_temperature: 1, logits: 0x1000n, top_k: 3, top_ids: 0x2000n }
says('tokenLogprobs', score, /null context/)
says('tokenLogprobs', with_(score, { top_k: 11 }), /top_k/)
const f = z.ropeFrequencies(z.ROPE.YARN, 64, 10000, { factor: 4, original: 4096, low: 1, high: 32 })
assert.strictEqual(f.table.length, 32)
assert.strictEqual(f.table[0], 1)
assert.ok(Math.abs(f.attnFactor - (0.1 * Math.log(4) + 1)) < 1e-6)
assert.ok(Math.abs(f.table[31] - Math.pow(10000, -62 / 64) / 4) < 1e-12)
assert.throws(() => z.ropeFrequencies(z.ROPE.LINEAR, 64, 10000, { factor: 0.5 }), /factor/)
console.log('js verify cpu checks ok')
