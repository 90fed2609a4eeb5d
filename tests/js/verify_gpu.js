// The verification dispatches through the JS host: inputs and outputs as files, checked by the Python test.
'use strict'
const fs = require('fs')
const path = require('path')
const z = require(path.join(__dirname, '..', '..', 'zero-tvm_amd', 'js', 'index.js'))
const dir = process.argv[2]
const meta = JSON.parse(fs.readFileSync(path.join(dir, 'meta.json'), 'utf8'))
const dev = new z.Device(0)
const put = (name) => {
  const data = fs.readFileSync(path.join(dir, name))
  const b = dev.createBuffer(data.length, name)
  dev.writeBuffer(b, 0, data)
  return b
}
const get = (b, name) => fs.writeFileSync(path.join(dir, name), Buffer.from(dev.readBuffer(b)))
const { tokens, heads, kvHeads, headDim, pageSize, vocab, k, sequences, maxQuery, maxKv, tableStride } = meta
const f = z.ropeFrequencies(z.ROPE.PLAIN, headDim, 10000)
const table = dev.createBuffer(f.table.byteLength, 'frequencies')
dev.writeBuffer(table, 0, f.table)
const pages = put('pages.bin'), scales = put('scales.bin')
const cache = dev.kvCache({ format: z.KV.INT8, kvHeads, headDim, pageSize, pages, scales })
const qkv = put('qkv.bin'), slots = put('slots.bin')
const width = (heads + 2 * kvHeads) * headDim
dev.ropeAppend({ tokens, heads, rotary_dim: headDim, qkv_stride: width, q_stride: width, attn_factor: f.attnFactor, qkv, q_out: qkv,
  frequencies: table, positions: put('positions.bin'), slots, cache })
get(qkv, 'q_out.bin')
const ko = dev.createBuffer(tokens * kvHeads * headDim * 2, 'k'), vo = dev.createBuffer(tokens * kvHeads * headDim * 2, 'v')
dev.kvRead({ tokens, out_stride: kvHeads * headDim, k_out: ko, v_out: vo, slots, cache })
get(ko, 'k_out.bin')
get(vo, 'v_out.bin')
get(pages, 'pages_out.bin')
get(scales, 'scales_out.bin')
const out = dev.createBuffer(tokens * heads * headDim * 2, 'attn'), lse = dev.createBuffer(tokens * heads * 4, 'lse')
dev.attention({ tokens, sequences, heads, max_query: maxQuery, max_kv: maxKv, q_stride: width, out_stride: heads * headDim,
  page_table_stride: tableStride, mask_words: 1, scale: 1 / Math.sqrt(headDim), q: qkv, out, lse, query_start: put('starts.bin'),
  kv_length: put('lengths.bin'), page_table: put('table.bin'), tree_mask: put('masks.bin'), cache })
get(out, 'attn.bin')
get(lse, 'lse.bin')
const lp = dev.createBuffer(tokens * 4, 'lp'), ids = dev.createBuffer(tokens * k * 4, 'ids')
dev.tokenLogprobs({ rows: tokens, vocab, row_stride: vocab, top_k: k, inv_temperature: 1, logits: put('logits.bin'), tokens: put('drafted.bin'),
  logprob: lp, top_ids: ids })
get(lp, 'lp.bin')
get(ids, 'ids.bin')
dev.close()
console.log('js verify gpu ok')
