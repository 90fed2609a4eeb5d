"""A whole verification step as a serving program runs it: the QKV matmul of the drafted rows, the rotary append, attention
over the tree, the LM head, the scores of the drafted tokens; eager and recorded, f16 and int8 cache."""
import numpy as np
import pytest

from . import verify_ref as ref
from .test_rope_append_gpu import f16_layout, int8_layout
from .util import Dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
def test_verify_step(ctx, capi, synth, oracle, int8):
    heads, kv_heads, dim, page, vocab, k = 8, 2, 64, 16, 1024, 5
    d_model, rows = heads * dim, (heads + 2 * kv_heads) * dim
    queries, history = [7, 1, 4], [40, 3, 0]
    tokens = sum(queries)
    rng = np.random.default_rng(11)
    starts = np.concatenate([[0], np.cumsum(queries)])
    lengths = [n + h for n, h in zip(queries, history)]
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 1
    order, table, at = rng.permutation(pages), np.full((3, max(need)), -1, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    masks, positions, slots = [], [], []
    for b, n in enumerate(queries):
        mine, depth = [], []
        for i in range(n):
            up = int(rng.integers(max(0, i - 3), i)) if i else -1
            mine.append((mine[up] if up >= 0 else 0) | 1 << i)
            depth.append(depth[up] + 1 if up >= 0 else 0)
            where = history[b] + i
            slots.append(table[b, where // page] * page + where % page)
        masks += mine
        positions += [history[b] + x for x in depth]
    x = synth.activations(tokens, d_model)
    wq, sq = synth.packed_weights(rows, d_model), synth.scales(rows, d_model)
    bq = synth.biases(rows, d_model, sq)
    wl, sl = synth.packed_weights(vocab, d_model, salt=3), synth.scales(vocab, d_model, salt=3)
    bl = synth.biases(vocab, d_model, sl, salt=3)
    freq, factor = capi.rope_frequencies(capi.ROPE_YARN, dim, 10000.0, 4.0, 4096.0, 1.0, 32.0)
    drafted = rng.integers(0, vocab, tokens)
    cache0 = ref.int8_cache(rng, pages, kv_heads, page, dim) if int8 else ref.f16_cache(rng, pages, kv_heads, page, dim)
    scale = float(np.float32(dim ** -0.5))
    with Dev(ctx) as d:
        i32 = lambda a: d.put(np.asarray(a, np.int32))  # noqa: E731
        qkv, attn, logits = d.empty(tokens * rows * 2), d.empty(tokens * d_model * 2), d.empty(tokens * vocab * 4)
        lp, ent, ids, best = d.empty(tokens * 4), d.empty(tokens * 4), d.empty(tokens * k * 4), d.empty(tokens * k * 4)
        if int8:
            pg, sc = d.put(cache0[0]), d.put(cache0[1])
            cache = int8_layout(capi, kv_heads, dim, page, pages=pg, pages_capacity=cache0[0].size // 4, scales=sc, scales_capacity=cache0[1].size)
        else:
            pg = d.put(cache0)
            cache = f16_layout(capi, kv_heads, dim, page, pages=pg, pages_capacity=cache0.size)
        mm = capi.MatmulDesc(bits=4, affine=1, M=tokens, N=rows, k_packed=d_model // 8, scales_per_row=d_model // 64, out=qkv, in_=d.put(x),
                             scales=d.put(sq), weights=d.put(wq), biases=d.put(bq))
        rope = capi.RopeAppendDesc(tokens=tokens, heads=heads, rotary_dim=dim, qkv_stride=rows, q_stride=rows, attn_factor=factor, qkv=qkv, q_out=qkv,
                                   frequencies=d.put(freq), positions=i32(positions), slots=i32(slots), cache=cache)
        attend = capi.AttentionDesc(tokens=tokens, sequences=3, heads=heads, max_query=max(queries), max_kv=max(lengths), q_stride=rows,
                                    out_stride=d_model, page_table_stride=table.shape[1], mask_words=1, scale=scale, q=qkv, out=attn,
                                    query_start=i32(starts), kv_length=i32(lengths), page_table=d.put(table),
                                    tree_mask=d.put(np.array(masks, np.uint64)), cache=cache)
        head = capi.MatmulDesc(bits=4, affine=1, out_f32=1, M=tokens, N=vocab, k_packed=d_model // 8, scales_per_row=d_model // 64, out=logits,
                               in_=attn, scales=d.put(sl), weights=d.put(wl), biases=d.put(bl))
        score = capi.TokenLogprobsDesc(rows=tokens, vocab=vocab, row_stride=vocab, top_k=k, inv_temperature=1.0, logits=logits,
                                       tokens=i32(drafted), logprob=lp, entropy=ent, top_ids=ids, top_logprobs=best)

        def step():
            ctx.matmul(mm)
            ctx.rope_append(rope)
            ctx.attention(attend)
            ctx.matmul(head)
            ctx.token_logprobs(score)

        def read():
            return (ctx.download(qkv, tokens * rows * 2, np.float16).reshape(tokens, rows), ctx.download(attn, tokens * d_model * 2, np.float16),
                    ctx.download(logits, tokens * vocab * 4, np.float32).reshape(tokens, vocab), ctx.download(lp, tokens * 4, np.float32),
                    ctx.download(ent, tokens * 4, np.float32), ctx.download(ids, tokens * k * 4, np.uint32).reshape(tokens, k))

        ctx.matmul(mm)
        raw = ctx.download(qkv, tokens * rows * 2, np.float16).reshape(tokens, -1, dim)
        step()
        eager = read()
        after = ctx.download(pg, cache0[0].nbytes if int8 else cache0.nbytes, np.uint8)
        scales = ctx.download(sc, cache0[1].nbytes, np.float16) if int8 else None
        ctx.record_begin()
        step()
        cb = ctx.record_end()
        try:
            for _ in range(3):
                for p, n in ((attn, tokens * d_model * 2), (logits, tokens * vocab * 4), (lp, tokens * 4), (ids, tokens * k * 4)):
                    ctx.fill(p, 0x3C, n)
                ctx.submit(cb)
                assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(eager, read()))
        finally:
            ctx.cmdbuf_destroy(cb)
    # each stage against the formula on the stage's own inputs
    want, norm = ref.rotated(raw[:, :heads], positions, freq, dim, False, factor)
    q = eager[0].reshape(tokens, -1, dim)[:, :heads]
    assert ref.close_rotated(q, want, norm)
    stored = (after.view(np.int8).reshape(cache0[0].shape), scales.reshape(cache0[1].shape)) if int8 else after.view(np.float16).reshape(cache0.shape)
    rows_now = ref.rows_of(stored)
    kwant, knorm = ref.rotated(raw[:, heads:heads + kv_heads], positions, freq, dim, False, factor)
    for t, s in enumerate(slots):
        got = rows_now[s // page, s % page]
        if int8:      # half a count of the row's scale, and the scale's own rounding on 127 counts
            step_k, step_v = np.abs(kwant[t]).max(-1, keepdims=True) / 127, np.abs(raw[t, heads + kv_heads:].astype(np.float64)).max(-1, keepdims=True) / 127
            assert np.all(np.abs(got[0] - kwant[t]) <= step_k * (0.5 + 127 * ref.HALF) * 1.01)
            assert np.all(np.abs(got[1] - raw[t, heads + kv_heads:]) <= step_v * (0.5 + 127 * ref.HALF) * 1.01)
        else:
            assert ref.close_rotated(got[0], kwant[t], knorm[t]) and np.array_equal(got[1], raw[t, heads + kv_heads:].astype(np.float64))
    w = ref.attention(q, rows_now, page, table, starts, lengths, masks, scale, heads)
    ref.close_attention(eager[1].reshape(tokens, heads, dim), None, *w, dim, max(lengths))
    lref = oracle.gemm(oracle.MODE_FORMULA_F64, 4, True, tokens, vocab, d_model, eager[1].view(np.uint16).reshape(tokens, d_model), wl, sl, bl)
    assert np.max(np.abs(eager[2] - lref) / (np.abs(lref) + 1e-2)) < 1e-2
    logp, entropy, top, _, _, m = ref.logprobs(eager[2], 1.0, drafted, k)
    assert np.array_equal(eager[5], top) and ref.close_logp(eager[3], logp, m, vocab)
