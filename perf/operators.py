"""Cases of the operators that verify drafted tokens over the paged KV cache, and their plain forms.

    rope    rotary positions on the rows of a fused QKV projection, K and V stored in the paged cache (f16 or int8)
    read    rows of the paged cache read back as f16
    attend  attention of drafted tokens (a tree, a chain, or one token) over the paged cache
    score   log probabilities of given tokens, entropy and the best alternatives of rows of logits

`own` chooses between the plain form (elementary torch operations in 32 bits) and the library's entry points.
"""
import importlib
import math

import numpy as np
import torch

own = False

PAGE = 16


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the decode step of one conversation: everything is launch latency
        {"name": "rope f16 one token", "op": "rope", "int8": False, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "far": 4000, "scaling": "none"},
        # a verify step of eight conversations with ragged trees, part of the head rotated, int8 cache
        {"name": "rope int8 verify", "op": "rope", "int8": True, "tokens": 391, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 64, "interleaved": True, "far": 30000, "scaling": "linear"},
        # a long prompt stored chunk by chunk, frequencies stretched for long contexts
        {"name": "rope f16 prompt", "op": "rope", "int8": False, "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "far": 120000, "scaling": "yarn"},
        # the accepted path of a few conversations taken out of an f16 cache
        {"name": "read f16 short", "op": "read", "int8": False, "tokens": 701, "kv_heads": 16, "dim": 96},
        # a prompt's int8 rows handed to another engine as f16
        {"name": "read int8 prompt", "op": "read", "int8": True, "tokens": 16390, "kv_heads": 8, "dim": 128},
        # one conversation, one token, short history: latency
        {"name": "attend one token", "op": "attend", "int8": False, "sequences": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "query": 1, "query_least": 1, "length": 1037, "length_least": 1037, "tree": False},
        # a decode batch of ragged conversations
        {"name": "attend decode batch", "op": "attend", "int8": False, "sequences": 48, "heads": 32, "kv_heads": 8, "dim": 128,
         "query": 1, "query_least": 1, "length": 8191, "length_least": 90, "tree": False},
        # ragged trees of drafted tokens over an int8 cache
        {"name": "attend trees int8", "op": "attend", "int8": True, "sequences": 16, "heads": 32, "kv_heads": 8, "dim": 128,
         "query": 61, "query_least": 5, "length": 4500, "length_least": 200, "tree": True},
        # one tree over one long document, a key/value head for each query head
        {"name": "attend tree long", "op": "attend", "int8": False, "sequences": 1, "heads": 16, "kv_heads": 16, "dim": 96,
         "query": 64, "query_least": 64, "length": 65537, "length_least": 65537, "tree": True},
        # the last token of one conversation, with twenty alternatives
        {"name": "score one row", "op": "score", "half": False, "rows": 1, "vocab": 128000, "top": 20, "masked": False, "pad": 0},
        # f16 logits in padded rows, a part of the vocabulary masked out
        {"name": "score f16 masked", "op": "score", "half": True, "rows": 67, "vocab": 50257, "top": 8, "masked": True, "pad": 47},
        # every drafted token of a verify step over a large vocabulary
        {"name": "score verify", "op": "score", "half": False, "rows": 384, "vocab": 248320, "top": 5, "masked": False, "pad": 0},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rope", "rope", "read", "attend", "attend", "attend", "score", "score"])
    dim = rng.choice([64, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    int8 = rng.random() < 0.5
    if op == "rope":
        heads = kv_heads * rng.choice([1, 2, 4, 7])
        most = 8192 * 48 * 128 // ((heads + 2 * kv_heads) * dim)
        return {"op": op, "int8": int8, "tokens": _spread(rng, 1, min(8192, most)), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2, 32]), "interleaved": rng.random() < 0.5, "far": _spread(rng, 16, 131072),
                "scaling": rng.choice(["none", "linear", "yarn"])}
    if op == "read":
        most = 16390 * 8 * 128 // (kv_heads * dim)
        return {"op": op, "int8": int8, "tokens": _spread(rng, 1, min(16390, most)), "kv_heads": kv_heads, "dim": dim}
    if op == "attend":
        heads = kv_heads * rng.choice([1, 2, 4, 7])
        tree = rng.random() < 0.6
        query = _spread(rng, 2, 64) if tree else 1
        sequences = _spread(rng, 1, 48)
        # bounded by the keys of the largest listed case, and by the products of queries and keys
        keys = min(65537, 48 * 4000 * 8 * 128 // (kv_heads * dim) // sequences)
        keys = min(keys, 65537 * 64 * 16 * 96 // (heads * query * dim) // sequences, 65537 * 64 * 16 // (heads * query) // sequences)
        length = _spread(rng, query, max(query, keys))
        return {"op": op, "int8": int8, "sequences": sequences, "heads": heads, "kv_heads": kv_heads, "dim": dim, "query": query,
                "query_least": rng.choice([query, 1]), "length": length, "length_least": rng.choice([length, query]), "tree": tree}
    vocab = _spread(rng, 100, 248320)
    return {"op": op, "half": rng.random() < 0.4, "rows": _spread(rng, 1, max(1, min(2048, 384 * 248320 // vocab))), "vocab": vocab,
            "top": _spread(rng, 1, 40), "masked": rng.random() < 0.4, "pad": rng.choice([0, 0, 8, 13])}


# --------------------------------------------------------------------------------------- shapes of a case

def _ragged(least, most, count):
    """`count` numbers from least to most, mixed, the same for everybody."""
    return [most - (most - least) * ((37 * b) % count) // max(count - 1, 1) for b in range(count)]


def _shape(case):
    """Query tokens and cached keys of each sequence of an attention case."""
    lengths = _ragged(case["length_least"], case["length"], case["sequences"])
    queries = _ragged(case["query_least"], case["query"], case["sequences"])[::-1]
    return [min(q, n) for q, n in zip(queries, lengths)], lengths


def work(case):
    op = case["op"]
    if op == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["half"] else 4) + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * n}
    d, hk = case["dim"], case["kv_heads"]
    row = 2 * hk * (d + 2 if case["int8"] else 2 * d)  # K and V of one slot in the cache
    if op == "rope":
        t, h = case["tokens"], case["heads"]
        size = t * (h + 2 * hk) * d * 2 + t * h * d * 2 + t * row + t * 8
        if case["int8"]:  # and read back
            size += t * row + t * 2 * hk * d * 2
        return {"bytes": size, "flops": 3 * t * (h + hk) * case["rotary"]}
    if op == "read":
        return {"bytes": case["tokens"] * (row + 2 * hk * d * 2 + 4), "flops": case["tokens"] * 2 * hk * d}
    queries, lengths = _shape(case)
    h = case["heads"]
    return {"bytes": sum(lengths) * row + sum(queries) * (2 * h * d * 2 + 4 * h),
            "flops": 4 * d * h * sum(q * n for q, n in zip(queries, lengths))}


# ------------------------------------------------------------------------------------------------ inputs

def _frequencies(rotary, scaling, far):
    """Radians per position of each rotated pair, in 64 bits."""
    j = np.arange(rotary // 2, dtype=np.float64)
    theta = 500000.0
    f = theta ** (-2.0 * j / rotary)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "yarn":
        factor, original = 16.0, 8192.0
        at = lambda turns: rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rotary - 1)
        ramp = np.clip((j - low) / max(high - low, 1e-3), 0.0, 1.0)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _cache(case, slots, g):
    """A paged cache with what earlier steps left in it. f16: [page][K, V][head][slot][dim]; int8: [page][head][slot][K, V][dim]."""
    pages, hk, d = -(-slots // PAGE), case["kv_heads"], case["dim"]
    if not case["int8"]:
        return {"pages": torch.randn(pages, 2, hk, PAGE, d, generator=g, device="cuda", dtype=torch.float16), "scales": None}
    q = torch.randn(pages, hk, PAGE, 2, d, generator=g, device="cuda", dtype=torch.float16).mul_(40).round_().clamp_(-127, 127)
    s = torch.rand(pages, hk, PAGE, 2, generator=g, device="cuda").mul_(0.01).add_(0.02).to(torch.float16)
    return {"pages": q.to(torch.int8), "scales": s}


def _tree(queries, rng):
    """A word for each drafted token: bit j is set where token j of its sequence is an ancestor of it or itself."""
    words = []
    for n in queries:
        mine = []
        for i in range(n):
            up = int(rng.integers(max(0, i - 6), i)) if i else -1
            mine.append((mine[up] if up >= 0 else 0) | 1 << i)
        if n > 2:
            mine[n - 1] = 0  # a place of the tree's template that this sequence does not use
        words += mine
    return np.array(words, np.uint64).view(np.int64)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    op = case["op"]
    s = {"case": case}
    i32 = lambda a: torch.as_tensor(np.asarray(a, np.int32)).cuda()  # noqa: E731
    if op == "score":
        rows, vocab, kind = case["rows"], case["vocab"], torch.float16 if case["half"] else torch.float32
        x = torch.randn(rows, vocab + case["pad"], generator=g, device="cuda").mul_(3.0)
        if case["masked"]:
            hide = torch.rand(rows, vocab + case["pad"], generator=g, device="cuda") < 0.3
            hide[:, min(5, vocab - 1)] = False
            x.masked_fill_(hide, -math.inf)
        s["logits"] = x.to(kind)[:, :vocab]
        tokens = rng.integers(0, vocab, rows)
        s["tokens"] = i32(tokens)
        s["scale"] = 1.0 / 0.7 if case["masked"] else 1.0
        s["out"] = (torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"),
                    torch.zeros(rows, case["top"], device="cuda", dtype=torch.int32), torch.zeros(rows, case["top"], device="cuda"))
    elif op == "attend":
        queries, lengths = _shape(case)
        b, t, h, d = case["sequences"], sum(queries), case["heads"], case["dim"]
        need = [-(-n // PAGE) for n in lengths]
        order = rng.permutation(sum(need) + 3)
        table = np.full((b, max(need)), -1, np.int32)
        at = 0
        for k, n in enumerate(need):
            table[k, :n] = order[at:at + n]
            at += n
        s.update(_cache(case, (sum(need) + 3) * PAGE, g))
        s["q"] = torch.randn(t, h * d, generator=g, device="cuda").mul_(2.0).to(torch.float16)
        s["out"] = torch.zeros(t, h * d, device="cuda", dtype=torch.float16)
        s["lse"] = torch.zeros(t, h, device="cuda")
        s["start"], s["length"] = i32(np.concatenate([[0], np.cumsum(queries)])), i32(lengths)
        s["table"] = torch.from_numpy(table).cuda()
        s["mask"] = torch.from_numpy(_tree(queries, rng)).cuda() if case["tree"] else None
        s["queries"], s["lengths"] = queries, lengths
    else:
        t, hk, d = case["tokens"], case["kv_heads"], case["dim"]
        slots = t + 64
        s.update(_cache(case, slots, g))
        where = rng.permutation(slots)[:t]
        if t > 4:
            where[t - 2] = -1  # a padded token
        s["slots"] = i32(where)
        s["k"] = torch.zeros(t, hk * d, device="cuda", dtype=torch.float16)
        s["v"] = torch.zeros(t, hk * d, device="cuda", dtype=torch.float16)
        if op == "rope":
            h = case["heads"]
            s["qkv"] = torch.randn(t, (h + 2 * hk) * d, generator=g, device="cuda").to(torch.float16)
            f, s["factor"] = _frequencies(case["rotary"], case["scaling"], case["far"])
            s["frequencies"] = torch.from_numpy(f).cuda()
            s["positions"] = i32(rng.integers(0, case["far"], t))
            s["q"] = torch.zeros(t, h * d, device="cuda", dtype=torch.float16)
    if own:
        _bind(s)
    return s


# ------------------------------------------------------------------------------------- the library's calls

_context = None


def _bind(s):
    """The library's context and the descriptors that a serving program keeps beside its buffers."""
    global _context
    capi = importlib.import_module("zero-tvm_amd").capi
    if _context is None:
        _context = capi.Context(torch.cuda.current_device())
    case, at = s["case"], lambda x: 0 if x is None else x.data_ptr()  # noqa: E731
    if case["op"] == "score":
        logprob, entropy, ids, best = s["out"]
        s["desc"] = capi.TokenLogprobsDesc(rows=case["rows"], vocab=case["vocab"], row_stride=s["logits"].stride(0),
                                           logits_f16=int(case["half"]), top_k=case["top"], inv_temperature=s["scale"],
                                           logits=at(s["logits"]), tokens=at(s["tokens"]), logprob=at(logprob), entropy=at(entropy),
                                           top_ids=at(ids), top_logprobs=at(best))
        return
    hk, d, pages = case["kv_heads"], case["dim"], s["pages"]
    if case["int8"]:
        cache = capi.KvCache(format=capi.KV_INT8, kv_heads=hk, head_dim=d, page_size=PAGE, pages_capacity=pages.numel() // 4,
                             scales_capacity=s["scales"].numel(), pages=at(pages), scales=at(s["scales"]))
    else:
        cache = capi.KvCache(format=capi.KV_F16, kv_heads=hk, head_dim=d, page_size=PAGE, head_page_stride=PAGE * d,
                             v_page_offset=hk * PAGE * d, kv_page_stride=2 * hk * PAGE * d, pages_capacity=pages.numel(), pages=at(pages))
    if case["op"] == "attend":
        s["desc"] = capi.AttentionDesc(tokens=s["q"].shape[0], sequences=case["sequences"], heads=case["heads"],
                                       max_query=max(s["queries"]), max_kv=max(s["lengths"]), q_stride=s["q"].shape[1],
                                       out_stride=s["q"].shape[1], page_table_stride=s["table"].shape[1],
                                       mask_words=1 if case["tree"] else 0, scale=1.0 / math.sqrt(d), q=at(s["q"]), out=at(s["out"]),
                                       lse=at(s["lse"]), query_start=at(s["start"]), kv_length=at(s["length"]),
                                       page_table=at(s["table"]), tree_mask=at(s["mask"]), cache=cache)
        return
    s["read"] = capi.KvReadDesc(tokens=case["tokens"], out_stride=hk * d, k_out=at(s["k"]), v_out=at(s["v"]), slots=at(s["slots"]),
                                cache=cache)
    if case["op"] == "rope":
        s["desc"] = capi.RopeAppendDesc(tokens=case["tokens"], heads=case["heads"], rotary_dim=case["rotary"],
                                        interleaved=int(case["interleaved"]), qkv_stride=s["qkv"].shape[1], q_stride=s["q"].shape[1],
                                        attn_factor=s["factor"], qkv=at(s["qkv"]), q_out=at(s["q"]), frequencies=at(s["frequencies"]),
                                        positions=at(s["positions"]), slots=at(s["slots"]), cache=cache)


def _own(s):
    op = s["case"]["op"]
    if op == "score":
        _context.token_logprobs(s["desc"])
        return s["out"]
    if op == "attend":
        _context.attention(s["desc"])
        return s["out"], s["lse"]
    if op == "read":
        _context.kv_read(s["read"])
        return s["k"], s["v"]
    _context.rope_append(s["desc"])
    if s["case"]["int8"]:
        _context.kv_read(s["read"])
        return s["q"], s["k"], s["v"]
    return s["q"], s["pages"]


# ------------------------------------------------------------------------------------------- plain forms

def _rotate(x, cos, sin, rotary, interleaved):
    """x [tokens, heads, dim] in 32 bits; cos and sin [tokens, 1, rotary / 2]."""
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y[..., 0:rotary:2], y[..., 1:rotary:2] = a * cos - b * sin, b * cos + a * sin
    else:
        half = rotary // 2
        a, b = x[..., :half], x[..., half:rotary]
        y[..., :half], y[..., half:rotary] = a * cos - b * sin, b * cos + a * sin
    return y


def _quantized(x):
    """int8 counts and the f16 scale of each row; x is what an f16 row holds."""
    scale = (x.abs().amax(-1, keepdim=True) / 127.0).clamp_min(1e-8)
    return torch.round(x / scale).clamp(-127, 127).to(torch.int8), scale[..., 0].to(torch.float16)


def _plain_rope(s):
    case = s["case"]
    t, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    angle = s["positions"].double()[:, None, None] * s["frequencies"]
    cos, sin = (torch.cos(angle) * s["factor"]).float(), (torch.sin(angle) * s["factor"]).float()
    x = s["qkv"].view(t, h + 2 * hk, d).float()
    turned = _rotate(x[:, :h + hk], cos, sin, case["rotary"], case["interleaved"])
    q = turned[:, :h].to(torch.float16).view(t, h * d)
    k, v = turned[:, h:].to(torch.float16), x[:, h + hk:].to(torch.float16)
    slots = s["slots"].long()
    kept = torch.nonzero(slots >= 0)[:, 0]
    page, slot = slots[kept] // PAGE, slots[kept] % PAGE
    if case["int8"]:
        s["pages"][page, :, slot, 0], s["scales"][page, :, slot, 0] = _quantized(k[kept].float())
        s["pages"][page, :, slot, 1], s["scales"][page, :, slot, 1] = _quantized(v[kept].float())
        return (q,) + _plain_read(s)
    s["pages"][page, 0, :, slot] = k[kept]
    s["pages"][page, 1, :, slot] = v[kept]
    return q, s["pages"]


def _plain_read(s):
    case = s["case"]
    slots = s["slots"].long()
    kept = (slots >= 0)[:, None, None]
    page, slot = slots.clamp_min(0) // PAGE, slots.clamp_min(0) % PAGE
    if case["int8"]:
        rows = s["pages"][page, :, slot].float() * s["scales"][page, :, slot].float()[..., None]  # [tokens, head, K|V, dim]
        k, v = rows[:, :, 0], rows[:, :, 1]
    else:
        k, v = s["pages"][page, 0, :, slot].float(), s["pages"][page, 1, :, slot].float()
    zero = torch.zeros((), device="cuda")
    return tuple(torch.where(kept, y, zero).to(torch.float16).reshape(case["tokens"], -1) for y in (k, v))


def _plain_attend(s):
    case = s["case"]
    b, h, hk, d = case["sequences"], case["heads"], case["kv_heads"], case["dim"]
    most, keys = max(s["queries"]), s["table"].shape[1] * PAGE
    page = s["table"].long().clamp_min(0)
    if case["int8"]:
        rows = s["pages"][page].float() * s["scales"][page].float()[..., None]           # [b, page, head, slot, K|V, dim]
        k, v = (rows[..., i, :].transpose(1, 2).reshape(b, hk, keys, d) for i in (0, 1))
    else:
        k, v = (s["pages"][:, i][page].float().transpose(1, 2).reshape(b, hk, keys, d) for i in (0, 1))
    start, length = s["start"].long(), s["length"].long()
    count = start[1:] - start[:-1]
    i, j = torch.arange(most, device="cuda"), torch.arange(keys, device="cuda")
    token = (start[:-1, None] + i).clamp_max(s["q"].shape[0] - 1)                        # [b, query]
    q = s["q"].view(-1, hk, h // hk, d)[token].float()                                   # [b, query, kv head, group, dim]
    q = q.permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    first = (length - count)[:, None, None]                                              # keys before the drafted tokens
    if s["mask"] is None:
        seen = j <= first + i[:, None]
    else:
        bit = s["mask"][token][:, :, None] >> (j - first).clamp(0, 63)
        seen = (j < first) | (bit & 1).bool()
    seen = seen & (j < length[:, None, None])                                            # [b, query, key]
    score = torch.matmul(q, k.transpose(-1, -2)).view(b, hk, h // hk, most, keys) * (1.0 / math.sqrt(d))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.clamp_min(-1e30))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, hk, -1, keys), v).view(b, hk, h // hk, most, d) / total.clamp_min(1e-30)
    lse = (top + torch.log(total))[..., 0]
    there = torch.nonzero((i < count[:, None]).reshape(-1))[:, 0]                        # the tokens that there are, in order
    out = out.permute(0, 3, 1, 2, 4).reshape(b * most, h * d)[there]
    lse = lse.permute(0, 3, 1, 2).reshape(b * most, h)[there]
    return out.to(torch.float16), lse


def _plain_score(s):
    x = s["logits"].float() * s["scale"]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    p = e / total
    logp = x - lse
    entropy = -torch.where(p > 0, p * logp, torch.zeros((), device="cuda")).sum(-1)
    order = torch.sort(s["logits"], dim=-1, descending=True, stable=True)[1][:, :s["case"]["top"]]
    token = s["tokens"].long()[:, None]
    return torch.gather(logp, 1, token)[:, 0], entropy, order.to(torch.int32), torch.gather(logp, 1, order)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"rope": _plain_rope, "read": _plain_read, "attend": _plain_attend, "score": _plain_score}[op](state)


# ---------------------------------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "read": _exact_read, "attend": _exact_attend, "score": _exact_score}[case["op"]](s)


def _exact_int8(row):
    """Rows of f16 values in 64 bits -> what their int8 form stands for, as f16 values."""
    scale = torch.maximum(row.abs().max(-1, keepdim=True)[0] / 127, torch.tensor(1e-8, dtype=torch.float64, device="cuda"))
    return (torch.clamp(torch.round(row / scale), -127, 127) * scale.half().double()).half().double()


def _exact_rope(s):
    case = s["case"]
    t, h, hk, d, r = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rotary"]
    f, factor = _frequencies(r, case["scaling"], case["far"])
    turn = torch.polar(torch.tensor(factor, dtype=torch.float64, device="cuda").expand(t, r // 2).contiguous(),
                       s["positions"].double()[:, None] * torch.from_numpy(f).cuda())[:, None]
    x = s["qkv"].double().view(t, h + 2 * hk, d)
    part = x[:, :h + hk, :r]
    pairs = torch.stack([part[..., 0::2], part[..., 1::2]] if case["interleaved"] else [part[..., :r // 2], part[..., r // 2:]], -1)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    part = z.flatten(-2) if case["interleaved"] else torch.cat([z[..., 0], z[..., 1]], -1)
    y = torch.cat([part, x[:, :h + hk, r:]], -1)
    q, k, v = y[:, :h].reshape(t, h * d), y[:, h:], x[:, h + hk:]
    where = s["slots"].tolist()
    if case["int8"]:
        k, v = (_exact_int8(z.half().double()).reshape(t, hk * d) for z in (k, v))
        for i in (i for i, w in enumerate(where) if w < 0):
            k[i], v[i] = 0, 0
        return q, k, v
    pages = s["pages"].double().permute(0, 3, 1, 2, 4).reshape(-1, 2, hk, d)  # [slot][K|V][head][dim]
    keep = [i for i, w in enumerate(where) if w >= 0]
    pages[torch.tensor([where[i] for i in keep]).cuda()] = torch.stack([k, v], 1)[torch.tensor(keep).cuda()]
    return q, pages.view(-1, PAGE, 2, hk, d).permute(0, 2, 3, 1, 4).contiguous()


def _exact_rows(s):
    """Every slot of the cache: [slot][K|V][head][dim] in 64 bits, page by page in memory's order."""
    if s["scales"] is None:
        return s["pages"].permute(0, 3, 1, 2, 4).flatten(0, 1).double()
    return (s["pages"].double() * s["scales"].double().unsqueeze(-1)).permute(0, 2, 3, 1, 4).flatten(0, 1)


def _exact_read(s):
    rows = _exact_rows(s)
    rows = torch.cat([rows, torch.zeros_like(rows[:1])])[s["slots"].long()]  # slot -1 is the row of zeros
    return rows[:, 0].flatten(1), rows[:, 1].flatten(1)


def _exact_attend(s):
    case = s["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    table, outs, lses, at = s["table"].cpu().numpy(), [], [], 0
    words = None if s["mask"] is None else s["mask"].cpu().numpy().view(np.uint64)
    for b, (n, length) in enumerate(zip(s["queries"], s["lengths"])):
        ids = torch.from_numpy(table[b, :-(-length // PAGE)].astype(np.int64)).cuda()
        part = {"pages": s["pages"][ids], "scales": None if s["scales"] is None else s["scales"][ids]}
        rows = _exact_rows(part)[:length]
        q = s["q"][at:at + n].double().view(n, h, d)
        can = np.tri(n, dtype=bool) if words is None else np.array([[bool(int(w) >> j & 1) for j in range(n)] for w in words[at:at + n]])
        shut = torch.zeros(n, length, dtype=torch.float64, device="cuda")
        shut[:, length - n:][torch.from_numpy(~can).cuda()] = -math.inf
        for head in range(h):
            x = q[:, head] @ rows[:, 0, head * hk // h].T / math.sqrt(d) + shut
            lse = torch.logsumexp(x, -1)
            outs.append(torch.exp(x - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[:, None]) @ rows[:, 1, head * hk // h])
            lses.append(lse)
        outs[-h:], lses[-h:] = [torch.stack(outs[-h:], 1).view(n, h * d)], [torch.stack(lses[-h:], 1)]
        at += n
    return torch.cat(outs), torch.cat(lses)


def _exact_score(s):
    got = [[], [], []]
    for row, token in zip(s["logits"], s["tokens"].tolist()):
        logp = torch.log_softmax(row.double() * s["scale"], 0)
        got[0].append(logp[token])
        got[1].append(torch.special.entr(torch.exp(logp)).sum())
        got[2].append(torch.topk(logp, s["case"]["top"])[0])
    return torch.stack(got[0]), torch.stack(got[1]), None, torch.stack(got[2])
