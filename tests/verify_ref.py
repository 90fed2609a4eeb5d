"""Plain float64 references of the verification dispatches (rotary append, cache read-back, attention over the paged
cache, token log probabilities), and the bounds that a kernel's rounding stays inside."""
import numpy as np

HALF = 2.0 ** -11          # a rounding to f16, relative
TINY = 2.0 ** -24          # the smallest f16 step; a rounding below the normal range is off by half of it


def rotated(x, positions, freq, rotary, interleaved, factor):
    """x [tokens, heads, dim] -> rotated, and the norm of the pair each element belongs to."""
    x = np.asarray(x, np.float64)
    a = np.asarray(positions, np.float64)[:, None, None] * np.asarray(freq, np.float64)
    c, s = np.cos(a) * factor, np.sin(a) * factor
    y, norm = x.copy(), np.zeros_like(x)
    i = (np.arange(0, rotary, 2), np.arange(1, rotary, 2)) if interleaved else (np.arange(rotary // 2), np.arange(rotary // 2, rotary))
    u, v = x[..., i[0]], x[..., i[1]]
    y[..., i[0]], y[..., i[1]] = u * c - v * s, v * c + u * s
    norm[..., i[0]] = norm[..., i[1]] = np.hypot(u, v) * factor
    return y, norm


def close_rotated(got, want, norm):
    """The angle is off by 2^-25 turns (2e-7 rad), cos and sin by two steps (2.4e-7), the factor and the two products and
    their sum by 2^-24 each: under 1e-6 of the pair's norm together; then one rounding to f16."""
    got = np.asarray(got, np.float64)
    return np.all(np.abs(got - want) <= HALF * np.abs(want) + TINY / 2 + 1.1e-6 * norm)


def f16_cache(rng, pages, kv_heads, page, dim, fill=None):
    """[page][K, V][head][slot][dim] as f16."""
    a = rng.standard_normal((pages, 2, kv_heads, page, dim)).astype(np.float16)
    if fill is not None:
        a[...] = fill
    return a


def int8_cache(rng, pages, kv_heads, page, dim):
    """counts [page][head][slot][K, V][dim] and scales [page][head][slot][K, V]."""
    q = np.clip(np.round(rng.standard_normal((pages, kv_heads, page, 2, dim)) * 40), -127, 127).astype(np.int8)
    s = (rng.random((pages, kv_heads, page, 2)) * 0.01 + 0.02).astype(np.float16)
    return q, s


def rows_of(cache):
    """Any cache as float64 values [page][slot][K, V][head][dim]."""
    if isinstance(cache, tuple):
        return (cache[0].astype(np.float64) * cache[1].astype(np.float64)[..., None]).transpose(0, 2, 3, 1, 4)
    return cache.astype(np.float64).transpose(0, 3, 1, 2, 4)


def attention(q, rows, page, table, starts, lengths, masks, scale, heads):
    """q [tokens, heads, dim]; rows as rows_of; masks: a list of python integers per token, or None (a chain). Returns
    out, lse and, for the bounds, sum p|v|, the largest score error per unit of 2^-24 and the count of visible keys."""
    tokens, _, dim = q.shape
    kv_heads = rows.shape[3]
    out = np.zeros((tokens, heads, dim))
    lse = np.full((tokens, heads), -np.inf)
    weight = np.zeros((tokens, heads, dim))
    slack = np.zeros((tokens, heads))
    total = np.ones((tokens, heads))
    q = q.astype(np.float64)
    for b, length in enumerate(lengths):
        n = starts[b + 1] - starts[b]
        context = length - n
        pos = np.arange(max(length, 0))
        page_no = np.array([table[b][p // page] for p in pos], np.int64) if length > 0 else np.zeros(0, np.int64)
        inside = (page_no >= 0) & (page_no < rows.shape[0])
        kv = rows[np.where(inside, page_no, 0), pos % page]       # [key][K, V][head][dim]
        for i in range(n):
            t = starts[b] + i
            rel = pos - context
            if masks is None:
                seen = rel <= i
            else:
                seen = np.array([r < 0 or bool(masks[t] >> int(r) & 1) for r in rel], bool).reshape(len(pos))
            seen = seen & inside
            if not seen.any():
                continue
            k, v = kv[seen, 0], kv[seen, 1]
            for h in range(heads):
                g = h * kv_heads // heads
                s = k[:, g] @ q[t, h] * scale
                m = s.max()
                p = np.exp(s - m)
                total[t, h] = p.sum()
                lse[t, h] = m + np.log(p.sum())
                p = p / p.sum()
                out[t, h] = p @ v[:, g]
                weight[t, h] = p @ np.abs(v[:, g])
                slack[t, h] = (np.abs(k[:, g]) @ np.abs(q[t, h])).max() * abs(scale)
    return out, lse, weight, slack, total


def close_attention(got, got_lse, want, lse, weight, slack, total, dim, keys):
    """f32 dot products of `dim` terms are off by (dim + 4) 2^-23 of the sum of their magnitudes, which moves a probability
    by twice that; each probability rounds to f16 once (2^-11), the running sums and exponentials add under 2^-18. A
    probability near f16's smallest step is off by at most 2^-25, which 127 counts multiply and the lift of 16 that int8
    probabilities enter with divides: under keys * 2^-22 over the sum of the probabilities. The result rounds to f16 once."""
    score = slack * (dim + 4) * 2.0 ** -23
    bound = HALF * np.abs(want) + TINY / 2 + weight * (HALF + 2 * score[..., None] + 2.0 ** -18) + keys * 4 * TINY / total[..., None]
    got = np.asarray(got, np.float64)
    assert np.all(np.isfinite(got)), "non-finite output"
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / bound))
    if got_lse is not None:
        empty = np.isneginf(lse)
        assert np.array_equal(np.isneginf(got_lse), empty)
        assert np.all(np.abs(got_lse[~empty] - lse[~empty]) <= (score + 2.0 ** -19 + 2.0 ** -22 * np.abs(lse))[~empty])


def logprobs(x, inv_temperature, tokens, k):
    """x [rows, vocab] float64 of the stored logits. logprob, entropy, ids, their log probabilities, and for the bounds
    sum p|y - m| + |lse - m| and |m| (0 where it is infinite). Everything relative to the maximum m: y - lse would lose
    the logarithm itself where y is a type's lowest value."""
    x = np.asarray(x, np.float64)
    y = x * np.float64(np.float32(inv_temperature))
    rows, vocab = y.shape
    logp, entropy, ids, best = np.full(rows, -np.inf), np.zeros(rows), np.zeros((rows, k), np.int64), np.full((rows, k), -np.inf)
    spread, top = np.zeros(rows), np.zeros(rows)
    for r in range(rows):
        order = np.argsort(-x[r], kind="stable")[:k]
        ids[r] = order
        m = y[r].max()
        if np.isneginf(m):
            continue
        e = np.exp(y[r] - m)
        log_total = np.log(e.sum())
        p = e / e.sum()
        d = np.where(p > 0, y[r] - m, 0.0)
        entropy[r] = log_total - (p * d).sum()
        spread[r] = (p * np.abs(d)).sum() + abs(log_total)
        top[r] = abs(m)
        best[r] = (y[r][order] - m) - log_total
        if 0 <= tokens[r] < vocab:
            logp[r] = (y[r][tokens[r]] - m) - log_total
    return logp, entropy, ids, best, spread, top


def close_logp(got, want, top, vocab):
    """y, the maximum (|m| = top), their difference and the logarithm round to f32 (2^-24 each of their size, and |y| is at
    most |m| + |log p| + ln vocab); the sum of vocab terms, kept in at least 256 running sums, is off by
    (vocab/256 + 64) 2^-24."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    y_most = np.asarray(top, np.float64).reshape((-1,) + (1,) * (want.ndim - 1)) + np.log(vocab)
    dead = np.isneginf(want)
    assert np.array_equal(np.isneginf(got), dead)
    bound = 2.0 ** -22 * (y_most + np.abs(np.where(dead, 0, want)) + 1) + (vocab / 256 + 64) * 2.0 ** -24
    return np.all(np.abs(np.where(dead, 0, got) - np.where(dead, 0, want)) <= bound)
