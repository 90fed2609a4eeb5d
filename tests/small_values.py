"""int8 caches whose softmax is peaked and whose values are small, and a bound of the attention over them that shrinks with
the values.

Scores are exact up to their scaling: queries are multiples of 1/8 within 2 and keys are whole counts, so a dot product of
512 terms is a whole number of eighths below 2^17, which f32 holds in any order of summation."""
import numpy as np

from . import verify_ref as ref


def step(Step, seed, heads, kv_heads, dim, work, value_scale, gap=12.0, page=16, peak=0, spread=0.0):
    """A Step whose key at position `peak` leads every other by about `gap` nats and has a value 64 times smaller than theirs;
    the values of a row lie around 60 counts, so that they add up. spread: the value scales lie within 2^-spread of value_scale."""
    s = Step(seed, heads, kv_heads, dim, page, work, True)
    rng = np.random.default_rng(seed + 1)
    q8 = rng.integers(8, 17, (s.tokens, heads, dim)) * np.where(np.arange(dim) % 2, 1, -1)
    s.q = (q8 / 8.0).astype(np.float16)
    counts, scales = s.cache
    counts[..., 0, :] = rng.integers(-3, 4, counts[..., 0, :].shape)
    counts[..., 1, :] = np.clip(rng.integers(40, 81, counts[..., 1, :].shape), -127, 127)
    scales[..., 0] = np.float16(0.01)
    scales[..., 1] = (value_scale * 2.0 ** (-spread * rng.random(scales[..., 1].shape))).astype(np.float16)
    per_count = np.abs(s.q.astype(np.float64)).sum(-1).mean() * s.scale * 0.01     # nats for a count that is aligned with the queries
    lead = int(min(127, np.ceil(gap / per_count)))
    scales[..., 0] = np.float16(0.01 * gap / (per_count * lead))
    for b, n in enumerate(s.lengths):
        at = min(peak, n - 1)
        p, slot = s.table[b, at // page], at % page
        counts[p, :, slot, 0] = lead * np.where(np.arange(dim) % 2, 1, -1)
        scales[p, :, slot, 1] = np.float16(value_scale / 64.0)
    return s


def bound(s, want, lse, weight, slack, total):
    """out and lse errors.

    A score meets five f32 roundings of its size (the scale's product with log2 e, the key's scale, the product with the exact
    dot product, the difference from the reference) and its exponential one more: under 2^-21 (|score| + 1), |score| <= slack.
    The sums run over at most 2^13 keys in parts of at most 2^10: under 2^-18 with the rescalings.

    A probability, times the value's scale or what its power of two leaves of it, rounds to f16 once: 2^-11, or half of f16's
    smallest step. They enter lifted by 2^9, so this step is 2^-34 of the largest of them; where the power of two is in the
    value instead, of the largest probability times that power, which is at most the scale but never under 2^-13.
    `keys` roundings, each times 127 counts. The result rounds to f16 once."""
    keys = max(s.lengths)
    value = max(float(np.max(s.cache[1][..., 1].astype(np.float64))), 2.0 ** -13)
    score = 2.0 ** -21 * (slack + 1)
    floor = keys * 127 * 2.0 ** -34 * value / total
    out = ref.HALF * np.abs(want) + ref.TINY / 2 + weight * (ref.HALF + 2 * score[..., None] + 2.0 ** -18) + floor[..., None]
    return out, score + 2.0 ** -17


def close(s, out, lse, w):
    """out [tokens, heads, dim] and lse [tokens, heads] against w = s.want()"""
    want, want_lse = w[:2]
    b, b_lse = bound(s, *w)
    out = np.asarray(out, np.float64)
    assert np.all(np.isfinite(out))
    worst = float(np.max(np.abs(out - want) / b))
    assert worst <= 1.0, worst
    assert np.all(np.abs(np.asarray(lse, np.float64) - want_lse) <= b_lse), float(np.max(np.abs(lse - want_lse) / b_lse))
    return worst
