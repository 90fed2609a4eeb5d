"""Attention where kv_length passes max_kv: positions past the bound are not seen, but which positions are history and which
are query tokens still goes by kv_length."""
import numpy as np
import pytest

from . import verify_ref as ref
from .test_attention_gpu import Step
from .util import Dev

pytestmark = pytest.mark.gpu


def cut_at(step, max_kv):
    """float64 results with positions from max_kv on taken away. The reference counts a mask's bits from the last n of the
    positions it is given, so what each token sees there is written out as such bits."""
    lengths, masks = [min(n, max_kv) for n in step.lengths], []
    for b, n in enumerate(step.lengths):
        count = int(step.starts[b + 1] - step.starts[b])
        context, first = n - count, lengths[b] - count
        for i in range(count):
            word = 0
            for r in range(count):
                rel = first + r - context
                own = rel <= i if step.masks is None else rel < 0 or bool(step.masks[step.starts[b] + i] >> rel & 1)
                word |= int(own and first + r >= 0) << r
            masks.append(word)
    return ref.attention(step.q, ref.rows_of(step.cache), step.page, step.table, step.starts, lengths, masks, step.scale, step.heads)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("tree", [None, "tree"])
@pytest.mark.parametrize("dim,heads,kv_heads,work,max_kv", [
    (128, 8, 2, [(5, 90), (3, 65), (2, 40), (4, 66)], 64),       # one part of the keys; the bound inside the query tokens, before them, past them
    (128, 8, 2, [(4, 3000), (2, 2203), (3, 900)], 2200),         # many parts, joined
    (128, 8, 2, [(40, 600), (33, 520), (9, 100)], 509),          # rows shared by several waves
    (96, 6, 6, [(30, 5000)], 4985),                              # and joined by a launch of their own
    (256, 4, 1, [(7, 300), (1, 280)], 277),
    (20, 4, 2, [(5, 90), (3, 65), (2, 40), (4, 66)], 64),        # the plain kernel
    (20, 2, 1, [(6, 700)], 513)])
def test_lengths_past_the_bound(ctx, capi, dim, heads, kv_heads, work, max_kv, tree, int8):
    s = Step(dim + max_kv, heads, kv_heads, dim, 16, work, int8, tree=tree)
    with Dev(ctx) as d:
        ctx.attention(s.desc(ctx, capi, d, max_kv=max_kv))
        out, lse = s.got(ctx)
    s.compare(out, lse, cut_at(s, max_kv))


@pytest.mark.parametrize("dim", [128, 20])
def test_bounds_of_nothing(ctx, capi, dim):
    """max_kv = 0 leaves no position to see."""
    s = Step(3, 4, 2, dim, 16, [(3, 40), (1, 1)])
    with Dev(ctx) as d:
        ctx.attention(s.desc(ctx, capi, d, max_kv=0))
        out, lse = s.got(ctx)
    assert not out.any() and np.all(np.isneginf(lse))
