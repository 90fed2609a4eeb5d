"""Attention over int8 rows of small values: the bits of the result do not depend on the values' size, nor on how many rows
share the keys."""
import numpy as np
import pytest

from . import small_values
from .test_attention_gpu import Step
from .util import Dev

pytestmark = pytest.mark.gpu


def run(ctx, capi, s):
    with Dev(ctx) as d:
        ctx.attention(s.desc(ctx, capi, d))
        out, lse = s.got(ctx)
    return out[:s.tokens, :s.heads * s.dim].reshape(s.tokens, s.heads, s.dim), lse[:s.tokens]


@pytest.mark.parametrize("value_scale", [1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("heads,kv_heads,dim,queries", [
    (1, 1, 128, 1), (8, 1, 128, 1), (8, 2, 64, 8), (2, 2, 256, 8), (4, 1, 96, 5),     # up to 32 rows a kv head
    (4, 1, 128, 12), (4, 1, 128, 40), (2, 1, 20, 3)])                                # waves that share the rows; the plain kernel
@pytest.mark.parametrize("keys", [60, 4000])
def test_peaked_rows(ctx, capi, keys, heads, kv_heads, dim, queries, value_scale):
    s = small_values.step(Step, keys + dim, heads, kv_heads, dim, [(queries, keys), (1, keys // 2 + 1)], value_scale)
    small_values.close(s, *run(ctx, capi, s), s.want())


@pytest.mark.parametrize("heads,kv_heads,dim,queries", [(8, 2, 128, 1), (4, 1, 64, 7), (4, 1, 128, 12)])
@pytest.mark.parametrize("peak", [0, 31, 1500])
@pytest.mark.parametrize("spread,value_scale", [(10.0, 1e-2), (10.0, 300.0), (4.0, 1e-4)])
def test_scales_of_all_sizes(ctx, capi, heads, kv_heads, dim, queries, peak, spread, value_scale):
    """The leading key first, inside a tile and far behind; the scales of one row a thousand times apart."""
    s = small_values.step(Step, peak + dim, heads, kv_heads, dim, [(queries, 2500), (queries, 1700)], value_scale, gap=9.0, peak=peak, spread=spread)
    small_values.close(s, *run(ctx, capi, s), s.want())


@pytest.mark.parametrize("queries", [1, 7, 40])
@pytest.mark.parametrize("keys", [40, 3000])
def test_scales_of_zero(ctx, capi, queries, keys):
    """Values that are all zero by their scale give zeros and the sums of the scores; so do some of them among others."""
    s = small_values.step(Step, 5, 4, 1, 128, [(queries, keys), (queries, keys // 2 + queries)], 1e-3)
    scales = s.cache[1]
    scales[:, :, 1::2, 1] = 0
    small_values.close(s, *run(ctx, capi, s), s.want())
    scales[..., 1] = 0
    out, lse = run(ctx, capi, s)
    assert not out.any()
    small_values.close(s, out, lse, s.want())
    scales[..., 0] = 0                                   # and all scores equal
    out, lse = run(ctx, capi, s)
    assert not out.any() and np.all(np.isfinite(lse))
    small_values.close(s, out, lse, s.want())
