"""GPU parity of token log probabilities, entropy and the best alternatives, through the C ABI, against float64."""
import numpy as np
import pytest

from . import verify_ref as ref
from .util import Dev

pytestmark = pytest.mark.gpu


def call(ctx, capi, x, tokens, k, inv_t=1.0, stride=None, outputs=("logprob", "entropy", "top_ids", "top_logprobs"), offset=0):
    rows, vocab = x.shape
    stride = stride or vocab
    wide = np.full(rows * stride + offset, np.nan, x.dtype)
    for r in range(rows):
        wide[offset + r * stride:offset + r * stride + vocab] = x[r]
    kinds = {"logprob": np.float32, "entropy": np.float32, "top_ids": np.uint32, "top_logprobs": np.float32}
    with Dev(ctx) as d:
        at = {n: d.put(np.full((rows + 1) * (k if n.startswith("top") else 1), 7, kinds[n])) for n in outputs}
        ctx.token_logprobs(capi.TokenLogprobsDesc(rows=rows, vocab=vocab, row_stride=stride, logits_f16=int(x.dtype == np.float16), top_k=k,
                                                  inv_temperature=inv_t, logits=d.put(wide) + offset * x.itemsize,
                                                  tokens=d.put(np.asarray(tokens, np.int32)), **at))
        got = {n: ctx.download(at[n], (rows + 1) * (k if n.startswith("top") else 1) * 4, kinds[n]) for n in outputs}
    for n, a in got.items():
        per = k if n.startswith("top") else 1
        assert np.all(a[rows * per:] == 7), "nothing is written past the rows"
        got[n] = a[:rows * per].reshape(rows, k) if n.startswith("top") else a[:rows]
    return got


def check(ctx, capi, x, tokens, k, inv_t=1.0, **kw):
    got = call(ctx, capi, x, tokens, k, inv_t, **kw)
    logp, entropy, ids, best, spread, top = ref.logprobs(x, inv_t, tokens, k)
    vocab = x.shape[1]
    if "logprob" in got:
        assert ref.close_logp(got["logprob"], logp, top, vocab)
    if "entropy" in got:
        # the weighted sum and its weights are off by what a log probability of a likely token is (|y| within |m| + 32, the
        # rest weighs nothing), times the spread they multiply
        assert np.all(np.abs(got["entropy"] - entropy) <= (2.0 ** -21 * (32 + top) + (vocab / 256 + 64) * 2.0 ** -23) * (1 + spread))
    if "top_ids" in got:
        assert np.array_equal(got["top_ids"], ids)
    if "top_logprobs" in got and k:
        assert ref.close_logp(got["top_logprobs"], best, top, vocab)
    return got


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,vocab,k,pad,offset", [
    (1, 1, 1, 0, 0), (1, 2, 2, 0, 0), (3, 5, 5, 0, 0), (2, 63, 7, 0, 0), (5, 64, 64, 0, 0), (4, 65, 64, 3, 1), (7, 255, 20, 0, 0),
    (2, 257, 20, 0, 3), (3, 1023, 1, 1, 0), (3, 1025, 33, 0, 0), (2, 4097, 64, 7, 0), (9, 32064, 20, 0, 0), (1, 50257, 8, 0, 1), (70, 8191, 5, 1, 0),
    (1, 248320, 20, 0, 0), (300, 2000, 3, 0, 0), (2, 131072, 64, 8, 0), (2, 16384, 0, 0, 0)])
def test_shapes(ctx, capi, rows, vocab, k, pad, offset, dtype):
    rng = np.random.default_rng(vocab + rows)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(dtype)
    tokens = rng.integers(0, vocab, rows)
    check(ctx, capi, x, tokens, k, 1.0, stride=vocab + pad, offset=offset)
    check(ctx, capi, x, tokens, k, 0.37, stride=vocab + pad, offset=offset)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_masked_logits(ctx, capi, dtype):
    """-inf, the type's lowest value, and what is left of a row that is masked out but for one, or altogether."""
    rng = np.random.default_rng(0)
    vocab = 5000
    x = (rng.standard_normal((6, vocab)) * 2).astype(dtype)
    x[0, rng.random(vocab) < 0.9] = -np.inf
    x[1] = -np.inf
    x[1, 777] = -3.0
    x[2] = -np.inf                                     # nothing is left
    x[3, rng.random(vocab) < 0.9] = np.finfo(dtype).min
    x[4] = np.finfo(dtype).min
    got = check(ctx, capi, x, [int(np.argmax(x[0])), 777, 5, 3, 9, 11], 20, 1.0)
    assert got["logprob"][1] == 0.0 and got["entropy"][1] == 0.0 and got["top_ids"][1, 0] == 777 and np.all(np.isneginf(got["top_logprobs"][1, 1:]))
    assert np.isneginf(got["logprob"][2]) and got["entropy"][2] == 0.0 and np.all(np.isneginf(got["top_logprobs"][2]))
    assert got["top_ids"][2].tolist() == list(range(20)) and got["top_ids"][4].tolist() == list(range(20))
    check(ctx, capi, x[:3], [1, 2, 3], 20, 1.0 / 0.7)  # given tokens among the masked ones: -inf


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", [300, 9000, 70000])
def test_ties_go_to_the_lower_id(ctx, capi, dtype, vocab):
    rng = np.random.default_rng(vocab)
    x = np.stack([np.zeros(vocab), rng.integers(0, 3, vocab), np.where(np.arange(vocab) % 2, 0.0, -0.0), rng.integers(0, 400, vocab) / 8.0,
                  np.arange(vocab) % 7, -(np.arange(vocab) // 50.0)]).astype(dtype)
    for k in (1, 20, 64):
        check(ctx, capi, x, [0] * 6, k)


def test_order_at_the_edges(ctx, capi):
    """The best values at the first and last places, all in one neighbourhood, and in ascending or descending rows."""
    vocab = 40001
    x = np.random.default_rng(3).standard_normal((6, vocab)).astype(np.float32)
    x[0, [0, vocab - 1, 1, vocab - 2]] = [50, 51, 52, 53]
    x[1, 12345:12345 + 70] = np.linspace(20, 30, 70)
    x[2] = np.linspace(-5, 5, vocab)
    x[3] = np.linspace(5, -5, vocab)
    x[4, ::997] = 9.0
    x[5, -64:] = 40.0
    check(ctx, capi, x, [0, 12400, vocab - 1, 0, 997, 5], 64)


def test_tokens_outside_the_vocabulary(ctx, capi):
    x = np.random.default_rng(4).standard_normal((5, 100)).astype(np.float32)
    got = check(ctx, capi, x, [-1, 100, 99, 2 ** 31 - 1, -2 ** 31], 3, stride=101)
    assert np.array_equal(np.isneginf(got["logprob"]), [True, True, False, True, True])


def test_nan_and_positive_infinity(ctx, capi):
    """NaN log probabilities and entropy in those rows only; the ids follow the order of the logits, NaN last."""
    vocab = 3000
    x = np.random.default_rng(5).standard_normal((4, vocab)).astype(np.float32)
    x[1, 1234] = np.nan
    x[2, 77] = np.inf
    x[3] = np.nan
    x[3, 5] = 1.0
    got = call(ctx, capi, x, [1, 1, 1, 5], 4)
    for r in (1, 2, 3):
        assert np.isnan(got["logprob"][r]) and np.isnan(got["entropy"][r]) and np.all(np.isnan(got["top_logprobs"][r])), r
    assert np.array_equal(got["top_ids"][1], np.argsort(-np.where(np.isnan(x[1]), -np.inf, x[1]), kind="stable")[:4])
    assert got["top_ids"][2, 0] == 77 and got["top_ids"][3].tolist() == [5, 0, 1, 2]
    clean = ref.logprobs(x[:1], 1.0, [1], 4)
    assert np.array_equal(got["top_ids"][0], clean[2][0]) and ref.close_logp(got["logprob"][:1], clean[0], clean[5], vocab)


@pytest.mark.parametrize("outputs", [("logprob",), ("entropy",), ("top_ids",), ("top_logprobs",), ("top_ids", "entropy")])
def test_some_outputs(ctx, capi, outputs):
    x = np.random.default_rng(6).standard_normal((3, 10000)).astype(np.float16)
    check(ctx, capi, x, [5, 6, 7], 6, outputs=outputs)


@pytest.mark.parametrize("scale", [1e30, 1e-30, 80.0])
def test_extreme_scales(ctx, capi, scale):
    """Logits far apart (one probability is 1) and all but equal."""
    x = (np.random.default_rng(7).standard_normal((2, 3000)) * scale).astype(np.float32)
    got = call(ctx, capi, x, [1, 2], 5)
    logp, entropy, ids, best, _, _ = ref.logprobs(x, 1.0, [1, 2], 5)
    assert np.array_equal(got["top_ids"], ids)
    assert np.allclose(got["logprob"], logp, rtol=2.0 ** -20, atol=1e-5) and np.allclose(got["top_logprobs"], best, rtol=2.0 ** -20, atol=1e-5)
    assert np.allclose(got["entropy"], entropy, atol=1e-4)


@pytest.mark.parametrize("dtype,vocab", [(np.float32, 2097148), (np.float32, 2097152), (np.float16, 4194300), (np.float16, 4200001)])
def test_rows_at_and_past_the_table_of_neighbourhoods(ctx, capi, dtype, vocab):
    x = (np.random.default_rng(10).standard_normal((2, vocab)) * 3).astype(dtype)
    check(ctx, capi, x, [7, vocab - 1], 3)


@pytest.mark.parametrize("rows", [513, 1500])
def test_many_rows(ctx, capi, rows):
    x = (np.random.default_rng(rows).standard_normal((rows, 9001)) * 3).astype(np.float16)
    check(ctx, capi, x, np.arange(rows), 9)


def test_offsets_past_32_bits(ctx, capi):
    """Rows whose elements lie past 2^32 of the array."""
    vocab, stride, rows = 2000, 1 << 31, 3
    x = np.random.default_rng(8).standard_normal((rows, vocab)).astype(np.float16)
    with Dev(ctx) as d:
        big = d.empty((rows - 1) * stride * 2 + vocab * 2)
        for r in range(rows):
            ctx.upload(big, x[r], r * stride * 2)
        lp = d.empty(rows * 4)
        ctx.token_logprobs(capi.TokenLogprobsDesc(rows=rows, vocab=vocab, row_stride=stride, logits_f16=1, inv_temperature=1.0, logits=big,
                                                  tokens=d.put(np.array([1, 2, 3], np.int32)), logprob=lp))
        got = ctx.download(lp, rows * 4, np.float32)
    assert ref.close_logp(got, ref.logprobs(x, 1.0, [1, 2, 3], 1)[0], np.abs(x.max(1)), vocab)


def test_recorded(ctx, capi):
    """A recorded dispatch replayed on new logits equals the eager one on each replay."""
    rng = np.random.default_rng(9)
    rows, vocab, k = 5, 30000, 8
    with Dev(ctx) as d:
        logits = d.empty(rows * vocab * 4)
        outs = [d.empty(rows * 4), d.empty(rows * 4), d.empty(rows * k * 4), d.empty(rows * k * 4)]
        desc = capi.TokenLogprobsDesc(rows=rows, vocab=vocab, row_stride=vocab, top_k=k, inv_temperature=1.0, logits=logits,
                                      tokens=d.put(np.arange(rows, dtype=np.int32)), logprob=outs[0], entropy=outs[1], top_ids=outs[2], top_logprobs=outs[3])
        ctx.token_logprobs(desc)
        ctx.record_begin()
        ctx.token_logprobs(desc)
        cb = ctx.record_end()
        read = lambda: [ctx.download(o, rows * (k if i > 1 else 1) * 4, np.uint32) for i, o in enumerate(outs)]  # noqa: E731
        try:
            for _ in range(4):
                ctx.upload(logits, (rng.standard_normal((rows, vocab)) * 3).astype(np.float32))
                for o in outs:
                    ctx.fill(o, 0x55, rows * 4)
                ctx.submit(cb)
                a = read()
                ctx.token_logprobs(desc)
                assert all(np.array_equal(x, y) for x, y in zip(a, read()))
        finally:
            ctx.cmdbuf_destroy(cb)
    ctx.token_logprobs(capi.TokenLogprobsDesc(rows=0, vocab=5, row_stride=5, inv_temperature=1.0, logits=0x1000))
