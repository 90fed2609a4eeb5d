"""Token log probabilities where one result a row replaces the given tokens: the same bits as beside them."""
import numpy as np
import pytest

from .util import Dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [100, 5000, 40000, 2097152])      # one launch, two, two, a row a workgroup with many passes
@pytest.mark.parametrize("field", ["logprob", "entropy", "top_ids"])
def test_in_place(ctx, capi, field, vocab):
    rows = 5
    rng = np.random.default_rng(vocab)
    x, tokens = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32), rng.integers(0, vocab, rows).astype(np.int32)
    fields = ("logprob", "entropy", "top_ids", "top_logprobs")
    with Dev(ctx) as d:
        logits, got = d.put(x), []
        for place in (None, field):
            at = {f: d.empty(rows * 4) for f in fields}
            given = d.put(tokens)
            if place:
                at[place] = given
            ctx.token_logprobs(capi.TokenLogprobsDesc(rows=rows, vocab=vocab, row_stride=vocab, top_k=1, inv_temperature=1.0, logits=logits, tokens=given, **at))
            got.append([ctx.download(at[f], rows * 4, np.uint32) for f in fields])
    assert all(np.array_equal(a, b) for a, b in zip(*got))
    assert np.array_equal(got[1][2], np.argmax(x, 1))
