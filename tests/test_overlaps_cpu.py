"""Overlapping arrays of the verification dispatches are refused; tried without a GPU, since descriptors are checked before
the context is looked at."""
import pytest

from .test_verify_ops_cpu import f16_cache, int8_cache, refusal

FAR = 1 << 45


@pytest.mark.parametrize("apart,fine", [(2, False), (254, False), (256, True)])
def test_rows_that_end_past_64_bits(capi, apart, fine):
    desc = capi.KvReadDesc(tokens=(1 << 31) - 1, out_stride=(1 << 32) - 1, k_out=FAR, v_out=FAR + apart, slots=0x5000, cache=int8_cache(capi))
    why = refusal(capi, "ztvm_kv_read", desc)[1]
    assert why == "null context" if fine else "overlap" in why, why


def says(capi, name, desc, needle):
    why = refusal(capi, name, desc)[1]
    assert why == "null context" if needle is None else "overlap" in why and needle in why, (needle, why)


# The caches of these tests. f16: four pages of 8 KiB, 0x10000 to 0x18000. int8: 64 pages of 4 KiB, 0x10000 to 0x50000, and
# their scales, 0x20000 to 0x22000 (the arrays that are only read may share memory).

def test_rope_append(capi):
    def desc(cache=None, **kw):
        return capi.RopeAppendDesc(**{**dict(tokens=3, heads=4, rotary_dim=64, qkv_stride=512, q_stride=256, attn_factor=1.0, qkv=0x100000,
                                             q_out=0x200000, frequencies=0x3000, positions=0x4000, slots=0x5000, cache=cache or f16_cache(capi)), **kw})
    for kw, needle in [
            ({}, None), (dict(q_out=0x17FFE), "pages"), (dict(q_out=0x18000), None), (dict(q_out=0x10000 - 3 * 512), None),
            (dict(q_out=0x10000 - 3 * 512 + 2), "pages"), (dict(qkv=0x17FFE), "pages"), (dict(q_out=0x3000), "frequencies"),
            (dict(q_out=0x3000 + 256), None), (dict(positions=0x200000 + 512), "positions"), (dict(slots=0x200000 + 3 * 512 - 4), "slots"),
            (dict(slots=0x200000 + 3 * 512), None),
            (dict(q_stride=512, slots=0x200000 + 512), None),          # between the rows of q_out
            (dict(q_stride=512, slots=0x200000 + 512 - 4), "slots"), (dict(tokens=0, q_out=0x10000), None),
            (dict(cache=int8_cache(capi), q_out=0x21000), "q_out"), (dict(cache=int8_cache(capi, pages=0x600000), q_out=0x21FFC), "scales"),
            (dict(cache=int8_cache(capi, pages=0x600000), qkv=0x21FFC), "scales"), (dict(cache=int8_cache(capi, pages=0x600000), q_out=0x22000), None)]:
        says(capi, "ztvm_rope_append", desc(**kw), needle)
    # the gap behind each of a cache's pages belongs to somebody else
    gaps = f16_cache(capi, kv_page_stride=8192, pages_capacity=3 * 8192 + 4096)
    says(capi, "ztvm_rope_append", desc(gaps, q_out=0x10000 + 8192, q_stride=8192), None)
    says(capi, "ztvm_rope_append", desc(gaps, q_out=0x10000 + 8190, q_stride=8192), "pages")
    says(capi, "ztvm_rope_append", desc(gaps, q_out=0x10000 + 8192, q_stride=4096), "pages")


def test_kv_read(capi):
    def desc(cache=None, **kw):
        return capi.KvReadDesc(**{**dict(tokens=3, out_stride=128, k_out=0x100000, v_out=0x200000, slots=0x5000, cache=cache or int8_cache(capi)), **kw})
    for kw, needle in [({}, None), (dict(k_out=0x12000), "k_out"), (dict(v_out=0x12000), "v_out"), (dict(v_out=0x5000 + 8), "slots"),
                       (dict(v_out=0x5000 + 12), None), (dict(k_out=0, v_out=0x20000), "v_out"), (dict(tokens=0, k_out=0x12000), None),
                       (dict(cache=f16_cache(capi), k_out=0x17FFE), "pages"), (dict(cache=f16_cache(capi), k_out=0x18000), None),
                       (dict(cache=f16_cache(capi, pages_offset=4096), k_out=0x10000), None)]:     # what lies before page 0
        says(capi, "ztvm_kv_read", desc(**kw), needle)


def test_attention(capi):
    def desc(**kw):
        return capi.AttentionDesc(**{**dict(tokens=5, sequences=2, heads=4, max_query=3, max_kv=100, q_stride=256, out_stride=256, page_table_stride=9,
                                            mask_words=1, scale=0.125, q=0x100000, out=0x200000, lse=0x300000, query_start=0x4000, kv_length=0x5000,
                                            page_table=0x6000, tree_mask=0x7000, cache=f16_cache(capi)), **kw})
    for kw, needle in [
            ({}, None), (dict(lse=0x200000 + 5 * 512 - 4), "lse"), (dict(lse=0x200000 + 5 * 512), None), (dict(lse=0x100000), "lse"),
            (dict(lse=0x5004), "kv_length"), (dict(lse=0x5008), None), (dict(out=0x4000), "query_start"), (dict(out=0x400C), None),
            (dict(out=0x6000), "page_table"), (dict(lse=0x6000 + 4 * 7, tokens=1, heads=2), None),     # behind a row's last page that is looked at
            (dict(out=0x7020), "tree_mask"), (dict(out=0x7028), None), (dict(out=0x10000), "pages"), (dict(lse=0x17FFC), "pages"),
            (dict(cache=int8_cache(capi, pages=0x600000), lse=0x20000), "scales"), (dict(out=0x4000, max_query=0), None),
            (dict(lse=0x4000, sequences=0), None), (dict(lse=0, tree_mask=0, mask_words=0, page_table=0, page_table_stride=0, sequences=1), None)]:
        says(capi, "ztvm_attention", desc(**kw), needle)


def test_token_logprobs(capi):
    def desc(**kw):
        return capi.TokenLogprobsDesc(**{**dict(rows=2, vocab=100, row_stride=128, top_k=5, inv_temperature=1.0, logits=0x1000, tokens=0x2000,
                                                logprob=0x3000, entropy=0x4000, top_ids=0x5000, top_logprobs=0x6000), **kw})
    for kw, needle in [({}, None), (dict(logprob=0x1000), "logits"), (dict(logprob=0x1000 + 400), None), (dict(logprob=0x1000 + 508), "logits"),
                       (dict(logprob=0x1000 + 504), None), (dict(entropy=0x3004), "entropy"), (dict(entropy=0x3008), None),
                       (dict(top_ids=0x2004), "tokens"), (dict(top_ids=0x2004, logprob=0), None), (dict(top_logprobs=0x5000), "top_logprobs"),
                       (dict(top_k=0, top_logprobs=0x5000), None), (dict(rows=0, logprob=0x1000), None), (dict(logits_f16=1, logprob=0x1000 + 200), None)]:
        says(capi, "ztvm_token_logprobs", desc(**kw), needle)


def test_one_result_a_row_may_replace_the_tokens(capi):
    base = dict(rows=3, vocab=100, row_stride=100, top_k=1, inv_temperature=1.0, logits=0x1000, tokens=0x8000, logprob=0x9000, entropy=0xA000, top_ids=0xB000)
    for kw, needle in [(dict(top_ids=0x8000), None), (dict(logprob=0x8000), None), (dict(entropy=0x8000), None), (dict(top_ids=0x8004), "tokens"),
                       (dict(top_ids=0x8000, top_k=2), "tokens"), (dict(top_ids=0x8000, entropy=0x8000), "top_ids")]:
        says(capi, "ztvm_token_logprobs", capi.TokenLogprobsDesc(**{**base, **kw}), needle)
