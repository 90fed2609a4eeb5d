"""The verification dispatches on a machine without a GPU: descriptor layouts, refusals (a null context is looked at
last, so a good descriptor gets as far as "null context"), the rotary frequency tables, the page arithmetic."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_page_arithmetic(tmp_path):
    exe = str(tmp_path / "kv_cache_test")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-o", exe, os.path.join(ROOT, "tests", "cpp", "kv_cache_test.cc")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


def test_descriptors_match_the_header(capi, tmp_path):
    names = {"ztvm_kv_cache": capi.KvCache, "ztvm_rope_append_desc": capi.RopeAppendDesc, "ztvm_kv_read_desc": capi.KvReadDesc,
             "ztvm_attention_desc": capi.AttentionDesc, "ztvm_token_logprobs_desc": capi.TokenLogprobsDesc}
    lines = ['#include "%s"' % os.path.join(ROOT, "include", "ztvm.h"), "#include <stdio.h>", "#include <stddef.h>", "int main(void) {"]
    for c, py in names.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (c, c))
        for f in py._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (c, f[0], c, f[0]))
    src, exe = tmp_path / "layout.c", str(tmp_path / "layout")
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-o", exe, str(src)], check=True)
    said = dict(l.rsplit(" ", 1) for l in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines())
    for c, py in names.items():
        assert int(said[c]) == ctypes.sizeof(py)
        for f in py._fields_:
            assert int(said["%s.%s" % (c, f[0])]) == getattr(py, f[0]).offset, f[0]


def f16_cache(capi, **kw):
    return capi.KvCache(**{**dict(format=capi.KV_F16, kv_heads=2, head_dim=64, page_size=16, head_page_stride=1024, v_page_offset=2048,
                                  kv_page_stride=4096, pages_capacity=4096 * 4, pages=0x10000), **kw})


def int8_cache(capi, **kw):
    return capi.KvCache(**{**dict(format=capi.KV_INT8, kv_heads=2, head_dim=64, page_size=16, pages_capacity=1 << 16,
                                  scales_capacity=1 << 12, pages=0x10000, scales=0x20000), **kw})


def refusal(capi, name, desc):
    lib = capi.load()
    rc = getattr(lib, name)(None, None if desc is None else ctypes.byref(desc))
    assert rc < 0
    return rc, lib.ztvm_last_error(None).decode()


def check_refusals(capi, name, make, good, bad):
    rc, why = refusal(capi, name, make(**good))
    assert why == "null context", why
    assert "null descriptor" in refusal(capi, name, None)[1]
    for change, needle in bad:
        rc, why = refusal(capi, name, make(**{**good, **change}))
        assert rc in (capi.E_INVALID, capi.E_UNSUPPORTED) and needle in why and name in why, (change, why)


def cache_refusals(capi):
    f = lambda **kw: dict(cache=f16_cache(capi, **kw))  # noqa: E731
    i = lambda **kw: dict(cache=int8_cache(capi, **kw))  # noqa: E731
    return [(f(format=2), "format"), (f(kv_heads=0), "kv_heads"), (f(head_dim=0), "head_dim"), (f(page_size=0), "page_size"),
            (f(head_dim=514), "512"), (f(pages=0), "null"), (f(pages=0x10008), "misaligned"), (f(pages_capacity=0), "capacities"),
            (f(head_page_stride=1023), "overlaps"), (f(v_page_offset=2047), "overlaps"), (f(kv_page_stride=4095), "overlaps"),
            (f(pages_capacity=1 << 60), "capacity"), (f(page_size=1 << 31), "page_size"),
            (i(scales=0), "null"), (i(scales=0x20002), "misaligned"), (i(scales_capacity=0), "capacities"), (i(head_dim=66), "multiple of 4")]


def test_rope_append_refuses(capi):
    good = dict(tokens=3, heads=4, rotary_dim=64, qkv_stride=512, q_stride=256, attn_factor=1.0, qkv=0x100000, q_out=0x200000,
                frequencies=0x3000, positions=0x4000, slots=0x5000, cache=f16_cache(capi))
    check_refusals(capi, "ztvm_rope_append", capi.RopeAppendDesc, good, cache_refusals(capi) + [
        (dict(heads=0), "heads"), (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=63), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"),
        (dict(interleaved=2), "interleaved"), (dict(qkv_stride=511), "qkv_stride"), (dict(q_stride=255), "q_stride"),
        (dict(attn_factor=0.0), "attn_factor"), (dict(attn_factor=math.nan), "attn_factor"), (dict(attn_factor=math.inf), "attn_factor"),
        (dict(qkv=0), "null"), (dict(q_out=0), "null"), (dict(frequencies=0), "null"), (dict(positions=0), "null"), (dict(slots=0), "null"),
        (dict(qkv=0x100001), "misaligned"), (dict(frequencies=0x3004), "misaligned"), (dict(positions=0x4002), "misaligned"),
        (dict(tokens=1 << 31), "tokens"), (dict(q_out=0x100000), "overlaps"), (dict(q_out=0x100000 + 1024, q_stride=512), "overlaps"),
        (dict(cache=f16_cache(capi, head_dim=63, head_page_stride=1024)), "even")])
    # in place, and a column window of one wider array
    for fine in (dict(q_out=0x100000, q_stride=512), dict(qkv_stride=768, q_out=0x100000 + 1024, q_stride=768), dict(tokens=0, q_out=0x100000)):
        assert refusal(capi, "ztvm_rope_append", capi.RopeAppendDesc(**{**good, **fine}))[1] == "null context"
    assert refusal(capi, "ztvm_rope_append", capi.RopeAppendDesc(**{**good, "cache": int8_cache(capi)}))[1] == "null context"


def test_kv_read_refuses(capi):
    good = dict(tokens=3, out_stride=128, k_out=0x100000, v_out=0x200000, slots=0x5000, cache=int8_cache(capi))
    check_refusals(capi, "ztvm_kv_read", capi.KvReadDesc, good, cache_refusals(capi) + [
        (dict(out_stride=127), "out_stride"), (dict(k_out=0, v_out=0), "null"), (dict(slots=0), "null"), (dict(k_out=0x100001), "misaligned"),
        (dict(slots=0x5001), "misaligned"), (dict(v_out=0x100000), "overlap"), (dict(tokens=1 << 31), "tokens")])
    for fine in (dict(k_out=0), dict(v_out=0), dict(out_stride=256, v_out=0x100000 + 256)):
        assert refusal(capi, "ztvm_kv_read", capi.KvReadDesc(**{**good, **fine}))[1] == "null context"


def test_attention_refuses(capi):
    good = dict(tokens=5, sequences=2, heads=4, max_query=3, max_kv=100, q_stride=256, out_stride=256, page_table_stride=7, mask_words=1,
                scale=0.125, q=0x100000, out=0x200000, lse=0x300000, query_start=0x4000, kv_length=0x5000, page_table=0x6000,
                tree_mask=0x7000, cache=f16_cache(capi))
    check_refusals(capi, "ztvm_attention", capi.AttentionDesc, good, cache_refusals(capi) + [
        (dict(heads=0), "heads"), (dict(heads=3), "heads"), (dict(q_stride=255), "q_stride"), (dict(out_stride=255), "out_stride"),
        (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(q=0), "null"), (dict(out=0), "null"),
        (dict(query_start=0), "null"), (dict(kv_length=0), "null"), (dict(q=0x100001), "misaligned"), (dict(lse=0x300002), "misaligned"),
        (dict(page_table=0x6001), "misaligned"), (dict(tree_mask=0x7004), "misaligned"), (dict(max_kv=113), "page_table_stride"),
        (dict(page_table=0), "page_table"), (dict(max_query=65), "mask_words"), (dict(mask_words=0), "mask_words"),
        (dict(sequences=65536), "sequences"), (dict(tokens=1 << 31), "tokens"), (dict(max_kv=1 << 31), "max_kv"), (dict(out=0x100200), "overlaps")])
    for fine in (dict(lse=0), dict(tree_mask=0, mask_words=0, max_query=900), dict(page_table=0, sequences=1, page_table_stride=0),
                 dict(max_kv=0), dict(cache=int8_cache(capi))):
        assert refusal(capi, "ztvm_attention", capi.AttentionDesc(**{**good, **fine}))[1] == "null context"


def test_token_logprobs_refuses(capi):
    good = dict(rows=2, vocab=100, row_stride=128, top_k=5, inv_temperature=1.0, logits=0x1000, tokens=0x2000, logprob=0x3000,
                entropy=0x4000, top_ids=0x5000, top_logprobs=0x6000)
    check_refusals(capi, "ztvm_token_logprobs", capi.TokenLogprobsDesc, good, [
        (dict(vocab=0), "vocab"), (dict(row_stride=99), "row_stride"), (dict(logits_f16=2), "logits_f16"), (dict(top_k=65), "top_k"),
        (dict(vocab=4), "top_k"), (dict(inv_temperature=0.0), "inv_temperature"), (dict(inv_temperature=math.inf), "inv_temperature"),
        (dict(inv_temperature=math.nan), "inv_temperature"), (dict(logits=0), "null"), (dict(tokens=0), "tokens"),
        (dict(logits=0x1002), "misaligned"), (dict(logits_f16=1, logits=0x1001), "misaligned"), (dict(top_ids=0x5002), "misaligned"),
        (dict(rows=1 << 31), "rows"), (dict(vocab=1 << 31, row_stride=1 << 31), "vocab")])
    for fine in (dict(top_k=0, top_ids=0, top_logprobs=0), dict(tokens=0, logprob=0), dict(entropy=0), dict(logits_f16=1, logits=0x1002)):
        assert refusal(capi, "ztvm_token_logprobs", capi.TokenLogprobsDesc(**{**good, **fine}))[1] == "null context"


def test_frequencies(capi):
    """Against the formulas, written again here; f64 throughout, so 1e-14 relative covers the library functions."""
    rotary, theta = 128, 500000.0
    j = np.arange(rotary // 2)
    base = np.exp(-2.0 * j / rotary * np.log(theta))
    got, factor = capi.rope_frequencies(capi.ROPE_PLAIN, rotary, theta)
    assert np.allclose(got, base, rtol=1e-13, atol=0) and factor == 1.0
    got, factor = capi.rope_frequencies(capi.ROPE_LINEAR, rotary, theta, 4.0)
    assert np.allclose(got, base / 4, rtol=1e-13, atol=0) and factor == 1.0
    got, factor = capi.rope_frequencies(capi.ROPE_PIECEWISE, rotary, theta, 8.0, 8192.0, 1.0, 4.0)
    wave = 2 * np.pi / base
    want = np.where(wave > 8192, base / 8, base)
    mid = (wave <= 8192) & (wave >= 8192 / 4)
    blend = (8192 / wave - 1.0) / 3.0
    want[mid] = ((1 - blend) * base / 8 + blend * base)[mid]
    assert np.allclose(got, want, rtol=1e-12, atol=0) and factor == 1.0
    assert got[0] == 1.0 and np.isclose(got[-1], base[-1] / 8) and mid.any()
    got, factor = capi.rope_frequencies(capi.ROPE_YARN, rotary, theta, 16.0, 8192.0, 1.0, 32.0)
    dim_of = lambda turns: rotary * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    low, high = math.floor(dim_of(32.0)), math.ceil(dim_of(1.0))
    ramp = np.clip((j - low) / (high - low), 0, 1)
    assert np.allclose(got, base / 16 * ramp + base * (1 - ramp), rtol=1e-13, atol=0)
    assert abs(factor - (0.1 * math.log(16) + 1)) < 1e-6 and 0 < low < high < rotary // 2
    assert np.all(np.diff(got) < 0)
    # a stretch of one changes nothing
    for kind in (capi.ROPE_LINEAR, capi.ROPE_PIECEWISE, capi.ROPE_YARN):
        got, factor = capi.rope_frequencies(kind, rotary, theta, 1.0, 8192.0, 1.0, 4.0)
        assert np.allclose(got, base, rtol=1e-13, atol=0) and factor == 1.0
    assert capi.rope_frequencies(capi.ROPE_PLAIN, 2, 10000.0)[0].tolist() == [1.0]


@pytest.mark.parametrize("args,needle", [
    ((4, 64, 1e4), "kind"), ((0, 63, 1e4), "rotary_dim"), ((0, 0, 1e4), "rotary_dim"), ((0, 514, 1e4), "rotary_dim"), ((0, 64, 1.0), "theta"),
    ((0, 64, math.nan), "theta"), ((1, 64, 1e4, 0.5), "factor"), ((2, 64, 1e4, 2.0, 0.0, 1.0, 4.0), "original"),
    ((3, 64, 1e4, 2.0, 8192.0, 4.0, 4.0), "low"), ((2, 64, 1e4, 2.0, 8192.0, 0.0, 4.0), "low"), ((3, 64, 1e4, math.inf, 8192.0, 1.0, 4.0), "factor")])
def test_frequencies_refuse(capi, args, needle):
    with pytest.raises(capi.ZtvmError, match=needle):
        capi.rope_frequencies(*args)


def test_limits_of_a_launch(capi):
    """The largest counts a launch takes, and one more."""
    rope = dict(tokens=(1 << 24) - 1, heads=4, rotary_dim=64, qkv_stride=512, q_stride=256, attn_factor=1.0, qkv=0x100000, q_out=1 << 45,
                frequencies=0x3000, positions=0x4000, slots=0x5000, cache=f16_cache(capi))
    check_refusals(capi, "ztvm_rope_append", capi.RopeAppendDesc, rope, [(dict(tokens=1 << 24), "tokens")])
    attention = dict(tokens=(1 << 24) - 1, sequences=1, heads=4, max_query=(1 << 30) - 1, max_kv=(1 << 30) - 1, q_stride=256, out_stride=256, scale=1e30,
                     q=0x100000, out=1 << 45, query_start=0x4000, kv_length=0x5000, cache=f16_cache(capi))
    check_refusals(capi, "ztvm_attention", capi.AttentionDesc, attention, [
        (dict(tokens=1 << 24), "tokens"), (dict(max_query=1 << 30), "max_query"), (dict(max_kv=1 << 30), "max_kv"), (dict(scale=1.1e30), "scale"),
        (dict(scale=-1.1e30), "scale")])
    score = dict(rows=(1 << 24) - 1, vocab=100, row_stride=128, inv_temperature=1.0, logits=0x1000)
    check_refusals(capi, "ztvm_token_logprobs", capi.TokenLogprobsDesc, score, [(dict(rows=1 << 24), "rows")])
