"""The verification dispatches through the JavaScript host: refusals on the CPU, a small step on the GPU."""
import json
import os
import subprocess

import numpy as np
import pytest

from . import verify_ref as ref
from .test_js_host import ADDON, NODE, ROOT, ensure_addon, needs_node


@needs_node
def test_refusals_and_tables():
    ensure_addon()
    r = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "verify_cpu.js")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "js verify cpu checks ok" in r.stdout, r.stdout + r.stderr


@needs_node
@pytest.mark.gpu
def test_step(tmp_path, capi):
    assert os.path.exists(ADDON), "the N-API addon must be built in-tree before GPU runs"
    heads, kv_heads, dim, page, vocab, k = 4, 2, 64, 16, 900, 4
    rng = np.random.default_rng(1)
    queries, lengths = [3, 2], [40, 5]
    tokens, starts = 5, np.array([0, 3, 5])
    table = np.array([[2, 0, 4], [1, -1, -1]], np.int32)
    masks = [0b1, 0b11, 0b101, 0b1, 0b11]
    positions = [37, 38, 38, 3, 4]
    slots = [table[0, p // page] * page + p % page for p in (37, 38, 39)] + [table[1, 0] * page + p for p in (3, 4)]
    pages, scales = ref.int8_cache(rng, 5, kv_heads, page, dim)
    qkv = rng.standard_normal((tokens, heads + 2 * kv_heads, dim)).astype(np.float16)
    logits = (rng.standard_normal((tokens, vocab)) * 3).astype(np.float32)
    drafted = rng.integers(0, vocab, tokens)
    i32 = lambda a: np.asarray(a, np.int32)  # noqa: E731
    for name, arr in (("pages", pages), ("scales", scales), ("qkv", qkv), ("slots", i32(slots)), ("positions", i32(positions)), ("starts", i32(starts)),
                      ("lengths", i32(lengths)), ("table", table), ("masks", np.array(masks, np.uint64)), ("logits", logits), ("drafted", i32(drafted))):
        arr.tofile(str(tmp_path / (name + ".bin")))
    (tmp_path / "meta.json").write_text(json.dumps({"tokens": tokens, "heads": heads, "kvHeads": kv_heads, "headDim": dim, "pageSize": page, "vocab": vocab,
                                                    "k": k, "sequences": 2, "maxQuery": 3, "maxKv": 40, "tableStride": 3}))
    r = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "verify_gpu.js"), str(tmp_path)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "js verify gpu ok" in r.stdout, r.stdout + r.stderr
    load = lambda name, kind: np.fromfile(str(tmp_path / (name + ".bin")), kind)  # noqa: E731
    freq, _ = capi.rope_frequencies(capi.ROPE_PLAIN, dim, 10000.0)
    want, norm = ref.rotated(qkv[:, :heads], positions, freq, dim, False, 1.0)
    q = load("q_out", np.float16).reshape(tokens, -1, dim)[:, :heads]
    assert ref.close_rotated(q, want, norm)
    cache = (load("pages_out", np.int8).reshape(pages.shape), load("scales_out", np.float16).reshape(scales.shape))
    rows = ref.rows_of(cache)
    for side, name in ((0, "k_out"), (1, "v_out")):
        got = load(name, np.float16).reshape(tokens, kv_heads, dim)
        for t, s in enumerate(slots):
            assert np.array_equal(got[t], rows[s // page, s % page, side].astype(np.float32).astype(np.float16))
    w = ref.attention(q, rows, page, table, starts, lengths, masks, float(np.float32(dim ** -0.5)), heads)
    ref.close_attention(load("attn", np.float16).reshape(tokens, heads, dim), load("lse", np.float32).reshape(tokens, heads), *w, dim, 40)
    logp, _, ids, _, _, top = ref.logprobs(logits, 1.0, drafted, k)
    assert ref.close_logp(load("lp", np.float32), logp, top, vocab) and np.array_equal(load("ids", np.uint32).reshape(tokens, k), ids)
