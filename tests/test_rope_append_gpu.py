"""GPU parity of the rotary append (Q rotated, K and V into the paged f16 or int8 cache) and of the cache read-back,
through the C ABI, against float64."""
import numpy as np
import pytest

from . import verify_ref as ref
from .util import Dev

pytestmark = pytest.mark.gpu


def f16_layout(capi, kv_heads, dim, page, **kw):
    hps = page * dim
    return capi.KvCache(**{**dict(format=capi.KV_F16, kv_heads=kv_heads, head_dim=dim, page_size=page, head_page_stride=hps,
                                  v_page_offset=kv_heads * hps, kv_page_stride=2 * kv_heads * hps), **kw})


def int8_layout(capi, kv_heads, dim, page, **kw):
    return capi.KvCache(**{**dict(format=capi.KV_INT8, kv_heads=kv_heads, head_dim=dim, page_size=page), **kw})


def freq_of(capi, rotary, theta=10000.0):
    return capi.rope_frequencies(capi.ROPE_PLAIN, rotary, theta)


def rope(ctx, capi, d, x, heads, cache, positions, slots, rotary, interleaved, freq, factor=1.0, qkv_stride=None, q_stride=None,
         q_fill=None):
    """x [tokens, heads + 2 kv, dim] -> q rows as stored [tokens, q_stride]"""
    tokens, rows, dim = x.shape
    qkv_stride, q_stride = qkv_stride or rows * dim, q_stride or heads * dim
    wide = np.full((tokens, qkv_stride), np.nan, np.float16)
    wide[:, :rows * dim] = x.reshape(tokens, -1)
    q = d.put(np.full((tokens, q_stride), 7.0, np.float16))
    ctx.rope_append(capi.RopeAppendDesc(tokens=tokens, heads=heads, rotary_dim=rotary, interleaved=int(interleaved), qkv_stride=qkv_stride,
                                        q_stride=q_stride, attn_factor=factor, qkv=d.put(wide), q_out=q, frequencies=d.put(freq),
                                        positions=d.put(np.asarray(positions, np.int32)), slots=d.put(np.asarray(slots, np.int32)), cache=cache))
    return ctx.download(q, tokens * q_stride * 2, np.float16).reshape(tokens, q_stride)


CASES = [  # tokens, heads, kv_heads, dim, page, rotary, interleaved, qkv padding, q padding
    (1, 32, 8, 128, 16, 128, False, 0, 0),      # a decode step
    (1, 4, 4, 64, 16, 64, True, 0, 0),
    (5, 7, 1, 96, 16, 96, False, 0, 0),         # six lanes of a group of eight
    (9, 6, 2, 128, 16, 64, True, 8, 16),        # part of the head, padded rows
    (9, 6, 2, 128, 16, 32, False, 8, 16),
    (3, 2, 1, 256, 7, 256, False, 0, 0),        # a page size that is no power of two
    (4, 3, 3, 512, 4, 128, True, 0, 0),
    (2, 2, 2, 16, 16, 16, False, 0, 0),
    (6, 2, 1, 32, 16, 32, True, 0, 0),
    (5, 3, 1, 80, 16, 40, False, 0, 0),         # a rotary part off 16: pair by pair
    (5, 3, 1, 100, 16, 100, True, 0, 0),        # a head off 16
    (3, 2, 2, 128, 16, 128, False, 3, 5),       # row strides off 16 bytes
    (1100, 8, 2, 64, 16, 64, False, 0, 0),      # a workgroup takes a whole token
]


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,page,rotary,interleaved,pad,q_pad", CASES)
def test_f16(ctx, capi, tokens, heads, kv_heads, dim, page, rotary, interleaved, pad, q_pad):
    rng = np.random.default_rng(tokens * 1000 + dim)
    pages = tokens // page + 3
    x = rng.standard_normal((tokens, heads + 2 * kv_heads, dim)).astype(np.float16)
    positions = rng.integers(0, 100000, tokens)
    slots = rng.permutation(pages * page)[:tokens]
    if tokens > 2:
        slots[1] = -1
    freq, _ = freq_of(capi, rotary)
    cache0 = ref.f16_cache(rng, pages, kv_heads, page, dim)
    with Dev(ctx) as d:
        kv = d.put(cache0)
        cache = f16_layout(capi, kv_heads, dim, page, pages=kv, pages_capacity=cache0.size)
        q = rope(ctx, capi, d, x, heads, cache, positions, slots, rotary, interleaved, freq, 1.25, (heads + 2 * kv_heads) * dim + pad,
                 heads * dim + q_pad)
        got = ctx.download(kv, cache0.nbytes, np.float16).reshape(cache0.shape)
    want, norm = ref.rotated(x[:, :heads + kv_heads], positions, freq, rotary, interleaved, 1.25)
    assert np.all(q[:, heads * dim:] == 7.0), "the padding of q rows stays"
    assert ref.close_rotated(q[:, :heads * dim].reshape(tokens, heads, dim), want[:, :heads], norm[:, :heads])
    left = np.ones((pages, page), bool)
    for t, s in enumerate(slots):
        if s < 0:
            continue
        left[s // page, s % page] = False
        assert ref.close_rotated(got[s // page, 0, :, s % page], want[t, heads:], norm[t, heads:])
        assert np.array_equal(got[s // page, 1, :, s % page], x[t, heads + kv_heads:]), "V is stored as it is"
        assert np.array_equal(got[s // page, 0, :, s % page, rotary:], x[t, heads:heads + kv_heads, rotary:]), "past the rotary part"
    rest = lambda a: a.transpose(0, 3, 1, 2, 4)[left]  # noqa: E731
    assert np.array_equal(rest(got).view(np.uint16), rest(cache0).view(np.uint16)), "the rest of the cache is untouched"


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,page,rotary,interleaved,pad,q_pad", [c for c in CASES if c[3] % 4 == 0])
def test_int8_equals_the_two_dispatches(ctx, capi, tokens, heads, kv_heads, dim, page, rotary, interleaved, pad, q_pad):
    """Rows stored as int8 are the f16 rows put through ztvm_kv_quantize_int8, bit for bit; Q is the same."""
    rng = np.random.default_rng(tokens * 1000 + dim + 1)
    pages = tokens // page + 3
    x = (rng.standard_normal((tokens, heads + 2 * kv_heads, dim)) * 3).astype(np.float16)
    x[0, heads:heads + 1] = 0                           # a row of zeros: the least scale
    positions = rng.integers(0, 100000, tokens)
    slots = rng.permutation(pages * page)[:tokens]
    if tokens > 2:
        slots[1] = -1
    freq, _ = freq_of(capi, rotary)
    q0, s0 = ref.int8_cache(rng, pages, kv_heads, page, dim)
    f0 = ref.f16_cache(rng, pages, kv_heads, page, dim)
    with Dev(ctx) as d:
        kv, pg, sc = d.put(f0), d.put(q0), d.put(s0)
        args = (positions, slots, rotary, interleaved, freq, 1.0, (heads + 2 * kv_heads) * dim + pad, heads * dim + q_pad)
        qa = rope(ctx, capi, d, x, heads, f16_layout(capi, kv_heads, dim, page, pages=kv, pages_capacity=f0.size), *args)
        qb = rope(ctx, capi, d, x, heads, int8_layout(capi, kv_heads, dim, page, pages=pg, pages_capacity=q0.size // 4, scales=sc,
                                                     scales_capacity=s0.size), *args)
        f16 = ctx.download(kv, f0.nbytes, np.float16).reshape(f0.shape)
        got_q, got_s = ctx.download(pg, q0.nbytes, np.int8).reshape(q0.shape), ctx.download(sc, s0.nbytes, np.uint16).reshape(s0.shape)
        keep = [t for t in range(tokens) if slots[t] >= 0]
        at = np.asarray(slots)[keep]
        k, v = (np.ascontiguousarray(f16[at // page, side, :, at % page]) for side in (0, 1))
        pg2, sc2 = d.put(q0), d.put(s0)
        ctx.kv_quantize_int8(capi.KvQuantizeDesc(kv_heads=kv_heads, head_dim=dim, page_size=page, tokens=len(keep), pages_capacity_words=q0.size // 4,
                                                 scales_capacity=s0.size, k_slot=d.put(k), v_slot=d.put(v), pages_i8=pg2, scales=sc2,
                                                 position_map=d.put(at.astype(np.int32))))
        want_q, want_s = ctx.download(pg2, q0.nbytes, np.int8).reshape(q0.shape), ctx.download(sc2, s0.nbytes, np.uint16).reshape(s0.shape)
    assert np.array_equal(qa.view(np.uint16), qb.view(np.uint16))
    assert np.array_equal(got_s, want_s)
    assert np.array_equal(got_q, want_q)
    assert not np.array_equal(got_q, q0)


@pytest.mark.parametrize("position", [131071, 2 ** 31 - 1, -5])
def test_far_positions_keep_their_angle(ctx, capi, position):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, 4, 128)).astype(np.float16)
    freq, _ = freq_of(capi, 128, 500000.0)
    f0 = np.zeros((1, 2, 1, 16, 128), np.float16)
    with Dev(ctx) as d:
        kv = d.put(f0)
        q = rope(ctx, capi, d, x, 2, f16_layout(capi, 1, 128, 16, pages=kv, pages_capacity=f0.size), [position], [3], 128, False, freq)
    want, norm = ref.rotated(x, [position], freq, 128, False, 1.0)
    assert ref.close_rotated(q.reshape(1, 2, 128), want[:, :2], norm[:, :2])


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dim", [64, 100])
def test_slots_outside_the_cache_store_nothing(ctx, capi, int8, dim):
    """Negative slots, pages past the capacity, and a page that is only partly inside."""
    rng = np.random.default_rng(2)
    kv_heads, heads, page = 2, 2, 8
    bad = [-1, -2 ** 31, 3 * page, 3 * page + 5, 4 * page, 2 ** 31 - 1]
    x = rng.standard_normal((len(bad), heads + 2 * kv_heads, dim)).astype(np.float16)
    freq, _ = freq_of(capi, dim)
    with Dev(ctx) as d:
        if int8:
            q0, s0 = ref.int8_cache(rng, 4, kv_heads, page, dim)
            pg, sc = d.put(q0), d.put(s0)
            cache = int8_layout(capi, kv_heads, dim, page, pages=pg, pages_capacity=q0.size // 4 - 1, scales=sc, scales_capacity=s0.size)
        else:
            q0, s0 = ref.f16_cache(rng, 4, kv_heads, page, dim), np.zeros(8, np.float16)
            pg, sc = d.put(q0), d.put(s0)
            cache = f16_layout(capi, kv_heads, dim, page, pages=pg, pages_capacity=q0.size - 1)
        q = rope(ctx, capi, d, x, heads, cache, np.arange(len(bad)), bad, dim, False, freq)
        assert np.array_equal(ctx.download(pg, q0.nbytes, np.uint8), q0.reshape(-1).view(np.uint8))
        assert np.array_equal(ctx.download(sc, s0.nbytes, np.uint16), s0.reshape(-1).view(np.uint16))
        k = d.put(np.full((len(bad), kv_heads * dim), 5.0, np.float16))
        ctx.kv_read(capi.KvReadDesc(tokens=len(bad), out_stride=kv_heads * dim, k_out=k, slots=d.put(np.array(bad, np.int32)), cache=cache))
        assert np.all(ctx.download(k, len(bad) * kv_heads * dim * 2, np.float16) == 5.0), "rows of such slots stay as they were"
    want, norm = ref.rotated(x, np.arange(len(bad)), freq, dim, False, 1.0)
    assert ref.close_rotated(q.reshape(len(bad), heads, dim), want[:, :heads], norm[:, :heads]), "Q is written all the same"


@pytest.mark.parametrize("dim,stride", [(128, 10 * 128), (100, 10 * 100 + 2)])
def test_in_place_and_offsets(ctx, capi, dim, stride):
    """q_out = qkv, and a cache that starts inside its buffer, with wider page and head strides."""
    rng = np.random.default_rng(3)
    heads, kv_heads, page, tokens = 4, 3, 4, 6
    x = rng.standard_normal((tokens, heads + 2 * kv_heads, dim)).astype(np.float16)
    wide = np.zeros((tokens, stride), np.float16)
    wide[:, :x[0].size] = x.reshape(tokens, -1)
    positions, slots = np.arange(tokens) * 7, np.array([0, 5, 9, 2, 11, 7])
    freq, _ = freq_of(capi, dim)
    hps, vpo = page * dim + 8, 3 * (page * dim + 8) + 16
    kps, off = vpo + 3 * hps + 24, 40
    f0 = rng.standard_normal(off + 3 * kps).astype(np.float16)
    with Dev(ctx) as d:
        buf, kv = d.put(wide), d.put(f0)
        cache = capi.KvCache(format=capi.KV_F16, kv_heads=kv_heads, head_dim=dim, page_size=page, head_page_stride=hps, v_page_offset=vpo,
                             kv_page_stride=kps, pages_offset=off, pages=kv, pages_capacity=f0.size)
        ctx.rope_append(capi.RopeAppendDesc(tokens=tokens, heads=heads, rotary_dim=dim, qkv_stride=stride, q_stride=stride, attn_factor=1.0,
                                            qkv=buf, q_out=buf, frequencies=d.put(freq), positions=d.put(positions.astype(np.int32)),
                                            slots=d.put(slots.astype(np.int32)), cache=cache))
        got = ctx.download(buf, wide.nbytes, np.float16).reshape(wide.shape)
        flat = ctx.download(kv, f0.nbytes, np.float16)
        k, v = d.empty(tokens * kv_heads * dim * 2), d.empty(tokens * kv_heads * dim * 2)
        ctx.kv_read(capi.KvReadDesc(tokens=tokens, out_stride=kv_heads * dim, k_out=k, v_out=v, slots=d.put(slots.astype(np.int32)), cache=cache))
        k = ctx.download(k, tokens * kv_heads * dim * 2, np.float16).reshape(tokens, kv_heads, dim)
        v = ctx.download(v, tokens * kv_heads * dim * 2, np.float16).reshape(tokens, kv_heads, dim)
    want, norm = ref.rotated(x[:, :heads + kv_heads], positions, freq, dim, False, 1.0)
    assert ref.close_rotated(got[:, :heads * dim].reshape(tokens, heads, dim), want[:, :heads], norm[:, :heads])
    assert np.array_equal(got[:, heads * dim:], wide[:, heads * dim:])
    touched = np.zeros(f0.size, bool)
    for t, s in enumerate(slots):
        for h in range(kv_heads):
            at = off + s // page * kps + h * hps + s % page * dim
            assert ref.close_rotated(flat[at:at + dim], want[t, heads + h], norm[t, heads + h])
            assert np.array_equal(flat[at + vpo:at + vpo + dim], x[t, heads + kv_heads + h])
            assert np.array_equal(k[t, h], flat[at:at + dim]) and np.array_equal(v[t, h], flat[at + vpo:at + vpo + dim])
            touched[at:at + dim] = touched[at + vpo:at + vpo + dim] = True
    assert np.array_equal(flat[~touched].view(np.uint16), f0[~touched].view(np.uint16))


@pytest.mark.parametrize("kv_heads,dim,page,tokens,pad", [(8, 128, 16, 45, 0), (3, 96, 16, 7, 8), (1, 256, 5, 1, 0), (2, 20, 16, 9, 0),
                                                          (2, 64, 16, 11, 3), (5, 12, 3, 4, 0), (1, 512, 16, 2000, 0)])
def test_read_back_int8(ctx, capi, kv_heads, dim, page, tokens, pad):
    rng = np.random.default_rng(dim)
    pages = tokens // page + 2
    q0, s0 = ref.int8_cache(rng, pages, kv_heads, page, dim)
    slots = rng.integers(0, pages * page, tokens)          # a slot may be read twice
    slots[tokens // 2] = -1 if tokens > 1 else slots[0]
    stride, n = kv_heads * dim + pad, tokens * (kv_heads * dim + pad)
    with Dev(ctx) as d:
        off_w, off_s = 12, 6
        pg = d.put(np.concatenate([np.zeros(off_w * 4, np.int8), q0.reshape(-1)]))
        sc = d.put(np.concatenate([np.zeros(off_s, np.float16), s0.reshape(-1)]))
        k, v = d.put(np.full(n, 5.0, np.float16)), d.put(np.full(n, 5.0, np.float16))
        ctx.kv_read(capi.KvReadDesc(tokens=tokens, out_stride=stride, k_out=k, v_out=v, slots=d.put(slots.astype(np.int32)),
                                    cache=int8_layout(capi, kv_heads, dim, page, pages=pg, scales=sc, pages_offset=off_w, scales_offset=off_s,
                                                      pages_capacity=q0.size // 4 + off_w, scales_capacity=s0.size + off_s)))
        got = [ctx.download(a, n * 2, np.float16).reshape(tokens, stride) for a in (k, v)]
    rows = (q0.astype(np.float32) * s0.astype(np.float32)[..., None]).astype(np.float16).transpose(0, 2, 3, 1, 4).reshape(pages * page, 2, -1)
    for side in (0, 1):
        want = np.full((tokens, stride), 5.0, np.float16)
        want[slots >= 0, :kv_heads * dim] = rows[slots[slots >= 0], side]
        assert np.array_equal(got[side].view(np.uint16), want.view(np.uint16))


def test_no_tokens(ctx, capi):
    cache = f16_layout(capi, 1, 64, 16, pages=0x10000, pages_capacity=1 << 20)
    ctx.rope_append(capi.RopeAppendDesc(tokens=0, heads=1, rotary_dim=64, qkv_stride=192, q_stride=64, attn_factor=1.0, qkv=0x1000, q_out=0x2000,
                                        frequencies=0x3000, positions=0x4000, slots=0x5000, cache=cache))
    ctx.kv_read(capi.KvReadDesc(tokens=0, out_stride=64, k_out=0x1000, slots=0x2000, cache=cache))
