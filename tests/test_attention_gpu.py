"""GPU parity of attention over the paged cache (one token, chains, trees of drafted tokens; f16 and int8 rows), through
the C ABI, against float64."""
import numpy as np
import pytest

from . import verify_ref as ref
from .test_rope_append_gpu import f16_layout, int8_layout
from .util import Dev

pytestmark = pytest.mark.gpu


class Step:
    """One dispatch's inputs: sequences of (query tokens, cached keys), pages dealt at random."""

    def __init__(self, seed, heads, kv_heads, dim, page, work, int8=False, tree=None, mask_words=1, sharp=1.0, spare=2, q_pad=0, out_pad=0):
        rng = self.rng = np.random.default_rng(seed)
        self.heads, self.kv_heads, self.dim, self.page, self.int8, self.mask_words = heads, kv_heads, dim, page, int8, mask_words
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in work])]).astype(np.int64)
        self.lengths = [n for _, n in work]
        self.tokens = int(self.starts[-1])
        need = [-(-n // page) for n in self.lengths]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(work), max(max(need), 1)), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.cache = ref.int8_cache(rng, pages, kv_heads, page, dim) if int8 else ref.f16_cache(rng, pages, kv_heads, page, dim)
        self.q = (rng.standard_normal((self.tokens, heads, dim)) * sharp).astype(np.float16)
        self.scale = float(np.float32(dim ** -0.5))
        self.q_pad, self.out_pad = q_pad, out_pad
        self.masks = None
        if tree == "tree":
            self.masks = []
            for n, _ in work:
                mine = []
                for i in range(n):
                    up = int(rng.integers(max(0, i - 5), i)) if i else -1
                    mine.append((mine[up] if up >= 0 else 0) | 1 << i)
                self.masks += mine
        elif tree is not None:
            self.masks = list(tree)

    def want(self):
        return ref.attention(self.q, ref.rows_of(self.cache), self.page, self.table, self.starts, self.lengths, self.masks, self.scale, self.heads)

    def desc(self, ctx, capi, d, tokens_behind=0, max_query=None, max_kv=None, lse=True, no_table=False):
        tokens, width = self.tokens + tokens_behind, self.heads * self.dim
        wide = np.full((max(tokens, 1), width + self.q_pad), np.nan, np.float16)
        wide[:self.tokens, :width] = self.q.reshape(self.tokens, -1)
        if self.int8:
            c, s = self.cache
            cache = int8_layout(capi, self.kv_heads, self.dim, self.page, pages=d.put(c), pages_capacity=c.size // 4, scales=d.put(s), scales_capacity=s.size)
        else:
            c = self.cache
            cache = f16_layout(capi, self.kv_heads, self.dim, self.page, pages=d.put(c), pages_capacity=c.size)
        self.out_bytes, self.lse_bytes = max(tokens, 1) * (width + self.out_pad) * 2, max(tokens, 1) * self.heads * 4
        self.out = d.put(np.full((max(tokens, 1), width + self.out_pad), 7.0, np.float16))
        self.lse = d.put(np.full((max(tokens, 1), self.heads), 7.0, np.float32)) if lse else 0
        words = 0
        if self.masks is not None:
            words = np.zeros((max(tokens, 1), self.mask_words), np.uint64)
            for t, m in enumerate(self.masks):
                for w in range(self.mask_words):
                    words[t, w] = m >> 64 * w & (1 << 64) - 1
            words = d.put(words)
        n = np.diff(self.starts)
        return capi.AttentionDesc(tokens=tokens, sequences=len(self.lengths), heads=self.heads,
                                  max_query=int(n.max()) if max_query is None else max_query,
                                  max_kv=max(max(self.lengths), 0) if max_kv is None else max_kv, q_stride=width + self.q_pad,
                                  out_stride=width + self.out_pad, page_table_stride=0 if no_table else self.table.shape[1],
                                  mask_words=self.mask_words if words else 0, scale=self.scale, q=d.put(wide), out=self.out, lse=self.lse,
                                  query_start=d.put(self.starts.astype(np.int32)), kv_length=d.put(np.array(self.lengths, np.int32)),
                                  page_table=0 if no_table else d.put(self.table), tree_mask=words, cache=cache)

    def got(self, ctx):
        width = self.heads * self.dim
        out = ctx.download(self.out, self.out_bytes, np.float16).reshape(-1, width + self.out_pad)
        lse = ctx.download(self.lse, self.lse_bytes, np.float32).reshape(-1, self.heads) if self.lse else None
        return out, lse

    def check(self, ctx, capi, want=None, **kw):
        with Dev(ctx) as d:
            ctx.attention(self.desc(ctx, capi, d, **kw))
            out, lse = self.got(ctx)
        self.compare(out, lse, want)
        return out, lse

    def compare(self, out, lse, want=None):
        w = self.want() if want is None else want
        width = self.heads * self.dim
        assert np.all(out[:, width:] == 7.0), "the padding of out rows stays"
        assert np.all(out[self.tokens:] == 7.0) and (lse is None or np.all(lse[self.tokens:] == 7.0)), "rows behind the last sequence stay"
        ref.close_attention(out[:self.tokens, :width].reshape(self.tokens, self.heads, self.dim), None if lse is None else lse[:self.tokens], *w, self.dim,
                            max(max(self.lengths), 1))


SHAPES = [  # heads, kv_heads, dim, page
    (8, 2, 128, 16), (4, 4, 64, 16), (7, 1, 96, 16), (2, 2, 256, 16), (16, 1, 128, 16), (6, 2, 128, 5), (3, 3, 32, 64), (8, 8, 128, 16),
    (2, 1, 80, 16), (5, 5, 48, 16), (4, 2, 512, 16), (2, 1, 20, 16), (40, 2, 64, 1), (2, 2, 160, 16), (1, 1, 192, 16),
]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_one_token(ctx, capi, heads, kv_heads, dim, page, int8):
    """The decode step of a ragged batch, with lengths around every tile's and page's end."""
    lengths = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257, 300]
    Step(dim + heads, heads, kv_heads, dim, page, [(1, n) for n in lengths], int8, q_pad=8, out_pad=16).check(ctx, capi, tokens_behind=2)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_trees(ctx, capi, heads, kv_heads, dim, page, int8):
    """Ragged trees: sequences without tokens, trees without a history, all sizes up to a word."""
    work = [(5, 90), (0, 30), (1, 1), (9, 9), (17, 40), (64, 70), (33, 200), (2, 65)]
    Step(dim, heads, kv_heads, dim, page, work, int8, tree="tree").check(ctx, capi, tokens_behind=1)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (14, 2, 96), (2, 1, 256)])
def test_chains_and_chunks(ctx, capi, heads, kv_heads, dim, int8):
    """No mask: drafted chains and a prompt chunk of more tokens than a mask word holds."""
    Step(dim + 1, heads, kv_heads, dim, 16, [(150, 150), (3, 100), (70, 131), (1, 40)], int8).check(ctx, capi)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,work", [
    (8, 8, 128, [(1, 5003)]), (32, 8, 128, [(1, 3001), (1, 7)]), (8, 1, 64, [(3, 9000)]), (4, 2, 128, [(64, 4100)]), (6, 6, 96, [(20, 2500), (1, 2600)]),
    (2, 2, 256, [(5, 3000)])])
def test_long_contexts(ctx, capi, heads, kv_heads, dim, work, int8):
    """Work split over the keys and joined again."""
    Step(dim + 2, heads, kv_heads, dim, 16, work, int8, tree="tree", sharp=2.0).check(ctx, capi)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dim", [128, 96, 20])
def test_rows_that_see_nothing(ctx, capi, int8, dim):
    """Masks of zero without a history, a chain longer than its cache, no keys at all: zeros and lse = -inf."""
    masks = [0b1, 0, 0b111, 0] + [1, 0] + [0b01, 0b10]
    s = Step(5, 4, 2, dim, 16, [(4, 4), (2, 50), (2, 2)], int8, tree=masks)
    out, lse = s.check(ctx, capi)
    assert np.all(np.isneginf(lse[1])) and not out[1].any() and np.all(np.isneginf(lse[3])) and np.all(np.isfinite(lse[4:6]))
    s = Step(6, 4, 2, dim, 16, [(5, 2), (3, 0), (1, 0), (2, 2)], int8)      # tokens before position 0 see nothing
    out, lse = s.check(ctx, capi)
    assert np.all(np.isneginf(lse[:3])) and np.all(np.isfinite(lse[3:5])) and np.all(np.isneginf(lse[5:9]))


@pytest.mark.parametrize("dim,heads", [(128, 4), (96, 14), (20, 2)])
def test_infinities_in_masked_places(ctx, capi, dim, heads):
    """What unwritten slots, masked tokens and foreign pages hold never reaches a result."""
    for bad in (np.inf, -np.inf, np.nan, 65504.0):
        s = Step(7, heads, 2, dim, 16, [(6, 37), (3, 3), (1, 70)], tree="tree")
        used = np.zeros((s.cache.shape[0], 16), bool)
        for b, n in enumerate(s.lengths):
            for p in range(n):
                used[s.table[b, p // 16], p % 16] = True
        s.cache.transpose(0, 3, 1, 2, 4)[~used] = bad
        s.check(ctx, capi)
        # a drafted token that only some of the others see: theirs is the formula's value, the rest never meet it
        s = Step(8, heads, 2, dim, 16, [(6, 37)], tree=[0b1, 0b11, 0b101, 0b1001, 0b10001, 0b100001])
        want = s.want()
        page, slot = s.table[0, 33 // 16], 33 % 16                          # token 2 of the tree
        s.cache[page, :, :, slot] = bad
        with Dev(ctx) as d:
            ctx.attention(s.desc(ctx, capi, d))
            out, lse = s.got(ctx)
        keep = [0, 1, 3, 4, 5]
        ref.close_attention(out[keep].reshape(5, heads, dim), lse[keep], *(w[keep] for w in want), dim, 37)
        if bad != 65504.0:
            assert not np.all(np.isfinite(out[2].astype(np.float64)))


@pytest.mark.parametrize("dim,heads,queries", [(128, 4, 6), (96, 14, 6), (64, 16, 6), (128, 2, 40), (20, 2, 6)])
def test_scales_that_are_no_numbers_in_masked_places(ctx, capi, dim, heads, queries):
    for bad in (np.inf, np.nan, -np.inf):
        s = Step(23, heads, 2, dim, 16, [(queries, 70), (3, 3), (1, 33)], True, tree="tree")
        q, sc = s.cache
        used = np.zeros((sc.shape[0], 16), bool)
        for b, n in enumerate(s.lengths):
            for p in range(n):
                used[s.table[b, p // 16], p % 16] = True
        sc.transpose(0, 2, 1, 3)[~used] = bad
        s.check(ctx, capi)
        s = Step(24, heads, 2, dim, 16, [(6, 37)], True, tree=[0b1, 0b11, 0b101, 0b1001, 0b10001, 0b100001])
        want = s.want()
        page, slot = s.table[0, 33 // 16], 33 % 16                          # token 2 of the tree
        s.cache[1][page, :, slot] = bad
        with Dev(ctx) as d:
            ctx.attention(s.desc(ctx, capi, d))
            out, lse = s.got(ctx)
        keep = [0, 1, 3, 4, 5]
        ref.close_attention(out[keep].reshape(5, heads, dim), lse[keep], *(w[keep] for w in want), dim, 37)
        if np.isnan(bad):                                                   # an infinite score may be one of probability zero
            assert not np.all(np.isfinite(out[2].astype(np.float64)))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dim", [128, 64, 20])
def test_bad_pages_and_lengths(ctx, capi, int8, dim):
    """Page numbers outside the cache hide their keys; lengths past the bounds, negative lengths and starts past the
    tokens are cut; nothing faults."""
    s = Step(9, 4, 2, dim, 16, [(3, 100), (2, 60)], int8, tree="tree")
    pages = ref.rows_of(s.cache).shape[0]
    s.table[0, 1], s.table[0, 3], s.table[1, 0], s.table[1, 2] = -1, pages, 2 ** 31 - 1, -2 ** 31
    s.check(ctx, capi)
    # a page that is only partly inside the capacity is outside
    s = Step(10, 4, 2, dim, 16, [(1, 64)], int8, spare=0)
    with Dev(ctx) as d:
        desc = s.desc(ctx, capi, d)
        desc.cache.pages_capacity -= 1
        ctx.attention(desc)
        out, lse = s.got(ctx)
    last = s.cache[0].shape[0] - 1 if int8 else s.cache.shape[0] - 1
    s.table[s.table == last] = -1
    s.compare(out, lse)
    # a length past max_kv is cut there, a negative one is none
    s = Step(11, 4, 2, dim, 16, [(1, 50), (1, 90), (1, 30)], int8)
    with Dev(ctx) as d:
        desc = s.desc(ctx, capi, d, max_kv=64)
        desc.kv_length = d.put(np.array([50, 10 ** 9, -3], np.int32))
        ctx.attention(desc)
        out, lse = s.got(ctx)
    s.lengths = [50, 64, 0]
    s.compare(out, lse)
    # tokens past max_query are not written, starts past the tokens name nothing
    s = Step(12, 4, 2, dim, 16, [(5, 40), (2, 20)], int8)
    with Dev(ctx) as d:
        desc = s.desc(ctx, capi, d, max_query=3)
        ctx.attention(desc)
        out, lse = s.got(ctx)
    w = s.want()
    keep = [0, 1, 2, 5, 6]
    ref.close_attention(out[keep].reshape(5, 4, dim), lse[keep], *(x[keep] for x in w), dim, 40)
    assert np.all(out[3:5] == 7.0) and np.all(lse[3:5] == 7.0)
    with Dev(ctx) as d:
        desc = s.desc(ctx, capi, d)
        desc.tokens = 6
        desc.query_start = d.put(np.array([0, 5, 10 ** 9], np.int32))
        desc.max_query = 5
        ctx.attention(desc)
        out, _ = s.got(ctx)
    assert np.all(out[6] == 7.0) and np.all(np.isfinite(out.astype(np.float32)))


def test_wide_masks(ctx, capi):
    """Trees of more than 64 tokens: several words a token."""
    Step(13, 4, 2, 128, 16, [(150, 190), (70, 70), (1, 9)], tree="tree", mask_words=3).check(ctx, capi)
    Step(14, 2, 2, 64, 16, [(100, 400)], True, tree="tree", mask_words=2).check(ctx, capi)


@pytest.mark.parametrize("int8", [False, True])
def test_one_sequence_without_a_table(ctx, capi, int8):
    s = Step(15, 8, 2, 128, 16, [(4, 77)], int8)
    s.table[0] = np.arange(s.table.shape[1])
    out, lse = s.check(ctx, capi, no_table=True)
    again, lse2 = s.check(ctx, capi)
    assert np.array_equal(out.view(np.uint16), again.view(np.uint16)) and np.array_equal(lse, lse2)
    s.check(ctx, capi, lse=False)


def test_order_of_pages_and_batch_do_not_matter(ctx, capi):
    """The same keys in other pages give the same bits, and a sequence gives the same bits in any company of equal
    bounds; launch after launch as well."""
    s = Step(16, 8, 2, 128, 16, [(9, 500), (9, 700), (9, 300)], tree="tree")
    a, la = s.check(ctx, capi)
    perm = np.random.default_rng(1).permutation(s.cache.shape[0])
    inv = np.argsort(perm)
    s.cache = np.ascontiguousarray(s.cache[perm])
    s.table = np.where(s.table >= 0, inv[np.maximum(s.table, 0)], -1).astype(np.int32)
    b, lb = s.check(ctx, capi)
    assert np.array_equal(a.view(np.uint16), b.view(np.uint16)) and np.array_equal(la, lb)
    for _ in range(3):
        c, lc = s.check(ctx, capi)
        assert np.array_equal(a.view(np.uint16), c.view(np.uint16)) and np.array_equal(la, lc)


def test_extreme_scores(ctx, capi):
    """Scores of hundreds, a negative and a zero scale, equal scores: the running maximum holds."""
    s = Step(17, 4, 2, 128, 16, [(5, 600)], tree="tree", sharp=60.0)
    s.check(ctx, capi)
    s.scale = -s.scale
    s.check(ctx, capi)
    s.scale = 0.0
    s.check(ctx, capi)


def test_huge_values_in_int8(ctx, capi):
    """Scales whose rows reach f16's largest values: the folded probabilities stay finite."""
    s = Step(18, 4, 2, 128, 16, [(3, 100)], True)
    q, sc = s.cache
    sc[..., 1] = np.float16(500.0)
    s.check(ctx, capi)
    sc[..., 1] = np.float16(6e-8)
    s.check(ctx, capi)


def test_offsets_past_32_bits(ctx, capi):
    """A cache of more than 4 GiB, and more than 2^32 elements of it: only the pages used are written."""
    heads, kv_heads, dim, page = 4, 1, 128, 16
    kps = 1 << 22                                            # a page every 8 MiB
    n = 1100
    s = Step(19, heads, kv_heads, dim, page, [(2, 60)])
    with Dev(ctx) as d:
        big = d.empty(n * kps * 2)
        pages = [3, 1099, 700, 513]
        desc = s.desc(ctx, capi, d)
        for i, p in enumerate(pages):
            ctx.upload(big, s.cache[s.table[0, i]], p * kps * 2)
        desc.cache.pages, desc.cache.pages_capacity, desc.cache.kv_page_stride = big, n * kps, kps
        desc.page_table = d.put(np.array([pages], np.int32))
        ctx.attention(desc)
        out, lse = s.got(ctx)
        s.compare(out, lse)
        # and stored there
        x = np.random.default_rng(0).standard_normal((1, 3, dim)).astype(np.float16)
        freq, _ = capi.rope_frequencies(capi.ROPE_PLAIN, dim, 10000.0)
        q = d.empty(dim * 2)
        one = capi.RopeAppendDesc(tokens=1, heads=1, rotary_dim=dim, qkv_stride=3 * dim, q_stride=dim, attn_factor=1.0, qkv=d.put(x), q_out=q,
                                  frequencies=d.put(freq), positions=d.put(np.array([0], np.int32)),
                                  slots=d.put(np.array([1099 * page + 15], np.int32)), cache=desc.cache)
        ctx.rope_append(one)
        k, v = d.empty(dim * 2), d.empty(dim * 2)
        ctx.kv_read(capi.KvReadDesc(tokens=1, out_stride=dim, k_out=k, v_out=v, slots=one.slots, cache=desc.cache))
        assert np.array_equal(ctx.download(k, dim * 2, np.float16), x[0, 1]) and np.array_equal(ctx.download(v, dim * 2, np.float16), x[0, 2])


def test_recorded_steps(ctx, capi):
    """A recorded dispatch replayed for growing lengths, with eager work of another shape between the replays."""
    s = Step(20, 8, 2, 128, 16, [(4, 900), (4, 1100)], tree="tree")
    other = Step(21, 32, 8, 64, 16, [(1, 3000), (2, 100)])
    with Dev(ctx) as d:
        desc = s.desc(ctx, capi, d)
        ctx.attention(desc)                                  # the scratch grows outside the recording
        ctx.record_begin()
        ctx.attention(desc)
        cb = ctx.record_end()
        try:
            for lengths in ([900, 1100], [4, 5], [333, 1100], [900, 17]):
                ctx.upload(desc.kv_length, np.array(lengths, np.int32))
                ctx.fill(s.out, 0x55, s.out_bytes)
                ctx.submit(cb)
                out, lse = s.got(ctx)
                s.lengths = lengths
                s.compare(out, lse)
                other.check(ctx, capi)
                ctx.attention(desc)
                eager, elase = s.got(ctx)
                assert np.array_equal(out.view(np.uint16), eager.view(np.uint16)) and np.array_equal(lse, elase)
        finally:
            ctx.cmdbuf_destroy(cb)


@pytest.mark.parametrize("int8", [False, True])
def test_loose_bounds(ctx, capi, int8):
    """Bounds far past what there is change neither results nor, in size, the scratch."""
    s = Step(25, 8, 2, 128, 16, [(3, 200), (1, 60)], int8, tree="tree", mask_words=1)
    s.table = np.concatenate([s.table, np.full((2, 4096), -1, np.int32)], 1)
    s.check(ctx, capi, max_kv=65536)
    s = Step(26, 8, 2, 128, 16, [(3, 200), (1, 60)], int8)
    s.check(ctx, capi, max_query=(1 << 30) - 1)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (16, 1, 64), (4, 1, 256), (3, 3, 20)])
def test_more_queries_than_keys(ctx, capi, heads, kv_heads, dim, int8):
    """The first tokens of such a sequence see nothing, over several row tiles."""
    Step(29, heads, kv_heads, dim, 16, [(100, 30), (70, 70), (40, 0), (5, 300)], int8).check(ctx, capi)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("queries", [1, 5, 12, 40])
@pytest.mark.parametrize("page", [32, 48, 256, 1024])
def test_page_sizes(ctx, capi, page, queries, int8):
    Step(page + queries, 8, 2, 128, page, [(queries, 700), (queries, 1025), (queries, 48)], int8, tree="tree").check(ctx, capi)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("queries", [1, 5, 12, 40])
def test_negative_and_zero_scales(ctx, capi, queries, int8):
    s = Step(30, 8, 2, 128, 16, [(queries, 700), (queries, 130)], int8)
    for scale in (-0.125, 0.0):
        s.scale = scale
        s.check(ctx, capi)


@pytest.mark.parametrize("dim", [128, 20])
@pytest.mark.parametrize("bound", [1, 7, 30])
def test_queries_past_the_bound_stay(ctx, capi, bound, dim):
    s = Step(31, 8, 2, dim, 16, [(40, 200), (3, 90)])
    with Dev(ctx) as d:
        ctx.attention(s.desc(ctx, capi, d, max_query=bound))
        out, lse = s.got(ctx)
    width = s.heads * s.dim
    written = np.array([t - s.starts[b] < bound for b in range(2) for t in range(s.starts[b], s.starts[b + 1])])
    assert np.all(out[~written] == 7.0) and np.all(lse[~written] == 7.0)
    want, want_lse, *rest = s.want()
    ref.close_attention(out[written].reshape(-1, s.heads, s.dim), lse[written], want[written], want_lse[written], *[r[written] for r in rest], s.dim, 200)


def test_recordings_that_share_the_scratch(ctx, capi):
    """Two recorded steps of one context, replayed in turn with eager calls between them."""
    a, b = Step(32, 8, 2, 128, 16, [(1, 4000), (1, 3000)]), Step(33, 8, 2, 128, 16, [(40, 2500), (12, 3999)], True, tree="tree")
    c = Step(34, 16, 2, 64, 16, [(4, 5000)])
    with Dev(ctx) as da, Dev(ctx) as db, Dev(ctx) as dc:
        x, y, z = a.desc(ctx, capi, da), b.desc(ctx, capi, db), c.desc(ctx, capi, dc)
        recorded = []
        for step in (x, y):
            ctx.attention(step)                              # the scratch grows outside the recording
            ctx.record_begin()
            ctx.attention(step)
            recorded.append(ctx.record_end())
        for _ in range(4):
            for step in (a, b, c):
                ctx.upload(step.out, np.full(step.out_bytes // 2, 7.0, np.float16))
                ctx.upload(step.lse, np.full(step.lse_bytes // 4, 7.0, np.float32))
            ctx.submit(recorded[0])
            ctx.submit(recorded[1])
            ctx.attention(z)
            ctx.submit(recorded[0])
            ctx.sync()
            for step in (a, b, c):
                step.compare(*step.got(ctx))
        for r in recorded:
            ctx.cmdbuf_destroy(r)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dim", [32, 160, 192, 224])
@pytest.mark.parametrize("queries", [1, 6, 40])
def test_other_head_sizes(ctx, capi, dim, queries, int8):
    """Heads of a multiple of 32, in every shape of workgroup, over one part of the keys and many."""
    Step(dim + queries, 8, 2, dim, 16, [(queries, 2100), (queries, 300), (queries, 47)], int8, tree="tree").check(ctx, capi)


@pytest.mark.parametrize("dim,queries", [(32, 5), (160, 5), (192, 5), (160, 40)])
def test_infinities_in_masked_places_of_other_head_sizes(ctx, capi, dim, queries):
    s = Step(dim, 4, 2, dim, 16, [(queries, 100)])
    for page in range(s.cache.shape[0]):
        if page not in s.table[0, :7]:
            s.cache[page] = np.inf
    s.cache[s.table[0, 6], :, :, 4:] = np.nan           # behind the last position
    s.check(ctx, capi)


def test_two_contexts_at_once(ctx, capi):
    """Two contexts on one GPU, their dispatches in flight together: scratch and counters are each one's own."""
    a, b = Step(27, 8, 2, 128, 16, [(1, 4000), (1, 3000)]), Step(28, 8, 2, 128, 16, [(1, 2500), (1, 3999)])
    other = capi.Context(0)
    try:
        with Dev(ctx) as da, Dev(other) as db:
            x, y = a.desc(ctx, capi, da), b.desc(other, capi, db)
            for _ in range(20):
                ctx.attention(x)
                other.attention(y)
            a.compare(*a.got(ctx))
            b.compare(*b.got(other))
    finally:
        other.close()


def test_nothing_to_do(ctx, capi):
    s = Step(22, 4, 2, 64, 16, [(2, 20)])
    with Dev(ctx) as d:
        for change in (dict(tokens=0), dict(sequences=0), dict(max_query=0)):
            desc = s.desc(ctx, capi, d)
            for k, v in change.items():
                setattr(desc, k, v)
            ctx.attention(desc)
            out, _ = s.got(ctx)
            assert np.all(out == 7.0)
