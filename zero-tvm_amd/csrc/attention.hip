// Attention of the query tokens of several sequences over the paged cache.
#include "internal.h"
#include "kv_cache.h"
#include "mma.h"
#include "quant.h"

#include <algorithm>
#include <type_traits>

namespace ztvm {
namespace {

// The sequence a query row belongs to: the last one that starts at or before it.
__device__ __forceinline__ bool find_sequence(const AttentionArgs& p, int32_t t, uint32_t& b, int32_t& i, int32_t& n) {
  uint32_t lo = 0, hi = p.sequences;  // start[lo] <= t < start[hi] is what the search keeps, where it holds at all
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (p.query_start[mid] <= t) lo = mid;
    else hi = mid;
  }
  b = lo;
  const int32_t start = p.query_start[lo], end = p.query_start[lo + 1];
  i = t - start;
  n = end - start;
  return t >= start && t < end && i < (int32_t)p.max_query;
}

// One workgroup per query row and head, a key per thread and turn, an online softmax over tiles of 256 keys.
constexpr uint32_t ANY_MAX_DIM = 512;
__global__ __launch_bounds__(256) void attention_any_kernel(const AttentionArgs p) {
  __shared__ float q[ANY_MAX_DIM], red[256], prob[256];
  __shared__ uint32_t key_page[256], key_slot[256];
  const uint32_t t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  uint32_t b;
  int32_t i, n;
  if (!find_sequence(p, (int32_t)t, b, i, n)) return;
  const KvView& c = p.cache;
  const uint32_t dim = c.head_dim, kvh = h / (p.heads / c.kv_heads);
  const int32_t cached = max(p.kv_length[b], 0), length = min(cached, (int32_t)p.max_kv);
  const int64_t context = (int64_t)cached - n;  // by all that is cached: the bound hides positions and moves none
  for (uint32_t d = tid; d < dim; d += 256u) q[d] = (float)p.q[(size_t)t * p.q_stride + (size_t)h * dim + d];
  // the product: `groups` groups of threads share the keys of a tile, a thread takes dims d0, d0 + 256
  uint32_t width = 1;
  while (width < dim && width < 256u) width *= 2;
  const uint32_t groups = 256u / width, group = tid / width, d0 = tid % width;
  float acc[2] = {0.f, 0.f};
  float m = -INFINITY, total = 0.f;
  for (int32_t k0 = 0; k0 < length; k0 += 256) {
    const int32_t pos = k0 + (int32_t)tid;
    bool seen = pos < length;
    uint32_t page = 0, slot = 0;
    if (seen) {
      const int64_t rel = (int64_t)pos - context;
      if (p.tree_mask) seen = rel < 0 || (rel < 64ll * p.mask_words && (p.tree_mask[(size_t)t * p.mask_words + rel / 64] >> (rel & 63) & 1));
      else seen = rel <= i;
      const uint32_t pno = fast_div(c.by_page, (uint32_t)pos);
      slot = (uint32_t)pos - pno * c.page_size;
      page = p.page_table ? (uint32_t)p.page_table[(size_t)b * p.page_table_stride + pno] : pno;
      seen = seen && page < c.num_pages;
    }
    __syncthreads();  // the last tile's probabilities have been read, q is there
    float s = -INFINITY;
    if (seen) {
      const char* row = c.pages + kv_row_offset(c, page, kvh, slot, 0);
      float dot = 0.f;
      if (c.int8) {
        for (uint32_t d = 0; d < dim; d++) dot = __builtin_fmaf(q[d], (float)reinterpret_cast<const int8_t*>(row)[d], dot);
        dot *= (float)__builtin_bit_cast(_Float16, c.scales[kv_scale_index(c, page, kvh, slot, 0)]);
      } else {
        for (uint32_t d = 0; d < dim; d++) dot = __builtin_fmaf(q[d], (float)reinterpret_cast<const _Float16*>(row)[d], dot);
      }
      s = dot * p.scale;
    }
    key_page[tid] = page;
    key_slot[tid] = slot;
    red[tid] = s != s ? INFINITY : s;  // a NaN score of a key that is seen must not be lost in the maximum
    __syncthreads();
    for (uint32_t o = 128; o > 0; o >>= 1) {
      if (tid < o) red[tid] = fmaxf(red[tid], red[tid + o]);
      __syncthreads();
    }
    const float m_new = fmaxf(m, red[0]);
    __syncthreads();
    if (m_new == -INFINITY) continue;  // nothing seen so far
    const float pr = seen ? expf(s - m_new) : 0.f;
    prob[tid] = pr;
    red[tid] = pr;
    __syncthreads();
    for (uint32_t o = 128; o > 0; o >>= 1) {
      if (tid < o) red[tid] += red[tid + o];
      __syncthreads();
    }
    const float keep = expf(m - m_new);
    total = total * keep + red[0];
    m = m_new;
    acc[0] *= keep;
    acc[1] *= keep;
    const uint32_t keys = min(256, length - k0);
    for (uint32_t k = group; k < keys; k += groups) {
      const float w = prob[k];
      if (w == 0.f) continue;  // a masked key's values never enter, whatever they are
      const char* row = c.pages + kv_row_offset(c, key_page[k], kvh, key_slot[k], 1);
      const float ws = c.int8 ? w * (float)__builtin_bit_cast(_Float16, c.scales[kv_scale_index(c, key_page[k], kvh, key_slot[k], 1)]) : w;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const uint32_t d = d0 + 256u * j;
        if (d < dim) acc[j] = __builtin_fmaf(ws, c.int8 ? (float)reinterpret_cast<const int8_t*>(row)[d] : (float)reinterpret_cast<const _Float16*>(row)[d], acc[j]);
      }
    }
  }
  // add the groups' sums in their order
  for (int j = 0; j < 2; j++) {
    __syncthreads();
    red[tid] = acc[j];
    __syncthreads();
    const uint32_t d = d0 + 256u * j;
    if (group == 0 && d < dim) {
      float sum = 0.f;
      for (uint32_t g = 0; g < groups; g++) sum += red[g * width + d0];
      p.out[(size_t)t * p.out_stride + (size_t)h * dim + d] = narrow_f32(m == -INFINITY ? 0.f : sum / total);
    }
  }
  if (tid == 0 && p.lse) p.lse[(size_t)t * p.heads + h] = m == -INFINITY ? -INFINITY : m + logf(total);
}

// ------------------------------------------------------------------------------- the matrix-core kernel ----
// A workgroup takes one sequence, one kv head, ROWS = 16*QT*RW query rows (row = token * group + head of the group) and
// one chunk of the keys. RW waves share keys and split the rows, KW waves share rows and split the keys.
//
//   S^T = K Q^T   v_mfma_f32_16x16x32: A = 16 keys x 32 dims straight from the staged rows, B = the query rows, kept in
//                 registers. Lane (c = lane/16, j = lane%16) then holds query j, keys 4c..4c+3 of each 16-key tile.
//   O^T += V^T P  B = the probabilities exactly where the first product left them: k index (c, e) means key
//                 16*(e/4) + 4c + e%4. A = 16 dims x 32 keys with the same meaning, which is what the transposing LDS
//                 reads deliver from rows of V as they lie in the cache (ds_read_b64_tr_b16 takes 4 keys x 16 dims a
//                 group of 16 lanes, ds_read_b64_tr_b8 8 keys x 16 dims), so nothing is shuffled between the products.
//
// The running maximum is lazy: a row's reference value moves only when what enters the second product passes CAP, so most
// tiles need no exchange between lanes and no rescaling. Probabilities are lifted by 2^LIFT before they round to f16, which
// keeps those within 2^-23 of the largest out of its subnormal range. int8 keys' scales multiply the scores, int8 values'
// scales the probabilities. Where the values are widened once for several waves, the scale's power of two goes into them
// (exact) and the rest, 1 to 2, into the probabilities. Where a wave widens its own, the whole scale goes into the
// probabilities and the reference follows their products: it is the largest score plus log2 of its key's scale, so that the
// products use f16's range however small the values are. The f32 sum of the probabilities has range for that: they are at
// most 2^24 times CAP.
//
// Keys and values travel global -> LDS without passing registers, 32 keys a wave and stage, 16-byte chunks XOR-swizzled
// so that neither kind of read meets bank conflicts. A page holds a multiple of 16 slots here, so 16 keys always lie in
// one page and their addresses are one scalar base and a constant per lane. int8 rows that four waves share are fetched
// into registers instead and widened once for all, 64 keys a turn (transfers and 32 keys: 98 us for the trees below, 77).
//
// Measured: 48 tokens of 32 heads over 90 to 8191 f16 keys of 8 x 128, 815 MB: 156 us, 5.2 TB/s, bound by memory, as is a
// tree of 64 over 65537 keys of 16 x 96 (403 MB, 85 us). 16 trees of 5 to 61 over 200 to 4500 int8 keys of 8 x 128 (87 MB,
// 21 GFLOP): 77 us, bound by the issue of vector instructions: 480 a wave and turn beside 64 matrix instructions. A token
// over 1037 keys: 8.9 us, a chain of dependent steps.

// chunk swizzles. A row of `KD` 64-byte units starts at bank slot 4*KD*row mod 16 (16 slots of 16 bytes): the XOR supplies
// the row bits that the pitch does not.
template <int KD>
__device__ __forceinline__ constexpr uint32_t swz_k(uint32_t row) {
  return KD % 4 == 0 ? row & 15u : KD % 2 == 0 ? (row >> 1) & 7u : (row >> 2) & 3u;
}
template <int KD>
__device__ __forceinline__ constexpr uint32_t swz_v(uint32_t row) {  // pairs of chunks over eight rows
  return KD % 4 == 0 ? (row & 7u) << 1 : KD % 2 == 0 ? ((row >> 1) & 3u) << 1 : ((row >> 2) & 1u) << 1;
}
template <int KD>
__device__ __forceinline__ constexpr uint32_t swz_i8(uint32_t row) {  // the 8-bit transposing read takes rows r and r + 16 together
  return swz_k<KD>(row) ^ ((row >> 4) << (KD % 4 == 0 ? 3 : KD % 2 == 0 ? 2 : 1));
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(4))) int32_t* const_i32;
typedef int i32x2 __attribute__((ext_vector_type(2)));

struct MfmaParams {
  AttentionArgs a;
  float* partial;   // [sequence][head][row of max_query tokens][split][dim], times 2^LIFT
  float2* partial_ml;  // reference value (log2) and sum, times 2^LIFT
  uint32_t* arrivals;  // of the workgroups that split a row tile, one counter each, zero between launches; null: a launch of its own joins
  uint32_t splits, chunk, group;
  float scale_log2;  // |scale| * log2 e
  uint32_t negate;   // scale < 0: the queries change sign
};

constexpr float LIFT = 9.f, CAP = 32768.f;  // log2; what enters the second product is LIFT above the reference and at most CAP
constexpr float LEAST_SCALE = 0x1p-24f;     // of f16: what a value scale of zero counts as where the reference is found
constexpr int MOST_SPLITS = 128, FUSED_SPLITS = 16;
constexpr float NOTHING = -3.0e38f;  // a row's reference value before its first key

__device__ __forceinline__ float across_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float across_groups_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// eight signed bytes -> eight f16, exactly: the byte with its sign bit flipped goes under 1024's exponent
__device__ __forceinline__ h8 widen_i8(u32x2 w) {
  const uint32_t a = w.x ^ 0x80808080u, b = w.y ^ 0x80808080u;
  const h2 bias = {(_Float16)1152.f, (_Float16)1152.f};
  const h2 r0 = as_h2(__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - bias;
  const h2 r1 = as_h2(__builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - bias;
  const h2 r2 = as_h2(__builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - bias;
  const h2 r3 = as_h2(__builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - bias;
  return h8{r0.x, r0.y, r1.x, r1.y, r2.x, r2.y, r3.x, r3.y};
}

// 2^s nearest to an f16 scale from below, with s in -13..9 so that 127 * 2^s and 2^s are f16 numbers; 1 for what is no number
__device__ __forceinline__ _Float16 power_of(uint16_t scale) {
  uint32_t e = scale >> 10 & 31u;
  e = e == 31u ? 15u : min(max(e, 2u), 24u);
  return __builtin_bit_cast(_Float16, (uint16_t)(e << 10));
}

// Which of the keys k0 .. k0+63 a query token sees: bit j. `limit`: the first position it cannot see in any case; words: its
// mask, null without a tree.
__device__ __forceinline__ uint64_t visible_bits(int64_t k0, int64_t context, int64_t limit, const uint64_t* words, uint32_t mask_words) {
  const int64_t left = limit - k0;
  uint64_t bits = left <= 0 ? 0ull : left >= 64 ? ~0ull : (1ull << left) - 1ull;
  if (words && bits) {
    const int64_t rel = k0 - context;  // bit of the first key; below zero: history
    if (rel < 0) {
      if (rel > -64) bits &= words[0] << -rel | ((1ull << -rel) - 1ull);
    } else {
      const uint64_t w = (uint64_t)rel >> 6;
      const uint32_t b = (uint32_t)rel & 63u;
      uint64_t v = (w < mask_words ? words[w] : 0ull) >> b;
      if (b && w + 1 < mask_words) v |= words[w + 1] << (64u - b);
      bits &= v;
    }
  }
  return bits;
}

// an address that is the same in all lanes, in scalar registers
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return reinterpret_cast<const char*>((uint64_t)hi << 32 | lo);
}

// NS: 32-key tiles that a wave takes a turn
template <int KD, bool INT8, int QT, int RW, int KW, int NS>
struct MfmaShape {
  static constexpr int DIM = 32 * KD;
  static constexpr int ROWS = 16 * QT * RW;
  // three where four waves meet at a barrier; two for heads past 128, so that two workgroups fit a CU (48 x 2 rows over 9000
  // keys 44.2 -> 31.8 us)
  static constexpr int STAGES = RW == 1 || KD > 4 ? 2 : 3;
  static constexpr int KEYS = 32 * NS;
  static constexpr int PART = 32 * DIM * (INT8 ? 2 : 4);  // bytes of 32 keys as they arrive: K then V (int8: rows of K | V)
  static constexpr int SCALES = INT8 ? 256 : 0;
  static constexpr int STAGE = KW * (PART + SCALES);
  static constexpr bool WIDEN = INT8 && RW > 1;            // int8 rows become f16 once for all waves
  static constexpr int PAIRS = KEYS * DIM * 4;             // in a widened tile: K, V, then the scales of each as f32,
  static constexpr int FLAGS = PAIRS + KEYS * 8;           // then which of its 16-key blocks are inside the cache
  static constexpr int WIDE = WIDEN ? FLAGS + 16 : 0;
  static_assert(WIDEN || NS == 1, "only the widened tiles are made of several");
  static_assert(!WIDEN || (RW == 4 && NS == 2), "a wave widens one 16-key block");
  static constexpr int PITCH = DIM + 4;                    // of the joined rows
  static constexpr int JOIN = KW > 1 ? std::max(KW * ROWS * PITCH * 4 + KW * ROWS * 8, ROWS * FUSED_SPLITS * 8) : 0;
  static constexpr int LDS = std::max(WIDEN ? 2 * WIDE : STAGES * STAGE, JOIN);
};

// two floats past the caches that are not shared by all of the device, in one access
__device__ __forceinline__ void put2(float* to, float x, float y) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(to), __builtin_bit_cast(uint64_t, make_float2(x, y)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* from) {
  return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

template <int KD, bool INT8, int QT, int RW, int KW, int NS>
__global__ __launch_bounds__(64 * RW * KW, KD > 4 ? 1 : RW > 1 && QT == 1 && NS == 1 ? 4 : 2) void attention_mfma_kernel(const MfmaParams p) {
  using Shape = MfmaShape<KD, INT8, QT, RW, KW, NS>;
  constexpr int DIM = Shape::DIM, ROWS = Shape::ROWS, ST = Shape::STAGES, KEYS = Shape::KEYS;
  constexpr bool RAW8 = INT8 && !Shape::WIDEN;
  constexpr int MOVES = INT8 ? KD * 2 : KD * 4;     // transfers of 1 KiB that bring 32 keys
  constexpr int MOVES_EACH = (MOVES + RW - 1) / RW;  // of which a wave makes so many (the last one twice where they do not share evenly)
  constexpr int DMA = MOVES_EACH + (INT8 ? 1 : 0);   // and the scales
  extern __shared__ __align__(16) char lds[];
  const AttentionArgs& a = p.a;
  const KvView& c = a.cache;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t rw = wave % RW, kw = wave / RW;
  const uint32_t lc = lane >> 4, lj = lane & 15u;

  uint32_t id = blockIdx.x;
  const uint32_t h = id % c.kv_heads;
  id /= c.kv_heads;
  const uint32_t b = id % a.sequences, split = id / a.sequences;
  const int32_t start = a.query_start[b];
  const int64_t n = (int64_t)a.query_start[b + 1] - start;
  // tokens of this sequence that exist and are asked for
  const int64_t tokens = min(min(n, (int64_t)a.max_query), (int64_t)a.tokens - start);
  const uint32_t row0 = blockIdx.y * ROWS;
  if (start < 0 || tokens <= 0 || row0 >= tokens * p.group) return;
  const uint32_t rows = (uint32_t)tokens * p.group;
  const int32_t cached = max(a.kv_length[b], 0), length = min(cached, (int32_t)a.max_kv);
  const int64_t context = cached - n;  // by all that is cached: the bound hides positions and moves none
  const bool tree = a.tree_mask != nullptr;
  const uint32_t last_row = min(row0 + ROWS, rows) - 1;
  const int64_t seen_by_all = tree ? context : context + row0 / p.group + 1;
  const int64_t seen_by_any = tree ? length : context + last_row / p.group + 1;
  const int32_t k_last = (int32_t)max(min(seen_by_any, (int64_t)length), (int64_t)0);
  const int32_t full = (int32_t)max(min(seen_by_all, (int64_t)length), (int64_t)0);  // keys below: every row sees them
  const uint32_t parts = max(1u, ((uint32_t)k_last + p.chunk - 1) / p.chunk);  // splits that have keys (one writes the empty rows)
  if (split >= parts) return;
  const int32_t k_begin = (int32_t)(split * p.chunk), k_end = min(k_last, k_begin + (int32_t)p.chunk);
  const int32_t turns = (k_end - k_begin + KEYS * KW - 1) / (KEYS * KW);

  // ---- the query rows, as B operands
  const uint32_t wave_row = row0 + rw * 16 * QT;
  h8 q[QT][KD];
  int32_t limit[QT];   // first position the lane's row cannot see
  uint32_t token[QT];  // whose mask it goes by
#pragma unroll
  for (int t = 0; t < QT; t++) {
    const uint32_t row = wave_row + 16 * t + lj, i = row / p.group;
    const bool there = row < rows;
    const _Float16* src = a.q + (size_t)(start + (there ? i : 0u)) * a.q_stride + (size_t)(h * p.group + (there ? row - i * p.group : 0u)) * DIM;
    limit[t] = there ? (tree ? length : (int32_t)max(min((int64_t)length, context + i + 1), (int64_t)0)) : 0;
    token[t] = start + (there ? i : 0u);
#pragma unroll
    for (int s = 0; s < KD; s++) {
      u32x4 v = *reinterpret_cast<const u32x4*>(src + 32 * s + 8 * lc);
      if (p.negate) v ^= 0x80008000u;
      if (!there) v = u32x4{0, 0, 0, 0};
      q[t][s] = __builtin_bit_cast(h8, v);
    }
  }

  // ---- transfers: the lane's constant part of each address
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  // KD transfers move 16 rows of one side (f16) or of both (int8, K | V). Transfer g of the MOVES that bring 32 keys:
  // f16: K of keys 0-15, of 16-31, then V; int8: keys 0-15, 16-31. A wave makes those of its turn among the RW.
  uint32_t voff[MOVES_EACH];
#pragma unroll
  for (int i = 0; i < MOVES_EACH; i++) {
    const uint32_t g = min((uint32_t)i * RW + rw, MOVES - 1u), within = g % (2 * KD);
    const uint32_t idx = within * 64 + lane, row = idx / (4 * KD), ch = idx - row * (4 * KD);
    const uint32_t swz = INT8 ? swz_i8<KD>(row) : g < 2 * KD ? swz_k<KD>(row) : swz_v<KD>(row);
    voff[i] = (row & 15u) * (2 * DIM) + ((ch ^ swz) * 16);
  }
  const char* head_base = c.pages + (uint64_t)h * c.head_bytes;
  // Page numbers come through the scalar cache (the constant address space makes the compiler load them so): a vector
  // load here would have to wait for every transfer in flight.
  const const_i32 table = (const_i32)(uintptr_t)(a.page_table ? a.page_table + (size_t)b * a.page_table_stride : nullptr);
  struct Block {  // 16 keys
    uint32_t page, slot;
    bool inside;
  };
  auto block_at = [&](int32_t pos) {
    Block x;
    const uint32_t at = (uint32_t)min(pos, k_end - 1);  // always a position there is
    const uint32_t pno = fast_div(c.by_page, at);
    x.slot = (at - pno * c.page_size) & ~15u;
    x.page = table ? (uint32_t)table[pno] : pno;
    x.inside = pos < k_end;
    return x;
  };
  auto settle_block = [&](Block& x) {  // some rows that exist where the page is none; nobody sees them
    x.inside = x.inside && x.page < c.num_pages;
    if (!x.inside) x.page = x.slot = 0;
  };
  auto base_of = [&](const Block& x) { return uniform(head_base + (uint64_t)x.page * c.page_bytes + (uint64_t)x.slot * c.slot_bytes); };
  auto key_of = [&](int32_t turn) { return k_begin + KEYS * (int32_t)(kw + KW * turn); };
  // starts the transfers of a turn's 32 keys; returns which halves are inside the cache
  auto issue = [&](Block x0, Block x1, uint32_t stage) -> uint32_t {
    settle_block(x0);
    settle_block(x1);
    const uint32_t at = lds_base + stage * Shape::STAGE + kw * Shape::PART;
    const char* base0 = base_of(x0);
    const char* base1 = base_of(x1);
    static_for<MOVES_EACH>([&](auto i_) {
      constexpr int i = decltype(i_)::value;
      const uint32_t g = min((uint32_t)i * RW + rw, MOVES - 1u);
      const char* base = g / KD % 2 ? base1 : base0;
      if (!INT8 && g >= 2 * KD) base += c.side_bytes;
      dma16<0>(base, voff[i], at + 1024u * g);
    });
    if constexpr (INT8) {  // a pair of scales for each key (lanes 32..63 repeat them)
      const uint32_t key = lane & 31u;
      const uint64_t s0 = kv_scale_index(c, x0.page, h, x0.slot, 0), s1 = kv_scale_index(c, x1.page, h, x1.slot, 0);
      dma4(reinterpret_cast<const char*>(c.scales + (key < 16 ? s0 : s1)) + 4u * (key & 15u), lds_base + stage * Shape::STAGE + KW * Shape::PART + kw * Shape::SCALES);
    }
    return (x0.inside ? 1u : 0u) | (x1.inside ? 2u : 0u);
  };

  f4 acc[QT][2 * KD];
  float m[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; t++) {
    m[t] = NOTHING;
    l[t] = 0.f;
#pragma unroll
    for (int d = 0; d < 2 * KD; d++) acc[t][d] = f4{0.f, 0.f, 0.f, 0.f};
  }

  // where a lane reads: its part of the addresses (a 16-row half and a stage are constants on top)
  uint32_t k_at[KD], v_at[2 * KD];
#pragma unroll
  for (int x = 0; x < KD; x++) {
    if constexpr (RAW8) k_at[x] = lj * (2 * DIM) + (((2 * x + (lc >> 1)) ^ swz_i8<KD>(lj)) * 16) + (lc & 1u) * 8;
    else k_at[x] = lj * (2 * DIM) + (((4 * x + lc) ^ swz_k<KD>(lj)) * 16);
  }
#pragma unroll
  for (int d = 0; d < 2 * KD; d++) {
    if constexpr (RAW8) {
      const uint32_t row = 16 * (lj >> 3) + 4 * lc + ((lj >> 1) & 3u);
      v_at[d] = row * (2 * DIM) + (((2 * KD + d) ^ swz_i8<KD>(row)) * 16) + (lj & 1u) * 8;
    } else {
      const uint32_t row = 4 * lc + (lj >> 2);
      v_at[d] = 2 * KEYS * DIM + row * (2 * DIM) + (((2 * d + ((lj & 3u) >> 1)) ^ swz_v<KD>(row)) * 16) + (lj & 1u) * 8;
    }
  }

  // One tile of KEYS keys. kv: the staged rows (f16, or int8 as they came); pairs: their scales; inside: which 16-key
  // blocks are in the cache.
  auto compute = [&](int32_t turn, uint32_t at, uint32_t pairs_at, uint32_t inside) {
    constexpr int H = 2 * NS;  // 16-key blocks
    const int32_t pos = key_of(turn);
    if (pos >= k_end) return;
    const char* kv = lds + at;
    const char* pairs = lds + at + pairs_at;
    const bool edge = pos + KEYS > full || inside != (1u << H) - 1u;  // some row does not see some key
    f4 s[QT][H];
#pragma unroll
    for (int t = 0; t < QT; t++)
#pragma unroll
      for (int half = 0; half < H; half++) s[t][half] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < KD; x++)
      static_for<H>([&](auto half_) {
        constexpr int half = decltype(half_)::value;
        h8 k;
        if constexpr (RAW8) {  // 8 bytes: half of a chunk
          constexpr uint32_t FLIP = 16u * (swz_i8<KD>(16));
          k = widen_i8(*reinterpret_cast<const u32x2*>(kv + (half ? (k_at[x] ^ FLIP) + 32 * DIM : k_at[x])));
        } else {
          k = *reinterpret_cast<const h8*>(kv + k_at[x] + half * 32 * DIM);
        }
#pragma unroll
        for (int t = 0; t < QT; t++) s[t][half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[t][x], s[t][half], 0, 0, 0);
      });
    // int8: the keys' scales
    auto scale_of = [&](int half, bool value, float* out) {  // of the lane's four keys of a block
      if constexpr (RAW8) {
        const u32x4 four = *reinterpret_cast<const u32x4*>(pairs + 64 * half + 16 * lc);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const h2 pair = as_h2(four[i]);
          out[i] = value ? (float)pair.y : (float)pair.x * p.scale_log2;
        }
      } else {
        const f4 four = *reinterpret_cast<const f4*>(pairs + (value ? 4 * KEYS : 0) + 64 * half + 16 * lc);
#pragma unroll
        for (int i = 0; i < 4; i++) out[i] = four[i];
      }
    };
    if constexpr (INT8) {
#pragma unroll
      for (int half = 0; half < H; half++) {
        float ks[4];
        scale_of(half, false, ks);
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) s[t][half][i] *= ks[i];
      }
    }
    const float units = INT8 ? 1.f : p.scale_log2;  // s * units: the scores in log2 units
    uint64_t there = ~0ull;
    if (edge) {
      there = 0;
#pragma unroll
      for (int half = 0; half < H; half++) there |= inside >> half & 1u ? 0xFFFFull << (16 * half) : 0ull;
    }
    // int8: a scale that is no number (of a slot nobody wrote, say) must not enter as 0 * inf where it is not seen
    uint32_t odd = 0;
    if constexpr (INT8) {
      if (edge) {
        bool any = false;
#pragma unroll
        for (int half = 0; half < H; half++) {
          float vs[4];
          scale_of(half, true, vs);
#pragma unroll
          for (int i = 0; i < 4; i++) any |= !(fabsf(vs[i]) <= 65504.f);
        }
        odd = __any(any) ? 1u : 0u;
      }
      odd = __builtin_amdgcn_readfirstlane(odd);
      asm volatile("" : "+s"(odd));  // a condition of its own: tied to `edge` the compiler doubles the code behind it
    }
    float raw[RAW8 ? H : 1][4], size[RAW8 ? H : 1][4];  // the value scales and their magnitudes within f16's numbers but zero
    if constexpr (RAW8) {
#pragma unroll
      for (int half = 0; half < H; half++) {
        scale_of(half, true, raw[half]);
#pragma unroll
        for (int i = 0; i < 4; i++) size[half][i] = fminf(fmaxf(fabsf(raw[half][i]), LEAST_SCALE), 65504.f);
      }
    }
    h8 pf[QT][NS];
#pragma unroll
    for (int t = 0; t < QT; t++) {
      uint32_t seen[NS];  // bit 16*half + i of a 32-key part: the lane's row sees key 16*half + 4*lc + i of it
      if (edge) {
        const uint64_t bits = visible_bits(pos, context, limit[t], tree ? a.tree_mask + (size_t)token[t] * a.mask_words : nullptr, a.mask_words) & there;
#pragma unroll
        for (int n = 0; n < NS; n++) seen[n] = (uint32_t)(bits >> (32 * n)) >> (4 * lc);
      }
      auto sees = [&](int half, int i) { return (seen[half / 2] >> (16 * (half & 1) + i) & 1u) != 0; };
      // probabilities against the reference value as it stands; where one of them passes CAP the reference moves and they
      // are taken again
      float e[H][4];
      auto weigh = [&]() {
        const float down = m[t] - LIFT;
#pragma unroll
        for (int half = 0; half < H; half++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            e[half][i] = __builtin_amdgcn_exp2f(INT8 ? s[t][half][i] - down : __builtin_fmaf(s[t][half][i], units, -down));
        if (edge) {
#pragma unroll
          for (int half = 0; half < H; half++)
#pragma unroll
            for (int i = 0; i < 4; i++) e[half][i] = sees(half, i) ? e[half][i] : 0.f;
        }
      };
      weigh();
      float most = 0.f;
#pragma unroll
      for (int half = 0; half < H; half++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if constexpr (RAW8) most = fmaxf(most, e[half][i] * size[half][i]);
          else most = fmaxf(most, e[half][i]);
        }
      if (__any(most > CAP)) {
        float top = -INFINITY;
#pragma unroll
        for (int half = 0; half < H; half++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float x = s[t][half][i] * units;
            if constexpr (RAW8) x += __builtin_amdgcn_logf(size[half][i]);
            top = fmaxf(top, !edge || sees(half, i) ? x : -INFINITY);
          }
        const float next = fmaxf(m[t], across_groups_max(top));
        const float keep = __builtin_amdgcn_exp2f(m[t] - next);
        m[t] = next;
        l[t] *= keep;
#pragma unroll
        for (int d = 0; d < 2 * KD; d++) acc[t][d] *= keep;
        weigh();
      }
#pragma unroll
      for (int half = 0; half < H; half++) {
        float vs[4] = {1.f, 1.f, 1.f, 1.f};
        if constexpr (Shape::WIDEN) scale_of(half, true, vs);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if constexpr (RAW8) vs[i] = raw[half][i];
          l[t] += e[half][i];
          pf[t][half / 2][4 * (half & 1) + i] = (_Float16)(INT8 ? e[half][i] * vs[i] : e[half][i]);
        }
      }
      if (INT8 && odd) {
#pragma unroll
        for (int half = 0; half < H; half++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (!sees(half, i)) pf[t][half / 2][4 * (half & 1) + i] = (_Float16)0.f;
      }
    }
#pragma unroll
    for (int d = 0; d < 2 * KD; d++) {
#pragma unroll
      for (int n = 0; n < NS; n++) {
        h8 v;
        if constexpr (RAW8) {
          const i32x2 raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(kv + v_at[d]));
          v = widen_i8(u32x2{(uint32_t)raw.x, (uint32_t)raw.y});
        } else {
          s16x4 r[2];
#pragma unroll
          for (int half = 0; half < 2; half++)
            r[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(kv + v_at[d] + (2 * n + half) * 32 * DIM));
          v = __builtin_bit_cast(h8, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
        if (!INT8 && edge) {
          // An infinity or NaN that nobody sees must not enter as 0 * inf: the product gets a zero, and rows that do
          // see it get it back by its sign.
          u16x8 bits = __builtin_bit_cast(u16x8, v);
          h8 up, down;
          bool odd = false;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const uint32_t e = bits[i];
            const bool bad = (e & 0x7C00u) == 0x7C00u, nan = (e & 0x3FFu) != 0;
            up[i] = bad && (nan || !(e & 0x8000u)) ? (_Float16)1.f : (_Float16)0.f;
            down[i] = bad && (nan || (e & 0x8000u)) ? (_Float16)1.f : (_Float16)0.f;
            bits[i] = bad ? 0 : e;
            odd |= bad;
          }
          v = __builtin_bit_cast(h8, bits);
          if (__any(odd)) {
#pragma unroll
            for (int t = 0; t < QT; t++) {
              h8 sees;
#pragma unroll
              for (int i = 0; i < 8; i++) sees[i] = pf[t][n][i] > (_Float16)0.f ? (_Float16)1.f : (_Float16)0.f;
              const f4 zero = {0.f, 0.f, 0.f, 0.f};
              const f4 ups = __builtin_amdgcn_mfma_f32_16x16x32_f16(up, sees, zero, 0, 0, 0);
              const f4 downs = __builtin_amdgcn_mfma_f32_16x16x32_f16(down, sees, zero, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; i++) {
                if (ups[i] > 0.f) acc[t][d][i] += INFINITY;
                if (downs[i] > 0.f) acc[t][d][i] -= INFINITY;
              }
            }
          }
        }
#pragma unroll
        for (int t = 0; t < QT; t++) acc[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[t][n], acc[t][d], 0, 0, 0);
      }
    }
  };

  // ---- the pipeline
  uint32_t halves = 0;  // two bits for each stage in flight, the oldest lowest
  if constexpr (RW == 1) {  // a wave's keys are its own: no barrier; a stage is filled again as soon as it has been used
#pragma unroll
    for (int i = 0; i < KD; i++) k_at[i] += kw * Shape::PART;
#pragma unroll
    for (int i = 0; i < 2 * KD; i++) v_at[i] += kw * Shape::PART;
#pragma unroll
    for (int i = 0; i < ST; i++)
      if (i < turns) halves |= issue(block_at(key_of(i)), block_at(key_of(i) + 16), i) << (2 * i);
    for (int32_t turn = 0; turn < turns; turn++) {
      const uint32_t stage = turn % ST;
      const Block x0 = block_at(key_of(turn + ST)), x1 = block_at(key_of(turn + ST) + 16);
      if (turn + ST - 1 < turns) wait_vm<(ST - 1) * DMA>();
      else wait_vm<0>();
      compute(turn, stage * Shape::STAGE, KW * Shape::PART + kw * Shape::SCALES, halves & 3u);
      halves >>= 2;
      wait_lgkm<0>();
      if (turn + ST < turns) halves |= issue(x0, x1, stage) << (2 * (ST - 1));
    }
  } else if constexpr (!Shape::WIDEN) {
#pragma unroll
    for (int i = 0; i < ST - 1; i++)
      if (i < turns) halves |= issue(block_at(key_of(i)), block_at(key_of(i) + 16), i) << (2 * i);
    for (int32_t turn = 0; turn < turns; turn++) {
      const Block x0 = block_at(key_of(turn + ST - 1)), x1 = block_at(key_of(turn + ST - 1) + 16);
      if (turn + ST - 2 < turns) wait_vm<(ST - 2) * DMA>();
      else wait_vm<0>();
      wg_barrier();  // everybody's transfers of this stage have landed, everybody has left the stage before
      if (turn + ST - 1 < turns) halves |= issue(x0, x1, (turn + ST - 1) % ST) << (2 * (ST - 1));
      compute(turn, turn % ST * Shape::STAGE, 0u, halves & 3u);
      halves >>= 2;
      wait_lgkm<0>();
    }
  } else {
    // int8 rows that several waves share: each wave fetches its part of a tile into registers a turn ahead and widens it
    // for all, so the products read f16 tiles.
    constexpr uint32_t SIDE = 32 * KD;                      // 16-byte chunks of K (and of V) in the wave's 16 keys
    constexpr int LOADS = KD;                               // 64 chunks each: K, then V (KD odd: the middle one holds both)
    uint32_t from[LOADS], to_at[LOADS], key[LOADS];
    bool is_v[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
      const uint32_t u = 64 * i + lane;
      is_v[i] = KD % 2 == 0 ? i >= KD / 2 : u >= SIDE;
      const uint32_t w = is_v[i] ? u - SIDE : u, row = w / (2 * KD), ch = w - row * (2 * KD);
      key[i] = row;
      from[i] = row * (2 * DIM) + (is_v[i] ? DIM : 0) + ch * 16;
      const uint32_t swz = is_v[i] ? swz_v<KD>(row) : swz_k<KD>(row);
      to_at[i] = (is_v[i] ? 2 * KEYS * DIM : 0) + (16 * rw + row) * (2 * DIM) + ((2 * ch) ^ swz) * 16;
    }
    u32x4 raw[LOADS];
    uint32_t pair;  // of key lane % 16
    bool have;
    auto fetch = [&](Block x) {
      settle_block(x);
      have = x.inside;
      const char* base = base_of(x);
      const char* scales = uniform(reinterpret_cast<const char*>(c.scales + kv_scale_index(c, x.page, h, x.slot, 0)));
#pragma unroll
      for (int i = 0; i < LOADS; i++) raw[i] = *reinterpret_cast<const u32x4*>(base + from[i]);
      pair = *reinterpret_cast<const uint32_t*>(scales + 4u * lj);
    };
    auto widen = [&](int32_t turn) {
      char* to = lds + (turn & 1) * Shape::WIDE;
      const h2 scales = as_h2(pair);
      const _Float16 sv = scales.y, power = power_of(__builtin_bit_cast(uint16_t, sv));
      if (lane < 16) {
        *reinterpret_cast<float*>(to + Shape::PAIRS + 4 * (16 * rw + lane)) = (float)scales.x * p.scale_log2;
        *reinterpret_cast<float*>(to + Shape::PAIRS + 4 * (KEYS + 16 * rw + lane)) = (float)sv / (float)power;
      }
      if (lane == 0) *reinterpret_cast<uint32_t*>(to + Shape::FLAGS + 4 * rw) = have ? 1u << rw : 0u;
      const int power_bits = (int)as_u32(h2{power, power});
#pragma unroll
      for (int i = 0; i < LOADS; i++) {
        h8 lo = widen_i8(u32x2{raw[i].x, raw[i].y}), hi = widen_i8(u32x2{raw[i].z, raw[i].w});
        if (KD % 2 != 0 || i >= KD / 2) {
          h2 f = as_h2((uint32_t)__builtin_amdgcn_ds_bpermute((int)(4 * key[i]), power_bits));
          if (KD % 2 != 0 && !is_v[i]) f = h2{(_Float16)1.f, (_Float16)1.f};
          lo *= h8{f.x, f.x, f.x, f.x, f.x, f.x, f.x, f.x};
          hi *= h8{f.x, f.x, f.x, f.x, f.x, f.x, f.x, f.x};
        }
        *reinterpret_cast<h8*>(to + to_at[i]) = lo;
        *reinterpret_cast<h8*>(to + (to_at[i] ^ 16u)) = hi;
      }
    };
    if (turns) {
      auto block_of = [&](int32_t turn) { return block_at(key_of(turn) + 16 * (int32_t)rw); };
      fetch(block_of(0));
      Block ahead = block_of(1);
      widen(0);
      fetch(ahead);
      ahead = block_of(2);
      for (int32_t turn = 0; turn < turns; turn++) {
        wait_lgkm<0>();
        wg_barrier();  // this tile is widened; everybody has left the one before
        if (turn + 1 < turns) widen(turn + 1);
        fetch(ahead);  // past the end: rows that exist, not looked at
        ahead = block_of(turn + 3);
        const u32x4 flags = *reinterpret_cast<const u32x4*>(lds + (turn & 1) * Shape::WIDE + Shape::FLAGS);
        compute(turn, (turn & 1) * Shape::WIDE, Shape::PAIRS, __builtin_amdgcn_readfirstlane(flags.x | flags.y | flags.z | flags.w));
      }
    }
  }

  // ---- join the key waves, then either the result or a partial one
#pragma unroll
  for (int t = 0; t < QT; t++) l[t] = across_groups_sum(l[t]);
  auto finish4 = [&](uint32_t row, uint32_t d, f4 v, float total) {  // four dims of a row; v and total are times 2^LIFT
    const uint32_t i = row / p.group;
    const float inv = total > 0.f || total != total ? 1.0f / total : 0.f;
    h4 o;
#pragma unroll
    for (int x = 0; x < 4; x++) o[x] = narrow_f32(v[x] * inv);
    *reinterpret_cast<h4*>(a.out + (size_t)(start + i) * a.out_stride + (size_t)(h * p.group + (row - i * p.group)) * DIM + d) = o;
  };
  auto finish_row = [&](uint32_t row, float top, float total) {
    const uint32_t i = row / p.group;
    if (a.lse) a.lse[(size_t)(start + i) * a.heads + h * p.group + (row - i * p.group)] = total > 0.f || total != total ? (top - LIFT + __log2f(total)) * 0.69314718055994531f : -INFINITY;
  };
  // where a row's partial results of split 0 are; the other splits follow
  auto partial_at = [&](uint32_t row) { return ((size_t)(b * c.kv_heads + h) * a.max_query * p.group + row) * p.splits; };
  if constexpr (KW == 1) {
#pragma unroll
    for (int t = 0; t < QT; t++) {
      const uint32_t row = wave_row + 16 * t + lj;
      if (row < rows) {
        if (parts == 1) {
          if (lc == 0) finish_row(row, m[t], l[t]);
#pragma unroll
          for (int d = 0; d < 2 * KD; d++) finish4(row, 16 * d + 4 * lc, acc[t][d], l[t]);
        } else {  // attention_join_kernel adds the parts
          const size_t at = partial_at(row) + split;
          if (lc == 0) p.partial_ml[at] = make_float2(m[t], l[t]);
#pragma unroll
          for (int d = 0; d < 2 * KD; d++) *reinterpret_cast<f4*>(p.partial + at * DIM + 16 * d + 4 * lc) = acc[t][d];
        }
      }
    }
  } else {
    float* joined = reinterpret_cast<float*>(lds);
    float2* ml = reinterpret_cast<float2*>(lds + KW * ROWS * Shape::PITCH * 4);
    __syncthreads();  // the stages are done with
#pragma unroll
    for (int t = 0; t < QT; t++)
      if (lc == 0) ml[kw * ROWS + rw * 16 * QT + 16 * t + lj] = make_float2(m[t], l[t]);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < QT; t++) {
      const uint32_t local = rw * 16 * QT + 16 * t + lj;
      float top = m[t];
#pragma unroll
      for (int k = 0; k < KW; k++) top = fmaxf(top, ml[k * ROWS + local].x);
      const float keep = __builtin_amdgcn_exp2f(m[t] - top);
#pragma unroll
      for (int d = 0; d < 2 * KD; d++) *reinterpret_cast<f4*>(joined + (kw * ROWS + local) * Shape::PITCH + 16 * d + 4 * lc) = acc[t][d] * keep;
    }
    __syncthreads();
    for (uint32_t i = tid; i < ROWS * (DIM / 4); i += 64 * RW * KW) {
      const uint32_t local = i / (DIM / 4), d = (i - local * (DIM / 4)) * 4, row = row0 + local;
      if (row >= rows) continue;
      float top = ml[local].x, total = 0.f;
#pragma unroll
      for (int k = 1; k < KW; k++) top = fmaxf(top, ml[k * ROWS + local].x);
      f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KW; k++) {
        total += ml[k * ROWS + local].y * __builtin_amdgcn_exp2f(ml[k * ROWS + local].x - top);
        v += *reinterpret_cast<const f4*>(joined + (k * ROWS + local) * Shape::PITCH + d);
      }
      if (parts == 1) {
        finish4(row, d, v, total);
        if (d == 0) finish_row(row, top, total);
      } else if (!p.arrivals) {  // attention_join_kernel adds the parts
        const size_t at = partial_at(row) + split;
        *reinterpret_cast<f4*>(p.partial + at * DIM + d) = v;
        if (d == 0) p.partial_ml[at] = make_float2(top, total);
      } else {
        const size_t at = partial_at(row) + split;
        put2(p.partial + at * DIM + d, v.x, v.y);
        put2(p.partial + at * DIM + d + 2, v.z, v.w);
        if (d == 0) put2(reinterpret_cast<float*>(p.partial_ml + at), top, total);
      }
    }
    if (parts == 1 || !p.arrivals) return;
    // The workgroup that arrives last adds the parts, in their order. Partial results go past the caches that the XCDs do
    // not share (relaxed device-scope stores and loads), every wave waits for its own stores before the barrier, and one
    // thread counts the arrival; nobody waits for another workgroup.
    uint32_t* flag = reinterpret_cast<uint32_t*>(lds);
    wait_vm<0>();
    __syncthreads();
    const uint32_t group_id = ((uint32_t)blockIdx.y * a.sequences + b) * c.kv_heads + h;
    if (tid == 0) *flag = __hip_atomic_fetch_add(p.arrivals + group_id, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const bool last = *flag == parts - 1;
    __syncthreads();
    if (!last) return;
    if (tid == 0) __hip_atomic_store(p.arrivals + group_id, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint32_t here = min(rows - row0, (uint32_t)ROWS);
    float2* weights = reinterpret_cast<float2*>(lds);  // [row][split]
    for (uint32_t i = tid; i < here * parts; i += 64 * RW * KW) {
      const uint32_t local = i / parts, s = i - local * parts;
      weights[local * parts + s] = get2(reinterpret_cast<const float*>(p.partial_ml + partial_at(row0 + local) + s));
    }
    __syncthreads();
    for (uint32_t i = tid; i < here * (DIM / 4); i += 64 * RW * KW) {
      const uint32_t local = i / (DIM / 4), d = (i - local * (DIM / 4)) * 4, row = row0 + local;
      const float* from = p.partial + partial_at(row) * DIM + d;
      const float2* w = weights + local * parts;
      float top = NOTHING, total = 0.f;
      for (uint32_t s = 0; s < parts; s++) top = fmaxf(top, w[s].x);
      f4 v = {0.f, 0.f, 0.f, 0.f};
      for (uint32_t s0 = 0; s0 < parts; s0 += 16) {
        float2 lo[16], hi[16];
#pragma unroll
        for (uint32_t k = 0; k < 16; k++) {
          const uint32_t s = min(s0 + k, parts - 1);
          lo[k] = get2(from + (size_t)s * DIM);
          hi[k] = get2(from + (size_t)s * DIM + 2);
        }
#pragma unroll
        for (uint32_t k = 0; k < 16; k++)
          if (s0 + k < parts) {
            const float f = __builtin_amdgcn_exp2f(w[s0 + k].x - top);
            total += w[s0 + k].y * f;
            v += f4{lo[k].x, lo[k].y, hi[k].x, hi[k].y} * f;
          }
      }
      finish4(row, d, v, total);
      if (d == 0) finish_row(row, top, total);
    }
  }
}

// Adds the partial results of a row's splits, in their order. WAVES waves per query row and head. BATCH: splits that a lane asks
// for at once (few splits: the instructions of an empty batch are what the launch would wait for).
template <uint32_t BATCH, uint32_t WAVES>
__global__ __launch_bounds__(256) void attention_join_kernel(const MfmaParams p, uint32_t tile_rows) {
  const AttentionArgs& a = p.a;
  const KvView& c = a.cache;
  const uint32_t lane = threadIdx.x & 63u, b = blockIdx.y;
  const uint32_t wave = threadIdx.x >> 6, unit = WAVES == 4 ? blockIdx.x : blockIdx.x * 4u + wave;  // (row, kv head)
  const uint32_t row = unit / c.kv_heads, h = unit - row * c.kv_heads;
  const int32_t start = a.query_start[b];
  const int64_t n = (int64_t)a.query_start[b + 1] - start;
  const int64_t tokens = min(min(n, (int64_t)a.max_query), (int64_t)a.tokens - start);
  if (start < 0 || tokens <= 0 || row >= tokens * p.group) return;
  const int32_t cached = max(a.kv_length[b], 0), length = min(cached, (int32_t)a.max_kv);
  const int64_t context = cached - n;
  // how many splits the row's workgroup had, as it worked it out
  const uint32_t last_row = min(row / tile_rows * tile_rows + tile_rows, (uint32_t)tokens * p.group) - 1;
  const int64_t seen_by_any = a.tree_mask ? length : context + last_row / p.group + 1;
  const int32_t k_last = (int32_t)max(min(seen_by_any, (int64_t)length), (int64_t)0);
  const uint32_t parts = max(1u, ((uint32_t)k_last + p.chunk - 1) / p.chunk);
  if (parts == 1) return;
  const size_t at = ((size_t)(b * c.kv_heads + h) * a.max_query * p.group + row) * p.splits;
  const float* acc = p.partial + at * c.head_dim;
  const float2* ml = p.partial_ml + at;
  // a lane takes four dims of every `steps`-th split; the first are asked for before the weights are known
  const uint32_t quads = c.head_dim / 4, ways = 64u / quads, way = lane / quads, d = (lane - way * quads) * 4;
  const uint32_t steps = ways * WAVES, first = WAVES == 4 ? wave * ways + way : way;
  f4 x[BATCH];
  auto batch = [&](uint32_t s1) {
#pragma unroll
    for (uint32_t k = 0; k < BATCH; k++) {
      const uint32_t s = s1 + k * steps + first;
      x[k] = s < parts && way < ways ? *reinterpret_cast<const f4*>(acc + (size_t)s * c.head_dim + d) : f4{0.f, 0.f, 0.f, 0.f};
    }
  };
  batch(0);
  float top = NOTHING;
  for (uint32_t s = lane; s < parts; s += 64u) top = fmaxf(top, ml[s].x);
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  float total = 0.f;
  f4 v = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t s0 = 0; s0 < parts; s0 += 64u) {
    const uint32_t here = min(parts - s0, 64u);
    const float2 mine = lane < here ? ml[s0 + lane] : make_float2(NOTHING, 0.f);
    const float w = lane < here ? __builtin_amdgcn_exp2f(mine.x - top) : 0.f;
    total += mine.y * w;
    for (uint32_t s1 = 0; s1 < here; s1 += BATCH * steps) {
      if (s0 + s1) batch(s0 + s1);
#pragma unroll
      for (uint32_t k = 0; k < BATCH; k++) {
        const uint32_t s = s1 + k * steps + first;
        const float ws = __shfl(w, (int)min(s, 63u));
        if (s < 64u) v += x[k] * ws;
      }
    }
  }
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
  f4 sum = v;
  for (uint32_t k = 1; k < ways; k++) {
    f4 other;
#pragma unroll
    for (int x = 0; x < 4; x++) other[x] = __shfl(v[x], (int)min(lane + k * quads, 63u));
    sum += other;  // of use in the first way only, where the ways are added in their order
  }
  if constexpr (WAVES > 1) {
    __shared__ f4 of_wave[WAVES][64];
    of_wave[wave][lane] = sum;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (uint32_t k = 1; k < WAVES; k++) sum += of_wave[k][lane];
  }
  const float inv = total > 0.f || total != total ? 1.0f / total : 0.f;
  const uint32_t i = row / p.group, head = h * p.group + (row - i * p.group);
  if (way == 0) {
    h4 o;
#pragma unroll
    for (int x = 0; x < 4; x++) o[x] = narrow_f32(sum[x] * inv);
    *reinterpret_cast<h4*>(a.out + (size_t)(start + i) * a.out_stride + (size_t)head * c.head_dim + d) = o;
  }
  if (a.lse && lane == 0) a.lse[(size_t)(start + i) * a.heads + head] = total > 0.f || total != total ? (top - LIFT + __log2f(total)) * 0.69314718055994531f : -INFINITY;
}

// What the matrix-core kernel takes: whole 64-byte units of a head, pages of whole 16-key blocks, 16-byte rows. (A token over
// 1037 keys of 2 x 160: 10.8 us here, 280 with the plain kernel.)
bool mfma_takes(const AttentionArgs& a) {
  const KvView& c = a.cache;
  const uint32_t kd = c.head_dim / 32;
  if (c.head_dim % 32 || c.slot_bytes != 2 * c.head_dim || kd < 1 || kd > 8 || kd == 7) return false;
  if (c.page_size % 16 || !c.num_pages || !a.max_kv) return false;
  const uint64_t at = reinterpret_cast<uint64_t>(c.pages) | c.page_bytes | c.head_bytes | c.side_bytes | c.slot_bytes;
  if (at % 16 || reinterpret_cast<uint64_t>(c.scales) % 4) return false;
  if ((reinterpret_cast<uint64_t>(a.q) | reinterpret_cast<uint64_t>(a.out)) & 15u || a.q_stride % 8 || a.out_stride % 8) return false;
  // the grid's limits
  const uint64_t rows = (uint64_t)a.max_query * (a.heads / c.kv_heads);
  return rows <= 64ull * 65535u && a.max_query * (uint64_t)a.heads < (1ull << 31) && (uint64_t)a.sequences * c.kv_heads < (1u << 20);
}

struct MfmaPlan {
  int qt, rw, kw;
  uint32_t rows, row_tiles, splits, chunk;
  size_t partial_bytes, bytes;
  bool fused;  // the workgroup that arrives last joins
};
MfmaPlan mfma_plan(const AttentionArgs& a) {
  MfmaPlan g{};
  const uint32_t group = a.heads / a.cache.kv_heads;
  const uint64_t rows = (uint64_t)a.max_query * group;
  const bool wide = a.cache.head_dim > 128;
  // Few rows: the waves of a workgroup split the keys, so that each key is read by one of them (two waves in flight: a batch
  // of 48 tokens 160 us, four 164). More: four waves share the staged keys and split the rows, two row tiles each up to
  // heads of 128 (int8 trees of up to 61 x 4 rows: one tile a wave 99 us, two 77, though the int8 instance for heads of 128
  // fills all 256 registers and spills 8 into its mask branch; heads of 256 spill in the loop: 15 trees of 74 rows over
  // 1846 int8 keys 108 us, with two 158).
  if (rows <= 16) g.qt = 1, g.rw = 1, g.kw = 2;
  else if (rows <= 32) g.qt = 2, g.rw = 1, g.kw = wide ? 2 : 4;
  else g.qt = rows <= 64 || wide ? 1 : 2, g.rw = 4, g.kw = 1;
  g.rows = 16 * g.qt * g.rw;
  g.row_tiles = (uint32_t)((rows + g.rows - 1) / g.rows);
  const uint64_t groups = (uint64_t)a.sequences * a.cache.kv_heads * g.row_tiles;
  // Workgroups that fill the CUs about once or twice; more cost their beginnings and the join. Measured with 1024 / 1536 /
  // 2048 where the waves split the keys: 16 sequences x 4000 int8 keys x 8 heads 28.7 / 34.2 / 34.6 us, 4 x 16000 f16
  // 56.2 / 58.1 / 58.4, and where there are many ragged sequences, whose ends finer parts even out, 48 x up to 8191 f16
  // 162.7 / 156.4 / 154.8, x up to 4000 int8 60.6 / 56.3 / 57.7. Heads past 128 leave room for one workgroup a CU; of 256: 256 / 512 / 2048 of
  // them 52.3 / 57.2 / 72.2 us for a token over 27155 keys, 55.7 / 58.8 / 91.5 for 8 x 4000. 
  // Where the waves split the rows, 512 fill the CUs once, and lengths that the host does not know (several sequences, of
  // which some are short) need finer parts where a group would have five or fewer. 512 / 1024, f16 and int8: one tree of 64
  // over 16000 keys (32 heads on 8 of 128) 45.0 / 57.8, 48.7 / 58.6; two over 8000 44.0 / 63.2, 48.0 / 63.4; trees of 32 over 4500
  // keys, 64 groups 50.9 / 67.1, 52.3 / 65.7, of 4 to 32 over 200 to 4500 41.5 / 44.2, 45.3 / 48.3; 80 groups of these 69.6 / 74.1,
  // 72.1 / 73.1, ragged 46.2 / 50.2, 51.0 / 54.0; 96 groups 86.2 / 83.6, 91.4 / 84.3, ragged 47.9 / 52.3, 53.4 / 57.3; 104 ragged of 64
  // 57.2 / 44.4, 62.2 / 61.5; 256 groups, trees of 61 over 4500 130 / 155, 140 / 150, of 5 to 61 over 200 to 4500 112 / 71, 127 / 78. One
  // prompt chunk of 2048 behind nothing, 512 groups: 88 / 119, 100 / 130; behind 8000 keys 411 / 458, 482 / 526.
  const bool ragged = a.sequences > 1 && groups >= 96;
  const uint64_t want = wide ? 256 : g.rw == 1 ? (groups > 256 ? 1536 : 1024) : ragged ? 1024 : 512;
  // A part is two turns of the key waves or more, four 64-key turns where the waves split the rows (one token over 1037
  // keys, one / two / four / eight turns: 9.9 / 8.9 / 10.0 / 11.5 us), and a row has at most 128: with 256 of them a step
  // of 8 rows x 8 heads over 64000 keys takes 65.6 instead of 58.3 us, their join being what grows.
  const uint32_t unit = std::max(32u * g.kw, 64u), least = unit * (g.kw > 1 ? 2u : 4u);
  uint64_t splits = (want + groups - 1) / groups;
  splits = std::max<uint64_t>(1, std::min<uint64_t>({splits, (a.max_kv + least - 1) / least, (uint64_t)MOST_SPLITS}));
  g.chunk = (uint32_t)(((a.max_kv + splits - 1) / splits + unit - 1) / unit * unit);
  g.splits = (a.max_kv + g.chunk - 1) / g.chunk;
  // Few partial rows are joined by the workgroup that arrives last, more by a launch of their own with four waves for each
  // row: 4 rows x 9 parts 8.9 against 10.7 us, 8 x 8 10.4 and 11.4, but 16 x 32 21.0 and 11.7, 16 x 128 57.8 and 13.7.
  g.fused = g.kw > 1 && g.splits <= FUSED_SPLITS && rows * g.splits <= 64;
  static_assert(ZTVM_ARRIVALS >= 2048, "a counter for every row tile that is split");
  if (g.splits > 1) {
    const uint64_t n = (uint64_t)a.sequences * a.heads * a.max_query * g.splits;
    g.partial_bytes = n * a.cache.head_dim * 4;
    g.bytes = g.partial_bytes + n * 8;
  }
  return g;
}

template <int KD, bool INT8, int QT, int RW, int KW, int NS>
hipError_t launch_mfma_shape(const MfmaParams& p, const MfmaPlan& g, hipStream_t s) {
  using Shape = MfmaShape<KD, INT8, QT, RW, KW, NS>;
  auto kernel = attention_mfma_kernel<KD, INT8, QT, RW, KW, NS>;
  if (Shape::LDS > 64 * 1024) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, Shape::LDS);
  const dim3 grid(p.a.sequences * p.a.cache.kv_heads * g.splits, g.row_tiles);
  hipLaunchKernelGGL(kernel, grid, dim3(64 * RW * KW), Shape::LDS, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || g.splits == 1 || p.arrivals) return e;
  const uint32_t units = p.a.max_query * p.a.heads;
  // many parts: four waves for a row (38 rows x 4 sequences x 128 parts 25.3 -> 23.3 us, 25 x 3 x 128 28.3 -> 22.5)
  if (g.splits > 16) {
    hipLaunchKernelGGL((attention_join_kernel<8, 4>), dim3(units, p.a.sequences), dim3(256), 0, s, p, g.rows);
    return hipGetLastError();
  }
  auto join = g.splits * KD <= 16 ? attention_join_kernel<2, 1> : attention_join_kernel<8, 1>;
  hipLaunchKernelGGL(join, dim3((units + 3) / 4, p.a.sequences), dim3(256), 0, s, p, g.rows);
  return hipGetLastError();
}
template <int KD, bool INT8>
hipError_t launch_mfma_dim(const MfmaParams& p, const MfmaPlan& g, hipStream_t s) {
  constexpr int KW = KD > 4 ? 2 : 4;
  constexpr int NS = INT8 ? 2 : 1;
  if (g.rw == 4 && g.qt == 2) return launch_mfma_shape<KD, INT8, (KD > 4 ? 1 : 2), 4, 1, NS>(p, g, s);
  if (g.rw == 4) return launch_mfma_shape<KD, INT8, 1, 4, 1, NS>(p, g, s);
  if (g.qt == 2) return launch_mfma_shape<KD, INT8, 2, 1, KW, 1>(p, g, s);
  return launch_mfma_shape<KD, INT8, 1, 1, 2, 1>(p, g, s);
}

}  // namespace

size_t attention_scratch_bytes(const AttentionArgs& a) { return mfma_takes(a) ? mfma_plan(a).bytes : 0; }

hipError_t launch_attention(const AttentionArgs& a, void* scratch, uint32_t* arrivals, hipStream_t s) {
  if (!mfma_takes(a)) {
    hipLaunchKernelGGL(attention_any_kernel, dim3(a.tokens, a.heads), dim3(256), 0, s, a);
    return hipGetLastError();
  }
  const MfmaPlan g = mfma_plan(a);
  if (!g.fused) arrivals = nullptr;
  MfmaParams p{a, static_cast<float*>(scratch), reinterpret_cast<float2*>(static_cast<char*>(scratch) + g.partial_bytes), arrivals, g.splits, g.chunk,
               a.heads / a.cache.kv_heads, std::max(fabsf(a.scale) * 1.4426950408889634f, 1e-30f), a.scale < 0.f};  // never 0: a masked score is -inf times it
  auto by_format = [&](auto kd) {
    constexpr int KD = decltype(kd)::value;
    return a.cache.int8 ? launch_mfma_dim<KD, true>(p, g, s) : launch_mfma_dim<KD, false>(p, g, s);
  };
  switch (a.cache.head_dim / 32) {
    case 1: return by_format(ic<1>{});
    case 2: return by_format(ic<2>{});
    case 3: return by_format(ic<3>{});
    case 4: return by_format(ic<4>{});
    case 5: return by_format(ic<5>{});
    case 6: return by_format(ic<6>{});
    default: return by_format(ic<8>{});
  }
}

}  // namespace ztvm
