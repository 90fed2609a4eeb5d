// Attention of the query tokens of several sequences over the paged cache.
#include "internal.h"
#include "kv_cache.h"
#include "quant.h"

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
  const int32_t length = min(max(p.kv_length[b], 0), (int32_t)p.max_kv);
  const int64_t context = (int64_t)length - n;
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

}  // namespace

size_t attention_scratch_bytes(const AttentionArgs&) { return 0; }

hipError_t launch_attention(const AttentionArgs& a, void*, hipStream_t s) {
  hipLaunchKernelGGL(attention_any_kernel, dim3(a.tokens, a.heads), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace ztvm
