// Rotary positions with the append of K and V to the paged cache (f16 or int8), and the read-back of cached rows.
// Both move bytes: every element is read once and written once, so they are bound by memory for many tokens and by
// the launch for few.
#include "internal.h"
#include "kv_cache.h"
#include "quant.h"

namespace ztvm {
namespace {

typedef uint8_t u8x8 __attribute__((ext_vector_type(8)));
typedef uint8_t u8x16 __attribute__((ext_vector_type(16)));

// cos and sin of position * frequency, scaled. The angle is formed in turns and reduced to [-1/2, 1/2] in 64 bits (an
// f32 product would carry position * 2^-24 of error in the angle); what is left rounds to f32 with an error of 2^-25
// turns at most, 2e-7 rad, against 2^-12 relative of the f16 result.
__device__ __forceinline__ void turn(int32_t position, double frequency, float factor, float& c, float& s) {
  const double t = (double)position * (frequency * 0.15915494309189533577);
  const float r = (float)(t - __builtin_rint(t));
  sincospif(2.0f * r, &s, &c);
  c *= factor;
  s *= factor;
}
__device__ __forceinline__ void rotate(float& x, float& y, float c, float s) {
  const float a = x * c - y * s, b = y * c + x * s;
  x = a;
  y = b;
}

// int8 form of a row (the arithmetic of kv_quantize_int8_kernel): scale from the row's largest magnitude
__device__ __forceinline__ float row_scale(float largest) {
  const float scale = largest / 127.0f;
  return scale < 1e-8f ? 1e-8f : scale;
}
__device__ __forceinline__ uint8_t count_of(float v, float inv_scale) {
  float q = __builtin_rintf(v * inv_scale);
  q = fminf(fmaxf(q, -127.f), 127.f);
  return (uint8_t)(int8_t)(int32_t)q;
}

struct RopeParams {
  const _Float16* qkv;
  _Float16* q_out;
  const double* frequencies;
  const int32_t* positions;
  const int32_t* slots;
  uint32_t qkv_stride, q_stride;
  uint32_t heads, rotary, interleaved;
  uint32_t rows_per_block;  // head rows of a token that one workgroup takes (a multiple of its row groups)
  float factor;
  KvView cache;
};

constexpr uint32_t ROPE_MAX_DIM = 512;

// One workgroup per token and block of head rows. cos and sin of the token are computed once into LDS; W lanes (the
// power of two from head_dim/16 on) then take one head row at a time, 16 elements each: in the half layout two
// 16-byte chunks half a rotary part away from each other, so that a lane holds both elements of its pairs and no
// value crosses lanes; otherwise two neighbouring chunks.
// 8192 tokens of 32 + 2 x 8 heads of 128 (201 MB read and written): 39.5 us, 5.1 TB/s, the rate of a large copy on the card
// (5.05); one token 3.9 us, a launch.
template <int W, bool INT8>
__global__ __launch_bounds__(256) void rope_append_kernel(const RopeParams p) {
  __shared__ float cs[ROPE_MAX_DIM / 2], sn[ROPE_MAX_DIM / 2];
  const uint32_t t = blockIdx.x, half = p.rotary / 2;
  const int32_t position = p.positions[t];
  for (uint32_t j = threadIdx.x; j < half; j += 256u) turn(position, p.frequencies[j], p.factor, cs[j], sn[j]);
  const uint32_t dim = p.cache.head_dim, kv = p.cache.kv_heads, rows = p.heads + 2 * kv;
  uint32_t page = 0, slot = 0;
  const bool stored = kv_locate(p.cache, p.slots[t], page, slot);
  __syncthreads();
  const uint32_t lane = threadIdx.x % W, chunks = dim / 8;
  const uint32_t first = blockIdx.y * p.rows_per_block;
  const uint32_t last = min(rows, first + p.rows_per_block);
  const uint32_t quarter = p.rotary / 16;  // chunk pairs of the rotated part
  const _Float16* in = p.qkv + (size_t)t * p.qkv_stride;
  for (uint32_t r = first + threadIdx.x / W; r < last; r += 256u / W) {
    const bool is_q = r < p.heads, is_v = r >= p.heads + kv;
    if (!is_q && !stored) continue;  // uniform within the W lanes of a row
    // the two chunks of this lane
    uint32_t c0 = 2 * lane, c1 = c0 + 1;
    const bool paired = !p.interleaved && lane < quarter;
    if (paired) {
      c0 = lane;
      c1 = lane + quarter;
    }
    const bool there = c0 < chunks;
    float x[16];
    const _Float16* src = in + (size_t)r * dim;
    if (there) {
      const h8 a = *reinterpret_cast<const h8*>(src + 8 * c0), b = *reinterpret_cast<const h8*>(src + 8 * c1);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[i] = (float)a[i];
        x[8 + i] = (float)b[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) x[i] = 0.f;
    }
    if (!is_v && there) {
      if (paired) {
#pragma unroll
        for (int i = 0; i < 8; i++) rotate(x[i], x[8 + i], cs[8 * c0 + i], sn[8 * c0 + i]);
      } else if (p.interleaved && lane < quarter) {
#pragma unroll
        for (int i = 0; i < 8; i++) rotate(x[2 * i], x[2 * i + 1], cs[8 * lane + i], sn[8 * lane + i]);
      }
    }
    h8 a, b;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      a[i] = narrow_f32(x[i]);
      b[i] = narrow_f32(x[8 + i]);
    }
    if (is_q) {
      if (there) {
        _Float16* o = p.q_out + (size_t)t * p.q_stride + (size_t)r * dim;
        *reinterpret_cast<h8*>(o + 8 * c0) = a;
        *reinterpret_cast<h8*>(o + 8 * c1) = b;
      }
      continue;
    }
    const uint32_t head = is_v ? r - p.heads - kv : r - p.heads;
    char* row = p.cache.pages + kv_row_offset(p.cache, page, head, slot, is_v);
    if constexpr (!INT8) {
      if (there) {
        *reinterpret_cast<h8*>(row + 16 * c0) = a;
        *reinterpret_cast<h8*>(row + 16 * c1) = b;
      }
    } else {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) m = fmaxf(m, fmaxf(fabsf((float)a[i]), fabsf((float)b[i])));
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));  // the W lanes of a row stay together
      const float scale = row_scale(m), inv = 1.0f / scale;
      u8x8 qa, qb;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        qa[i] = count_of((float)a[i], inv);
        qb[i] = count_of((float)b[i], inv);
      }
      if (there) {
        *reinterpret_cast<u8x8*>(row + 8 * c0) = qa;
        *reinterpret_cast<u8x8*>(row + 8 * c1) = qb;
      }
      if (lane == 0) {
        const _Float16 s = (_Float16)scale;
        p.cache.scales[kv_scale_index(p.cache, page, head, slot, is_v)] = __builtin_bit_cast(uint16_t, s);
      }
    }
  }
}

// Head sizes, rotary parts, strides and addresses that the 16-byte form cannot take: one wave per head row, a pair of
// elements per lane and turn (the pair that is rotated together, or two neighbours).
template <bool INT8>
__global__ __launch_bounds__(256) void rope_append_any_kernel(const RopeParams p) {
  constexpr int TURNS = ROPE_MAX_DIM / 2 / 64;
  const uint32_t t = blockIdx.x, half = p.rotary / 2, lane = threadIdx.x & 63u;
  const uint32_t dim = p.cache.head_dim, kv = p.cache.kv_heads, rows = p.heads + 2 * kv;
  const int32_t position = p.positions[t];
  uint32_t page = 0, slot = 0;
  const bool stored = kv_locate(p.cache, p.slots[t], page, slot);
  const uint32_t first = blockIdx.y * p.rows_per_block;
  const uint32_t last = min(rows, first + p.rows_per_block);
  for (uint32_t r = first + (threadIdx.x >> 6); r < last; r += 4u) {
    const bool is_q = r < p.heads, is_v = r >= p.heads + kv;
    if (!is_q && !stored) continue;  // uniform per wave
    const _Float16* src = p.qkv + (size_t)t * p.qkv_stride + (size_t)r * dim;
    _Float16 x[TURNS][2];
    uint32_t at[TURNS][2];
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < TURNS; k++) {
      const uint32_t j = lane + 64u * k;
      at[k][0] = 2 * j;
      at[k][1] = 2 * j + 1;
      if (!p.interleaved && j < half) {
        at[k][0] = j;
        at[k][1] = j + half;
      }
      if (2 * j >= dim) continue;
      float a = (float)src[at[k][0]], b = (float)src[at[k][1]];
      if (!is_v && j < half) {
        float c, s;
        turn(position, p.frequencies[j], p.factor, c, s);
        rotate(a, b, c, s);
      }
      x[k][0] = narrow_f32(a);
      x[k][1] = narrow_f32(b);
      m = fmaxf(m, fmaxf(fabsf((float)x[k][0]), fabsf((float)x[k][1])));
    }
    const uint32_t head = is_v ? r - p.heads - kv : r - p.heads;
    char* row = is_q ? reinterpret_cast<char*>(p.q_out + (size_t)t * p.q_stride + (size_t)r * dim)
                     : p.cache.pages + kv_row_offset(p.cache, page, head, slot, is_v);
    float inv = 0.f;
    if (INT8 && !is_q) {
      for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
      const float scale = row_scale(m);
      inv = 1.0f / scale;
      const _Float16 s = (_Float16)scale;
      if (lane == 0) p.cache.scales[kv_scale_index(p.cache, page, head, slot, is_v)] = __builtin_bit_cast(uint16_t, s);
    }
#pragma unroll
    for (int k = 0; k < TURNS; k++) {
      if (2 * (lane + 64u * k) >= dim) continue;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        if (INT8 && !is_q) reinterpret_cast<uint8_t*>(row)[at[k][i]] = count_of((float)x[k][i], inv);
        else reinterpret_cast<_Float16*>(row)[at[k][i]] = x[k][i];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- kv_read ----
struct ReadParams {
  _Float16* out[2];  // K, V (null: not wanted)
  const int32_t* slots;
  uint32_t tokens, out_stride;
  KvView cache;
};

// A thread reads 16 bytes. f16: 8 elements of K (grid y 0) or V (1). int8: 16 elements of a slot's K | V row, which lies in one
// piece, so both sides travel together: 16390 rows of 8 x 128 take 20.8 us (4.8 TB/s, the rate of a large copy), with K and V
// in workgroups of their own and 8 elements a thread 26.
template <bool INT8>
__global__ __launch_bounds__(256) void kv_read_kernel(const ReadParams p) {
  const uint32_t dim = p.cache.head_dim, chunks = dim / 8, per_token = chunks * p.cache.kv_heads;
  const uint64_t total = (uint64_t)p.tokens * per_token, step = (uint64_t)gridDim.x * 256u;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < total; i += step) {
    const uint32_t t = (uint32_t)(i / per_token), rest = (uint32_t)(i - (uint64_t)t * per_token);
    const uint32_t head = rest / chunks, c = rest - head * chunks;
    const uint32_t side = INT8 ? c >= chunks / 2 : blockIdx.y;
    _Float16* out = p.out[side];
    uint32_t page, slot;
    if (!out || !kv_locate(p.cache, p.slots[t], page, slot)) continue;
    const char* row = p.cache.pages + kv_row_offset(p.cache, page, head, slot, INT8 ? 0 : side);
    out += (size_t)t * p.out_stride + (size_t)head * dim;
    if constexpr (INT8) {
      const u8x16 q = *reinterpret_cast<const u8x16*>(row + 16 * c);
      const float scale = (float)__builtin_bit_cast(_Float16, p.cache.scales[kv_scale_index(p.cache, page, head, slot, side)]);
      h8 lo, hi;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        lo[k] = narrow_f32((float)(int8_t)q[k] * scale);
        hi[k] = narrow_f32((float)(int8_t)q[8 + k] * scale);
      }
      h8* to = reinterpret_cast<h8*>(out + 16 * (c - side * (chunks / 2)));
      to[0] = lo;
      to[1] = hi;
    } else {
      *reinterpret_cast<h8*>(out + 8 * c) = *reinterpret_cast<const h8*>(row + 16 * c);
    }
  }
}

// any head size and alignment: one element per thread
template <bool INT8>
__global__ __launch_bounds__(256) void kv_read_any_kernel(const ReadParams p) {
  const uint32_t side = blockIdx.y, dim = p.cache.head_dim, per_token = dim * p.cache.kv_heads;
  _Float16* out = p.out[side];
  if (!out) return;
  const uint64_t total = (uint64_t)p.tokens * per_token, step = (uint64_t)gridDim.x * 256u;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < total; i += step) {
    const uint32_t t = (uint32_t)(i / per_token), rest = (uint32_t)(i - (uint64_t)t * per_token);
    const uint32_t head = rest / dim, d = rest - head * dim;
    uint32_t page, slot;
    if (!kv_locate(p.cache, p.slots[t], page, slot)) continue;
    const char* row = p.cache.pages + kv_row_offset(p.cache, page, head, slot, side);
    _Float16 v;
    if constexpr (INT8) {
      const float scale = (float)__builtin_bit_cast(_Float16, p.cache.scales[kv_scale_index(p.cache, page, head, slot, side)]);
      v = narrow_f32((float)reinterpret_cast<const int8_t*>(row)[d] * scale);
    } else {
      v = reinterpret_cast<const _Float16*>(row)[d];
    }
    out[(size_t)t * p.out_stride + (size_t)head * dim + d] = v;
  }
}

// every row of the cache starts at a multiple of what the wide kernels load from it
bool wide_rows(const KvView& c) {
  const uint64_t at = reinterpret_cast<uint64_t>(c.pages) | c.page_bytes | c.head_bytes | c.side_bytes | c.slot_bytes;
  return c.head_dim % 16 == 0 && at % 16 == 0;
}

}  // namespace

hipError_t launch_rope_append(const RopeAppendArgs& a, hipStream_t s) {
  RopeParams p{a.qkv, a.q_out, a.frequencies, a.positions, a.slots, a.qkv_stride, a.q_stride, a.heads, a.rotary_dim, a.interleaved, 0,
               a.attn_factor, a.cache};
  const uint32_t dim = a.cache.head_dim, rows = a.heads + 2 * a.cache.kv_heads;
  const bool wide = wide_rows(a.cache) && !((reinterpret_cast<uint64_t>(a.qkv) | reinterpret_cast<uint64_t>(a.q_out)) & 15u) &&
                    a.qkv_stride % 8 == 0 && a.q_stride % 8 == 0 && a.rotary_dim % 16 == 0;
  uint32_t w = 1;
  while (w < dim / 16) w *= 2;
  const uint32_t groups = wide ? 256 / w : 4;  // head rows a workgroup takes at a time
  // few tokens: a workgroup per group of head rows, so that the rows of a token travel side by side; many: a
  // workgroup takes a whole token and computes its cosines once
  // (391 int8 tokens of 32 + 16 heads of 128: 4.7 split, 5.4 us whole; 8192 of 28 + 8 heads of 96, int8: 29.8 and 26.7;
  // of 56 + 16 heads of 64: 32.5 and 29.7; of 32 + 16 heads of 128: 38.8 and 39.5)
  uint32_t turns = (rows + groups - 1) / groups;
  const uint32_t split = a.tokens >= 1024 ? 1 : turns;
  turns = (turns + split - 1) / split;
  p.rows_per_block = turns * groups;
  const dim3 grid(a.tokens, (rows + p.rows_per_block - 1) / p.rows_per_block), block(256);
  if (!wide) {
    if (a.cache.int8) hipLaunchKernelGGL(rope_append_any_kernel<true>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(rope_append_any_kernel<false>, grid, block, 0, s, p);
    return hipGetLastError();
  }
  auto go = [&](auto k16, auto k8) {
    if (a.cache.int8) hipLaunchKernelGGL(k8, grid, block, 0, s, p);
    else hipLaunchKernelGGL(k16, grid, block, 0, s, p);
  };
  switch (w) {
    case 1: go(rope_append_kernel<1, false>, rope_append_kernel<1, true>); break;
    case 2: go(rope_append_kernel<2, false>, rope_append_kernel<2, true>); break;
    case 4: go(rope_append_kernel<4, false>, rope_append_kernel<4, true>); break;
    case 8: go(rope_append_kernel<8, false>, rope_append_kernel<8, true>); break;
    case 16: go(rope_append_kernel<16, false>, rope_append_kernel<16, true>); break;
    default: go(rope_append_kernel<32, false>, rope_append_kernel<32, true>); break;
  }
  return hipGetLastError();
}

hipError_t launch_kv_read(const KvReadArgs& a, hipStream_t s) {
  const ReadParams p{{a.k_out, a.v_out}, a.slots, a.tokens, a.out_stride, a.cache};
  const bool wide = wide_rows(a.cache) && !((reinterpret_cast<uint64_t>(a.k_out) | reinterpret_cast<uint64_t>(a.v_out)) & 15u) && a.out_stride % 8 == 0;
  const uint64_t units = (uint64_t)a.tokens * a.cache.kv_heads * (wide ? a.cache.head_dim / 8 : a.cache.head_dim);
  const uint64_t blocks = (units + 255) / 256;
  const dim3 grid((uint32_t)(blocks > 65536 ? 65536 : blocks), wide && a.cache.int8 ? 1 : 2), block(256);
  if (wide) {
    if (a.cache.int8) hipLaunchKernelGGL(kv_read_kernel<true>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(kv_read_kernel<false>, grid, block, 0, s, p);
  } else {
    if (a.cache.int8) hipLaunchKernelGGL(kv_read_any_kernel<true>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(kv_read_any_kernel<false>, grid, block, 0, s, p);
  }
  return hipGetLastError();
}

}  // namespace ztvm
