// What rows of logits say: log probability of a given token, entropy, the best alternatives.
#include "internal.h"
#include "quant.h"

namespace ztvm {
namespace {

// A logit's place in the descending order as an unsigned number (larger is better); NaN comes last.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);  // -0 and +0 are one value
  return v != v ? 0u : (b & 0x80000000u ? ~b : b | 0x80000000u);
}

// Rows too long for the table of neighbourhoods below: one workgroup per row, one pass for the maximum, one for the
// sums, one for each alternative.
template <class T>
__global__ __launch_bounds__(256) void logprobs_any_kernel(const LogprobsArgs p) {
  __shared__ float red[256];
  __shared__ unsigned long long best[256];
  const uint32_t r = blockIdx.x, tid = threadIdx.x;
  const T* x = reinterpret_cast<const T*>(p.logits) + (size_t)r * p.row_stride;
  float m = -INFINITY;
  for (uint32_t i = tid; i < p.vocab; i += 256u) m = fmaxf(m, (float)x[i] * p.inv_temperature);
  red[tid] = m;
  __syncthreads();
  for (uint32_t o = 128; o > 0; o >>= 1) {
    if (tid < o) red[tid] = fmaxf(red[tid], red[tid + o]);
    __syncthreads();
  }
  const bool low = red[0] == -INFINITY;  // nothing but -inf and NaN
  m = low ? 0.f : red[0];
  __syncthreads();
  float total = 0.f, weighted = 0.f;
  for (uint32_t i = tid; i < p.vocab; i += 256u) {
    float d = (float)x[i] * p.inv_temperature - m;
    d = d < -1e4f ? -1e4f : d;  // exp is 0 there; keeps 0 * -inf out of the entropy, lets NaN through
    const float e = expf(d);
    total += e;
    weighted += e * d;
  }
  red[tid] = total;
  __syncthreads();
  for (uint32_t o = 128; o > 0; o >>= 1) {
    if (tid < o) red[tid] += red[tid + o];
    __syncthreads();
  }
  total = red[0];
  __syncthreads();
  red[tid] = weighted;
  __syncthreads();
  for (uint32_t o = 128; o > 0; o >>= 1) {
    if (tid < o) red[tid] += red[tid + o];
    __syncthreads();
  }
  weighted = red[0];
  const bool nothing = low && total == 0.f;  // every logit is -inf (a NaN would be in the sum)
  const float log_total = logf(total);
  auto logp = [&](float v) { return nothing ? -INFINITY : (v * p.inv_temperature - m) - log_total; };
  if (tid == 0) {
    if (p.logprob) {
      const int32_t t = p.tokens[r];
      p.logprob[r] = t >= 0 && (uint32_t)t < p.vocab ? logp((float)x[t]) : -INFINITY;
    }
    if (p.entropy) p.entropy[r] = nothing ? 0.f : log_total - weighted / total;
  }
  if (!p.top_k) return;
  unsigned long long last = ~0ull;  // order in the high half, ~id in the low: larger is better, ties to the lower id
  for (uint32_t k = 0; k < p.top_k; k++) {
    unsigned long long mine = 0;
    for (uint32_t i = tid; i < p.vocab; i += 256u) {
      const unsigned long long key = (unsigned long long)order_of((float)x[i]) << 32 | (uint32_t)~i;
      if (key < last && key > mine) mine = key;
    }
    best[tid] = mine;
    __syncthreads();
    for (uint32_t o = 128; o > 0; o >>= 1) {
      if (tid < o) best[tid] = best[tid] > best[tid + o] ? best[tid] : best[tid + o];
      __syncthreads();
    }
    last = best[0];
    __syncthreads();
    if (tid == 0) {
      const uint32_t id = ~(uint32_t)last;
      if (p.top_ids) p.top_ids[(size_t)r * p.top_k + k] = id;
      if (p.top_logprobs) p.top_logprobs[(size_t)r * p.top_k + k] = logp((float)x[id]);
    }
  }
}

// ---- the usual path: one pass over the logits by independent waves, then one workgroup per row that joins them (rows of
// up to four segments: both in one launch)
//
// A wave takes a segment of a row, GROUPS loads of 16 bytes per lane, keeps it in registers and leaves the segment's
// maximum, sum and weighted sum, and the maximum of each neighbourhood (two loads of the wave: 512 f32 or 1024 f16
// logits that lie side by side). The best top_k logits lie in the top_k neighbourhoods with the largest maxima (ties:
// the lower one), so the joining workgroup looks at those again and at nothing else. Bound by the one read of the logits
// where there are many rows (384 rows of 248320 f32, 381 MB: 65 us for the read, 5.8 TB/s, and 10 for the join), by the
// chain of dependent steps behind it where there are few (one row of 128000 f32: 3.6 us and 7.8). Both in one launch, a
// workgroup of 1024 threads a row, took 151 us for the 384 rows and is not faster for one.
constexpr int GROUPS = 8;
constexpr int HOODS = GROUPS / 2;          // neighbourhoods of a segment
constexpr uint32_t MAX_HOODS = 4096;       // of a row
constexpr uint32_t MAX_SEGMENTS = MAX_HOODS / HOODS;
constexpr uint32_t MAX_CANDIDATES = 1024;  // logits that are ranked at once

template <class T>
constexpr uint32_t per_load = 16 / sizeof(T);
template <class T>
constexpr uint32_t hood_size = 2 * 64 * per_load<T>;
template <class T>
constexpr uint32_t segment_size = GROUPS * 64 * per_load<T>;

// What a segment leaves: its maximum, the sums of e = 2^d and of e*d with d = (x - maximum) * c, and the maxima of its
// neighbourhoods.
struct SegmentStats {
  float top, total, weighted, hood[HOODS];
};

// Elements of a row are numbered from the 16-byte boundary at or before its first one, so that every load is aligned.
template <class T>
__device__ __forceinline__ uint32_t lead_of(const T* row) {
  return (uint32_t)(reinterpret_cast<uint64_t>(row) & 15u) / sizeof(T);
}
// per_load<T> logits from place `at` (a multiple of per_load); places outside the row read as -inf
template <class T>
using Group = T __attribute__((ext_vector_type(16 / sizeof(T))));
template <class T>
__device__ __forceinline__ Group<T> load_group(const T* row, uint32_t lead, uint32_t vocab, uint32_t at) {
  constexpr uint32_t N = per_load<T>;
  if (at >= lead && at + N <= lead + vocab) return *reinterpret_cast<const Group<T>*>(row + (at - lead));
  Group<T> v;
#pragma unroll
  for (uint32_t i = 0; i < N; i++) v[i] = at + i >= lead && at + i < lead + vocab ? row[at + i - lead] : (T)-INFINITY;
  return v;
}

__device__ __forceinline__ float max_of_wave(float v) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ float sum_of_wave(float v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// value and id of a candidate as one number: larger is better, ties to the lower id
__device__ __forceinline__ unsigned long long rank_key(float v, uint32_t id) { return (unsigned long long)order_of(v) << 32 | (uint32_t)~id; }
// the logit that has this place in the order
__device__ __forceinline__ float value_of(uint32_t order) {
  return order ? __builtin_bit_cast(float, order & 0x80000000u ? order & 0x7FFFFFFFu : ~order) : NAN;
}

// One wave reads one segment.
template <class T>
__device__ __forceinline__ SegmentStats read_segment(const T* row, uint32_t lead, uint32_t vocab, uint32_t seg, float c) {
  constexpr uint32_t N = per_load<T>;
  const uint32_t lane = threadIdx.x & 63u, first = seg * segment_size<T>;
  Group<T> x[GROUPS];
#pragma unroll
  for (int g = 0; g < GROUPS; g++) x[g] = load_group(row, lead, vocab, first + (g * 64 + lane) * N);
  SegmentStats s;
  s.top = -INFINITY;
#pragma unroll
  for (int n = 0; n < HOODS; n++) {
    float m = -INFINITY;
#pragma unroll
    for (int g = 2 * n; g < 2 * n + 2; g++)
#pragma unroll
      for (uint32_t i = 0; i < N; i++) m = fmaxf(m, (float)x[g][i]);
    s.hood[n] = max_of_wave(m);
    s.top = fmaxf(s.top, s.hood[n]);
  }
  const float from = s.top == -INFINITY ? 0.f : s.top;
  s.total = s.weighted = 0.f;
#pragma unroll
  for (int g = 0; g < GROUPS; g++)
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
      const float d = ((float)x[g][i] - from) * c, e = __builtin_amdgcn_exp2f(d);  // the difference first: exact or nearly so
      s.total += e;
      s.weighted = __builtin_fmaf(e, fmaxf(d, -1e4f), s.weighted);  // e is 0 there; keeps 0 * -inf out of the sum
    }
  s.total = sum_of_wave(s.total);
  s.weighted = sum_of_wave(s.weighted);
  return s;
}

template <class T>
__global__ __launch_bounds__(256) void logits_segments_kernel(const LogprobsArgs p, SegmentStats* stats, uint32_t segments, float c) {
  const uint64_t unit = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
  const uint32_t r = (uint32_t)(unit / segments), seg = (uint32_t)(unit - (uint64_t)r * segments);
  if (r >= p.rows) return;  // whole waves leave together
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)r * p.row_stride;
  const SegmentStats s = read_segment(row, lead_of(row), p.vocab, seg, c);
  if ((threadIdx.x & 63u) == 0) stats[unit] = s;
}

// The answer for row r from its segments' statistics, by a workgroup of NT threads. A chain of dependent steps bounds it
// (statistics, their joint maximum, the bound, the neighbourhoods, the places), so what does not wait for anything is
// fetched first, and all waves look at the neighbourhoods at once.
template <class T, int NT, uint32_t MOST>
__device__ __forceinline__ void answer_row(const LogprobsArgs& p, uint32_t r, const SegmentStats* stats, uint32_t segments, float c) {
  constexpr uint32_t N = per_load<T>, WAVES = NT / 64;
  __shared__ float red[3][WAVES];
  __shared__ __align__(16) uint32_t most[256];
  __shared__ uint32_t above[256];
  __shared__ unsigned long long candidates[MAX_CANDIDATES], best[WAVES];
  __shared__ uint16_t chosen[MOST * HOODS];
  __shared__ uint32_t count, chosen_count, bound;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)r * p.row_stride;
  const uint32_t lead = lead_of(row);
  int32_t token = -1;
  if (tid == 0 && p.logprob) token = p.tokens[r];
  const bool in_vocab = token >= 0 && (uint32_t)token < p.vocab;
  float given = 0.f;
  SegmentStats first;
  first.top = -INFINITY;
  if (tid < segments) first = stats[tid];
  if (tid < 256u) above[tid] = 0;
  if (tid == 0) count = chosen_count = bound = 0;

  // ---- the sums, and the largest logit of each of 256 parts of the row
  const uint32_t K = p.top_ids || p.top_logprobs ? p.top_k : 0;
  const uint32_t hoods = (lead + p.vocab + hood_size<T> - 1) / hood_size<T>;
  const bool by_hood = hoods >= K;
  auto hood_order = [&](uint32_t n) { return order_of(stats[n / HOODS].hood[n % HOODS]); };
  if (K && tid < 256u) {
    uint32_t mine = 0;
    if (by_hood) {
      for (uint32_t n = tid; n < hoods; n += 256u) mine = max(mine, hood_order(n));
    } else {
      for (uint32_t i = tid; i < p.vocab; i += 256u) mine = max(mine, order_of((float)row[i]));
    }
    most[tid] = mine;
  }
  if (in_vocab) given = (float)row[token];
  float top = first.top;
  for (uint32_t s = tid + NT; s < segments; s += NT) top = fmaxf(top, stats[s].top);
  top = max_of_wave(top);
  if (lane == 0) red[0][wave] = top;
  __syncthreads();
  top = red[0][0];
#pragma unroll
  for (uint32_t w = 1; w < WAVES; w++) top = fmaxf(top, red[0][w]);
  const bool low = top == -INFINITY;  // nothing but -inf and NaN
  const float m = low ? 0.f : top;
  float total = 0.f, weighted = 0.f;
  auto add = [&](const SegmentStats& v) {  // e' = e * 2^d, (e*d)' = 2^d * (e*d + d * e)
    const bool none = v.top == -INFINITY;
    const float d = ((none ? 0.f : v.top) - m) * c;
    const float f = none ? (low ? 1.f : 0.f) : __builtin_amdgcn_exp2f(d);
    total += v.total != v.total ? v.total : v.total * f;
    weighted += v.total != v.total ? v.total : f == 0.f ? 0.f : f * (v.weighted + (none ? 0.f : d) * v.total);
  };
  if (tid < segments) add(first);
  for (uint32_t s = tid + NT; s < segments; s += NT) add(stats[s]);
  total = sum_of_wave(total);
  weighted = sum_of_wave(weighted);
  if (lane == 0) {
    red[1][wave] = total;
    red[2][wave] = weighted;
  }
  // ---- a bound: the K-th largest of those maxima; at least K logits reach it. A thread compares one part with 64 or 256.
  if (K) {
    const uint32_t mine = most[tid & 255u], own = (tid & 255u) >> 6;
    uint32_t before = 0;  // parts that come before this one; an equal maximum of a lower part does
#pragma unroll 1
    for (uint32_t w = NT == 1024 ? tid >> 8 : 0; w < (NT == 1024 ? (tid >> 8) + 1 : 4); w++) {
      const uint32_t limit = w < own ? mine - 1u : mine;
      if (w != own) {
#pragma unroll 8
        for (uint32_t j = 64 * w; j < 64 * w + 64; j += 4) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(&most[j]);
          before += (v.x > limit) + (v.y > limit) + (v.z > limit) + (v.w > limit);
        }
      } else {
#pragma unroll 8
        for (uint32_t j = 0; j < 64; j += 4) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(&most[64 * w + j]);
          before += v.x > mine || (v.x == mine && j < lane);
          before += v.y > mine || (v.y == mine && j + 1 < lane);
          before += v.z > mine || (v.z == mine && j + 2 < lane);
          before += v.w > mine || (v.w == mine && j + 3 < lane);
        }
      }
    }
    atomicAdd(&above[tid & 255u], before);
  }
  __syncthreads();
  if (K && tid < 256u && most[tid] && above[tid] == K - 1) bound = most[tid];
  total = weighted = 0.f;
#pragma unroll
  for (uint32_t w = 0; w < WAVES; w++) {
    total += red[1][w];
    weighted += red[2][w];
  }
  constexpr float LN2 = 0.69314718055994531f;
  const bool nothing = low && total == 0.f;  // every logit is -inf (a NaN would be in the sum)
  const float log_total = logf(total);
  auto logp = [&](float v) { return nothing ? -INFINITY : ((v - m) * c) * LN2 - log_total; };
  if (tid == 0) {
    if (p.logprob) p.logprob[r] = in_vocab ? logp(given) : -INFINITY;
    if (p.entropy) p.entropy[r] = nothing ? 0.f : log_total - weighted / total * LN2;
  }
  if (!K) return;
  __syncthreads();
  auto answer = [&](uint32_t place, unsigned long long key) {
    if (p.top_ids) p.top_ids[(size_t)r * K + place] = ~(uint32_t)key;
    if (p.top_logprobs) p.top_logprobs[(size_t)r * K + place] = logp(value_of((uint32_t)(key >> 32)));
  };
  const uint32_t least = bound;

  // ---- the neighbourhoods that reach the bound, and every logit of theirs that does
  if (by_hood) {
    for (uint32_t n = tid; n < hoods; n += NT)
      if (hood_order(n) >= least) chosen[atomicAdd(&chosen_count, 1u)] = (uint16_t)n;
    __syncthreads();
  }
  // f(value, id) for every logit that can be among the best
  auto each = [&](auto&& f) {
    if (by_hood) {
      for (uint32_t k = wave; k < chosen_count; k += WAVES) {
        const uint32_t from = (uint32_t)chosen[k] * hood_size<T>;
        Group<T> x[2];
#pragma unroll
        for (uint32_t g = 0; g < 2; g++) x[g] = load_group(row, lead, p.vocab, from + (g * 64 + lane) * N);
#pragma unroll
        for (uint32_t g = 0; g < 2; g++) {
          const uint32_t at = from + (g * 64 + lane) * N;
#pragma unroll
          for (uint32_t i = 0; i < N; i++)
            if (at + i >= lead && at + i < lead + p.vocab) f((float)x[g][i], at + i - lead);
        }
      }
    } else {
      for (uint32_t i = tid; i < p.vocab; i += NT) f((float)row[i], i);
    }
  };
  auto collect = [&](uint32_t from) {  // logits whose order is at least `from`
    each([&](float v, uint32_t id) {
      if (order_of(v) >= from) {
        const uint32_t at = atomicAdd(&count, 1u);
        if (at < MAX_CANDIDATES) candidates[at] = rank_key(v, id);
      }
    });
    __syncthreads();
  };
  auto rank = [&](uint32_t n) {  // places of the first n candidates
    for (uint32_t i = tid; i < n; i += NT) {
      const unsigned long long key = candidates[i];
      uint32_t place = 0;
#pragma unroll 8
      for (uint32_t j = 0; j < n; j++) place += candidates[j] > key;
      if (place < K) answer(place, key);
    }
  };
  collect(least);
  const uint32_t reached = count;
  if (reached >= K && reached <= MAX_CANDIDATES) {
    rank(reached);
    return;
  }
  // ---- many equal logits (a row that is masked but for a few): those above the bound, then the bound's own value in
  // the order of the ids
  __syncthreads();
  if (tid == 0) count = 0;
  __syncthreads();
  if (reached > MAX_CANDIDATES) {
    collect(least + 1);
    const uint32_t over = count;
    if (over < K) {
      rank(over);
      uint32_t have = over;
      for (uint32_t i0 = 0; i0 < p.vocab && have < K; i0 += NT) {
        const uint32_t i = i0 + tid;
        const bool hit = i < p.vocab && order_of((float)row[i]) == least;
        const unsigned long long ballot = __ballot(hit);
        if (lane == 0) most[wave] = (uint32_t)__popcll(ballot);
        __syncthreads();
        uint32_t place = have + (uint32_t)__popcll(ballot & ((1ull << lane) - 1ull));
        for (uint32_t w = 0; w < wave; w++) place += most[w];
        if (hit && place < K) answer(place, rank_key((float)row[i], i));
        for (uint32_t w = 0; w < WAVES; w++) have += most[w];
        __syncthreads();
      }
      return;
    }
    if (over <= MAX_CANDIDATES) {
      rank(over);
      return;
    }
  }
  // ---- anything else (rows in order, rows of NaN): one alternative after the other
  unsigned long long last = ~0ull;
  for (uint32_t k = 0; k < K; k++) {
    unsigned long long key = 0;
    auto look = [&](float v, uint32_t id) {
      const unsigned long long x = rank_key(v, id);
      if (x < last && x > key) key = x;
    };
    if (reached >= K) each(look);
    else
      for (uint32_t i = tid; i < p.vocab; i += NT) look((float)row[i], i);
    for (int o = 32; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor(key, o);
      key = other > key ? other : key;
    }
    if (lane == 0) best[wave] = key;
    __syncthreads();
    last = best[0];
    for (uint32_t w = 1; w < WAVES; w++) last = best[w] > last ? best[w] : last;
    __syncthreads();
    if (tid == 0) answer(k, last);
  }
}

template <class T, int NT>
__global__ __launch_bounds__(NT) void logits_answer_kernel(const LogprobsArgs p, const SegmentStats* stats, uint32_t segments, float c) {
  answer_row<T, NT, MAX_SEGMENTS>(p, blockIdx.x, stats + (uint64_t)blockIdx.x * segments, segments, c);
}

template <class T>
__global__ __launch_bounds__(256) void logits_row_kernel(const LogprobsArgs p, uint32_t segments, float c) {
  __shared__ SegmentStats stats[4];
  const uint32_t seg = threadIdx.x >> 6;
  if (seg < segments) {
    const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)blockIdx.x * p.row_stride;
    const SegmentStats s = read_segment(row, lead_of(row), p.vocab, seg, c);
    if ((threadIdx.x & 63u) == 0) stats[seg] = s;
  }
  __syncthreads();
  answer_row<T, 256, 4>(p, blockIdx.x, stats, segments, c);
}

// Segments of a row, whatever its alignment; 0: too long for the table of neighbourhoods.
template <class T>
uint32_t segments_of(uint32_t vocab) {
  if ((uint64_t)vocab + per_load<T> > (uint64_t)MAX_HOODS * hood_size<T>) return 0;
  return (uint32_t)(((uint64_t)vocab + per_load<T> - 1 + segment_size<T> - 1) / segment_size<T>);
}
template <class T>
hipError_t launch_typed(const LogprobsArgs& a, void* scratch, hipStream_t s) {
  const uint32_t segments = segments_of<T>(a.vocab);
  const float c = a.inv_temperature * 1.4426950408889634f;
  if (!segments) {
    hipLaunchKernelGGL(logprobs_any_kernel<T>, dim3(a.rows), dim3(256), 0, s, a);
    return hipGetLastError();
  }
  if (segments <= 4) {
    hipLaunchKernelGGL(logits_row_kernel<T>, dim3(a.rows), dim3(256), 0, s, a, segments, c);
    return hipGetLastError();
  }
  SegmentStats* stats = static_cast<SegmentStats*>(scratch);
  const uint64_t waves = (uint64_t)a.rows * segments;
  hipLaunchKernelGGL(logits_segments_kernel<T>, dim3((uint32_t)((waves + 3) / 4)), dim3(256), 0, s, a, stats, segments, c);
  // few rows: as many waves as a row can use; many: as many rows as fit (1024 / 256 threads: a row of
  // 128000 logits 11.0 / 12.4 us; of 32000, 256 rows 15.6 / 17.3, 512 21.9 / 22.5, 700 30.2 / 27.0, 2048 75.9 / 63.8)
  if (a.rows <= 512) hipLaunchKernelGGL((logits_answer_kernel<T, 1024>), dim3(a.rows), dim3(1024), 0, s, a, stats, segments, c);
  else hipLaunchKernelGGL((logits_answer_kernel<T, 256>), dim3(a.rows), dim3(256), 0, s, a, stats, segments, c);
  return hipGetLastError();
}

}  // namespace

size_t logprobs_scratch_bytes(const LogprobsArgs& a) {
  const uint32_t segments = a.f16 ? segments_of<_Float16>(a.vocab) : segments_of<float>(a.vocab);
  return segments > 4 ? (size_t)a.rows * segments * sizeof(SegmentStats) : 0;
}

hipError_t launch_logprobs(const LogprobsArgs& a, void* scratch, hipStream_t s) {
  return a.f16 ? launch_typed<_Float16>(a, scratch, s) : launch_typed<float>(a, scratch, s);
}

}  // namespace ztvm
