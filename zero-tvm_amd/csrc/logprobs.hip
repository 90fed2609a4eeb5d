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

// One workgroup per row, one pass for the maximum, one for the sums, one for each alternative.
template <class T>
__global__ __launch_bounds__(256) void logprobs_kernel(const LogprobsArgs p) {
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

}  // namespace

hipError_t launch_logprobs(const LogprobsArgs& a, hipStream_t s) {
  if (a.f16) hipLaunchKernelGGL(logprobs_kernel<_Float16>, dim3(a.rows), dim3(256), 0, s, a);
  else hipLaunchKernelGGL(logprobs_kernel<float>, dim3(a.rows), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace ztvm
