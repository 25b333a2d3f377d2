// Log probabilities of given ids, the entropy and the likeliest ids of logits rows.
//
// With d_i = x_i - max x and the sum l' of exp(d_i) over all ids but the (first) maximum:
//   log p_i = d_i - log1p(l'),   entropy = log1p(l') - sum_i exp(d_i) d_i / (1 + l').
// Keeping the maximum's own 1 out of the sum keeps log p of a nearly certain id exact to f32.
// Nothing here allocates, keeps state between calls or synchronizes.
#include "kernels.h"

namespace qc {
namespace {

// Order of the alternatives: larger logits first, equal ones by the lower id; NaN below everything.
__device__ __forceinline__ unsigned long long logit_key(float x, uint32_t id) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 counts as 0)
  const uint32_t k = x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
  return (unsigned long long)k << 32 | (0xffffffffu - id);
}

template <class T, class F>
__device__ T block_fold(T x, T* tmp, F f) {
  for (int o = 16; o; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = x;
  __syncthreads();
  x = tmp[0];
  for (uint32_t w = 1; w < blockDim.x / 32; w++) x = f(x, tmp[w]);
  return x;
}

__global__ void __launch_bounds__(512) k_logprobs(LogprobArgs a) {
  __shared__ unsigned long long tk[16];
  __shared__ float tf[16];
  const uint32_t row = blockIdx.x;
  const float* x = a.logits + (uint64_t)(a.src ? a.src[row] : row) * a.stride;
  unsigned long long best = 0;
  float mx = -INFINITY;
  bool nan = false;
  for (uint32_t i = threadIdx.x; i < a.n; i += blockDim.x) {
    const unsigned long long k = logit_key(x[i], i);
    best = k > best ? k : best;
    mx = fmaxf(mx, x[i]);
    nan |= x[i] != x[i];
  }
  best = block_fold(best, tk, [](unsigned long long u, unsigned long long v) { return u > v ? u : v; });
  mx = block_fold(mx, tf, [](float u, float v) { return fmaxf(u, v); });
  nan = __syncthreads_or(nan);
  const uint32_t arg = 0xffffffffu - (uint32_t)best;
  float l = 0.f, t = 0.f;
  for (uint32_t i0 = threadIdx.x; i0 < a.n; i0 += 64 * blockDim.x) {  // sums of sums: few additions in a row
    float pl = 0.f, pt = 0.f;
    for (uint32_t i = i0; i < min(a.n, i0 + 64 * blockDim.x); i += blockDim.x) {
      const float d = x[i] - mx, ex = expf(d);
      if (i != arg) pl += ex;
      if (ex > 0.f) pt = fmaf(ex, d, pt);
    }
    l += pl;
    t += pt;
  }
  l = block_fold(l, tf, [](float u, float v) { return u + v; });
  t = block_fold(t, tf, [](float u, float v) { return u + v; });
  const float qnan = __int_as_float(0x7fc00000);
  const bool ok = !nan && isfinite(mx);
  const float lg = log1pf(l);
  auto lp = [&](float v) { return ok ? (v - mx) - lg : qnan; };
  for (uint32_t j = threadIdx.x; j < a.n_ids; j += blockDim.x) {
    const uint32_t id = a.ids[(uint64_t)row * a.n_ids + j];
    a.logprobs[(uint64_t)row * a.n_ids + j] = id < a.n ? lp(x[id]) : qnan;
  }
  if (a.entropy && threadIdx.x == 0) a.entropy[row] = ok ? lg - t / (1.f + l) : qnan;
  unsigned long long last = ~0ull;
  for (uint32_t j = 0; j < a.top; j++) {
    best = 0;
    for (uint32_t i = threadIdx.x; i < a.n; i += blockDim.x) {
      const unsigned long long k = logit_key(x[i], i);
      if (k < last && k > best) best = k;
    }
    best = block_fold(best, tk, [](unsigned long long u, unsigned long long v) { return u > v ? u : v; });
    last = best;
    const uint32_t id = 0xffffffffu - (uint32_t)best;
    if (threadIdx.x == 0) {
      a.top_ids[(uint64_t)row * a.top + j] = id;
      a.top_logprobs[(uint64_t)row * a.top + j] = lp(x[id]);
    }
  }
}

}  // namespace

cudaError_t launch_logprobs(const LogprobArgs& a, cudaStream_t st) {
  k_logprobs<<<a.rows, 512, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace qc
