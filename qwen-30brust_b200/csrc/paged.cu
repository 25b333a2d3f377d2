// Paged key-value cache of one layer: append, attention of new tokens, eviction by accumulated
// attention weight.
//
// The cache is two pools of pages [n_pages][kvheads][page][D] (keys, values; f32, f16 or bf16) and a
// table [n_seqs][max_pages] of page numbers: slot j of sequence s lies in page table[s][j / page] at
// slot j % page.  The order within a page is the contiguous cache's ([kv head][position][D], batch.cu).
// Nothing here allocates, keeps state between calls or synchronizes, so every call can be captured,
// and calls on different data may overlap.
//
// Page numbers, sequence numbers and lengths are device data that the host cannot check, so every
// kernel checks them against the pools' and the table's sizes before it uses them.
#include <cuda_bf16.h>
#include <float.h>

#include "kernels.h"

namespace qc {
namespace {

constexpr uint32_t kMaxD = 256;

template <class T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Row number (of D elements) of slot j of sequence s and KV head h in a pool; the page must be valid.
__device__ __forceinline__ uint64_t pool_row(const PagedKV& c, const uint32_t* table, uint32_t s, uint32_t h, uint32_t j) {
  const uint32_t p = table[(uint64_t)s * c.max_pages + j / c.page];
  return ((uint64_t)p * c.kvheads + h) * c.page + j % c.page;
}

// Row i's k and v (f32, rounded to nearest) to slot pos[i] of sequence seq[i]; its weights become 0.
template <class T>
__global__ void __launch_bounds__(256) k_paged_append(PagedKV c, const float* __restrict__ k, const float* __restrict__ v,
                                                       const uint32_t* __restrict__ seq, const uint32_t* __restrict__ pos,
                                                       float* __restrict__ weights) {
  const uint32_t i = blockIdx.x, s = seq ? seq[i] : i, j = pos[i];
  if (s >= c.n_seqs || j >= c.max_pages * c.page) return;
  if (c.table[(uint64_t)s * c.max_pages + j / c.page] >= c.n_pages) return;
  for (uint32_t e = threadIdx.x; e < c.kvheads * c.D; e += blockDim.x) {
    const uint32_t h = e / c.D, d = e % c.D;
    const uint64_t o = pool_row(c, c.table, s, h, j) * c.D + d, from = (uint64_t)i * c.kvheads * c.D + e;
    static_cast<T*>(c.k)[o] = from_float<T>(k[from]);
    static_cast<T*>(c.v)[o] = from_float<T>(v[from]);
  }
  if (weights)
    for (uint32_t h = threadIdx.x; h < c.kvheads; h += blockDim.x)
      weights[((uint64_t)s * c.kvheads + h) * c.max_pages * c.page + j] = 0.f;
}

// One block a (row, KV head); with weights, the block of a sequence's first row takes all its rows.
template <class T>
__global__ void __launch_bounds__(256) k_paged_attention(PagedKV c, PagedRows r) {
  __shared__ float sm[8], sl[8], sacc[8][kMaxD];
  __shared__ float hm[32], hl[32];  // every head's maximum and sum
  __shared__ uint32_t s_bad;
  const uint32_t h = blockIdx.x % c.kvheads, first = blockIdx.x / c.kvheads, D = c.D, G = r.heads / c.kvheads;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cap = c.max_pages * c.page;
  const uint32_t s = r.seq ? r.seq[first] : first;
  if (s >= c.n_seqs) return;
  if (r.weights && r.seq)
    for (uint32_t i = 0; i < first; i++)
      if (r.seq[i] == s) return;
  for (uint32_t i = first; i < r.rows; i++) {
    if (i > first && (!r.weights || !r.seq)) break;
    if (r.seq && r.seq[i] != s) continue;
    const uint32_t len = r.len[i];
    __syncthreads();
    if (threadIdx.x == 0) s_bad = len > cap;
    __syncthreads();
    if (len <= cap)
      for (uint32_t p = threadIdx.x; p < (len + c.page - 1) / c.page; p += blockDim.x)
        if (c.table[(uint64_t)s * c.max_pages + p] >= c.n_pages) s_bad = 1;
    __syncthreads();
    const bool bad = s_bad;
    for (uint32_t g = 0; g < G; g++) {
      const uint64_t qh = (uint64_t)i * r.heads + h * G + g;
      float* out = r.out + qh * D;
      if (bad || len == 0) {
        for (uint32_t d = threadIdx.x; d < D; d += blockDim.x) out[d] = bad ? __int_as_float(0x7fc00000) : 0.f;
        if (r.lse && threadIdx.x == 0) r.lse[qh] = bad ? __int_as_float(0x7fc00000) : -INFINITY;
        continue;
      }
      float q[kMaxD / 32], acc[kMaxD / 32], m = -FLT_MAX, l = 0.f;
#pragma unroll
      for (uint32_t t = 0; t < kMaxD / 32; t++) {
        q[t] = lane + 32 * t < D ? r.q[qh * D + lane + 32 * t] : 0.f;
        acc[t] = 0.f;
      }
      auto score = [&](uint32_t j) {
        const T* kr = static_cast<const T*>(c.k) + pool_row(c, c.table, s, h, j) * D;
        float dot = 0.f;
#pragma unroll
        for (uint32_t t = 0; t < kMaxD / 32; t++)
          if (lane + 32 * t < D) dot = fmaf(q[t], to_float<T>(kr[lane + 32 * t]), dot);
        for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        return dot * r.scale;
      };
      for (uint32_t j = warp; j < len; j += 8) {
        const float x = score(j), mn = fmaxf(m, x), f = expf(m - mn), p = expf(x - mn);
        const T* vr = static_cast<const T*>(c.v) + pool_row(c, c.table, s, h, j) * D;
        m = mn;
        l = l * f + p;
#pragma unroll
        for (uint32_t t = 0; t < kMaxD / 32; t++)
          if (lane + 32 * t < D) acc[t] = fmaf(acc[t], f, p * to_float<T>(vr[lane + 32 * t]));
      }
      if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
      }
      for (uint32_t t = 0; t < kMaxD / 32; t++)
        if (lane + 32 * t < D) sacc[warp][lane + 32 * t] = acc[t];
      __syncthreads();
      float M = sm[0], L = 0.f;
      for (int w = 1; w < 8; w++) M = fmaxf(M, sm[w]);
      for (int w = 0; w < 8; w++)
        L += sl[w] * expf(sm[w] - M);
      for (uint32_t d = threadIdx.x; d < D; d += blockDim.x) {
        float o = 0.f;
        for (int w = 0; w < 8; w++) o = fmaf(sacc[w][d], expf(sm[w] - M), o);
        out[d] = L == 0.f ? 0.f : o / L;
      }
      if (r.lse && threadIdx.x == 0) r.lse[qh] = M + logf(L);
      if (threadIdx.x == 0) {
        hm[g] = M;
        hl[g] = L;
      }
      __syncthreads();
    }
    if (!r.weights || bad) continue;
    for (uint32_t j = warp; j < len; j += 8) {
      const T* kr = static_cast<const T*>(c.k) + pool_row(c, c.table, s, h, j) * D;
      float sum = 0.f;
      for (uint32_t g = 0; g < G; g++) {
        const float* qr = r.q + ((uint64_t)i * r.heads + h * G + g) * D;
        float dot = 0.f;
        for (uint32_t t = lane; t < D; t += 32) dot = fmaf(qr[t], to_float<T>(kr[t]), dot);
        for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (hl[g] != 0.f) sum += expf(dot * r.scale - hm[g]) / hl[g];
      }
      if (lane == 0) r.weights[((uint64_t)s * c.kvheads + h) * cap + j] += sum;
    }
  }
}

// A weight's place in the order of eviction: larger weights have larger keys, NaN the smallest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t b = __float_as_uint(w + 0.f);  // (-0 counts as 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ uint32_t block_sum(uint32_t x, uint32_t* tmp) {
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0;
  for (uint32_t w = 0; w < blockDim.x / 32; w++) x += tmp[w];
  return x;
}

// The slots that (sequence, KV head) keeps, ascending, to kept[..][keep]; kNoSlot behind them, and in
// the first place when the sequence's length or pages are invalid.
__global__ void __launch_bounds__(1024) k_evict_select(PagedKV c, PagedEvict e) {
  __shared__ uint32_t tmp[32], s_bad, s_at;
  const uint32_t s = blockIdx.x / c.kvheads, tid = threadIdx.x;
  const uint32_t n = e.len[s], cap = c.max_pages * c.page, m = min(n, e.keep);
  uint32_t* kept = e.kept + (uint64_t)blockIdx.x * e.keep;
  if (tid == 0) {
    s_bad = n > cap;
    s_at = 0;
  }
  __syncthreads();
  if (n <= cap) {
    for (uint32_t p = tid; p < (n + c.page - 1) / c.page; p += blockDim.x)
      if (c.table[(uint64_t)s * c.max_pages + p] >= c.n_pages) s_bad = 1;
    for (uint32_t p = tid; p < (m + c.page - 1) / c.page; p += blockDim.x)
      if (e.dst_table[(uint64_t)s * c.max_pages + p] >= c.n_pages) s_bad = 1;
  }
  __syncthreads();
  if (s_bad || n <= e.keep) {
    for (uint32_t i = tid; i < e.keep; i += blockDim.x) kept[i] = !s_bad && i < n ? i : kNoSlot;
    return;
  }
  const float* w = e.weights + (uint64_t)blockIdx.x * cap;
  const uint32_t old = n - e.recent, want = e.keep - e.recent;
  uint32_t T = 0;  // the want-th largest key
  for (int b = 31; b >= 0 && want; b--) {
    const uint32_t cand = T | 1u << b;
    uint32_t cnt = 0;
    for (uint32_t i = tid; i < old; i += blockDim.x) cnt += weight_key(w[i]) >= cand;
    if (block_sum(cnt, tmp) >= want) T = cand;
  }
  uint32_t above = 0;
  for (uint32_t i = tid; i < old; i += blockDim.x) above += weight_key(w[i]) > T;
  uint32_t ties = want - block_sum(above, tmp);  // slots with key T that stay: the first ones
  if (!want) ties = 0;
  __syncthreads();
  if (tid == 0)
    for (uint32_t i = 0; i < n; i++) {
      const uint32_t key = i < old ? weight_key(w[i]) : 0;
      bool take = i >= old || (want && key > T);
      if (i < old && want && key == T && ties) {
        take = true;
        ties--;
      }
      if (take) kept[s_at++] = i;
    }
}

// Rows kept[i] of K (blockIdx.y 0) or V (1) and their weights to slot i.  In place this is a move to
// lower slots: kept[i] >= i ascending, so a tile may be written once it has been read.
template <class T>
__global__ void __launch_bounds__(256) k_evict_move(PagedKV c, PagedEvict e) {
  const uint32_t s = blockIdx.x / c.kvheads, h = blockIdx.x % c.kvheads, D = c.D, cap = c.max_pages * c.page;
  const uint32_t* kept = e.kept + (uint64_t)blockIdx.x * e.keep;
  if (kept[0] == kNoSlot) {  // nothing cached, or an invalid sequence
    if (h == 0 && blockIdx.y == 0 && threadIdx.x == 0) e.new_len[s] = e.len[s];
    return;
  }
  const uint32_t m = min(e.len[s], e.keep);
  T* pool = static_cast<T*>(blockIdx.y ? c.v : c.k);
  const float* w = e.weights + (uint64_t)blockIdx.x * cap;
  float* wo = e.weights_out + (uint64_t)blockIdx.x * cap;
  for (uint32_t i = 0; i < m; i++) {
    const uint64_t from = pool_row(c, c.table, s, h, kept[i]), to = pool_row(c, e.dst_table, s, h, i);
    T x{};
    float y = 0.f;
    if (threadIdx.x < D) x = pool[from * D + threadIdx.x];
    if (threadIdx.x == 0 && !blockIdx.y) y = w[kept[i]];
    __syncthreads();
    if (threadIdx.x < D) pool[to * D + threadIdx.x] = x;
    if (threadIdx.x == 0 && !blockIdx.y) wo[i] = y;
    __syncthreads();
  }
  if (h == 0 && blockIdx.y == 0 && threadIdx.x == 0) e.new_len[s] = m;
}

}  // namespace

cudaError_t paged_prepare() { return cudaSuccess; }

#define QC_BY_KIND(KIND, CALL)                        \
  switch (KIND) {                                     \
    case F32: { using T = float; CALL; break; }       \
    case F16: { using T = __half; CALL; break; }      \
    default: { using T = __nv_bfloat16; CALL; break; } \
  }

cudaError_t launch_paged_append(const PagedKV& c, const float* k, const float* v, uint32_t rows, const uint32_t* seq,
                                const uint32_t* pos, float* weights, cudaStream_t st) {
  QC_BY_KIND(c.kind, (k_paged_append<T><<<rows, 256, 0, st>>>(c, k, v, seq, pos, weights)));
  return cudaGetLastError();
}

cudaError_t launch_paged_attention(const PagedKV& c, const PagedRows& r, cudaStream_t st) {
  QC_BY_KIND(c.kind, (k_paged_attention<T><<<r.rows * c.kvheads, 256, 0, st>>>(c, r)));
  return cudaGetLastError();
}

cudaError_t launch_paged_evict(const PagedKV& c, const PagedEvict& e, cudaStream_t st) {
  k_evict_select<<<c.n_seqs * c.kvheads, 1024, 0, st>>>(c, e);
  QC_BY_KIND(c.kind, (k_evict_move<T><<<dim3(c.n_seqs * c.kvheads, 2), 256, 0, st>>>(c, e)));
  return cudaGetLastError();
}

}  // namespace qc
