// Log probabilities of given ids, the entropy and the likeliest ids of logits rows.
//
// With m = max x, d_i = x_i - m and l' the sum of exp(d_i) over all ids but one of the largest:
//   log p_i = d_i - log1p(l'),   entropy = log1p(l') - t / (1 + l'),   t = sum_i exp(d_i) d_i.
// Keeping the maximum's own 1 out of the sum keeps log p of a nearly certain id exact to f32.  Two parts
// of a row join as
//   l' = l'_a + (1 + l'_b) f,  t = t_a + f (t_b + (m_b - m_a)(1 + l'_b)),  f = exp(m_b - m_a),  m_a >= m_b;
// the empty part is (-FLT_MAX, -1, 0).
//
// One pass over the row: a cluster of up to 16 blocks shares it, and a block's warps take chunks of 512
// values (128 where a block has few) in turn, 16 a lane in registers.  A warp sums its values relative to
// its own running maximum and keeps the values above the block's threshold.  The threshold needs no
// selection among the values: a warp's largest lane maxima are different values, so the k-th largest of
// the warps' has k values at or above it; it is taken after the first chunk, and again after the second
// and the eighth.  A warp whose room for candidates runs out selects its k best and goes by them.  The
// warps' parts are joined in shared memory, the blocks' parts and k best through distributed shared
// memory.  No workspace, no atomics on global memory; the sums' order is fixed.  (Candidates are listed and ranked with
// atomics in shared memory: their keys differ, so their order does not depend on it.)  VEC = 4 spills 44 bytes a
// thread to hold four blocks an SM.
#include <float.h>

#include "kernels.h"

namespace qc {
namespace {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kLpTurns = 3;                        // thresholds: before chunk 0, and after 2 and 8
constexpr int kLpTop = 16;                         // lane maxima a warp shows for them, at most
constexpr int kLpMaxCluster = 16;
constexpr uint32_t kLpKeep = 128;  // candidates a warp has room for

// Order of the alternatives: larger logits first, equal ones by the lower id; NaN below everything.
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 counts as 0)
  return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {  // (0: NaN)
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : k ? ~k : 0x7fc00000u);
}
__device__ __forceinline__ unsigned long long full_key(uint32_t k, uint32_t id) {
  return (unsigned long long)k << 32 | (0xffffffffu - id);
}

// Two f32 in one register pair (add, multiply, fused multiply-add to nearest, both at once).
struct F2 {
  unsigned long long v;
  __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ float2 get() const {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
};
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(a.v) : "l"(a.v), "l"(b.v));
  return a;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(a.v) : "l"(a.v), "l"(b.v));
  return a;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(a.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return a;
}

struct Part {
  float m, l, t;
};
__device__ __forceinline__ Part join(Part a, Part b) {
  const bool sw = b.m > a.m;
  const float m = sw ? b.m : a.m, d = (sw ? a.m : b.m) - m, f = expf(d);
  const float la = sw ? b.l : a.l, ta = sw ? b.t : a.t, lb = 1.f + (sw ? a.l : b.l), tb = sw ? a.t : b.t;
  return Part{m, fmaf(lb, f, la), f == 0.f ? ta : ta + f * fmaf(d, lb, tb)};
}

__device__ __forceinline__ uint32_t lp_cluster_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void lp_cluster_arrive() {
  __syncwarp();  // (the barrier wants a warp's threads together)
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void lp_cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Shared memory; behind it the chunks on their way, later the block's candidates.
struct LpShared {
  unsigned long long kept[kLpWarps][kLpKeep];          // a warp's candidates
  unsigned long long best[kMaxTop];                    // the block's k best, sorted
  unsigned long long in_best[kLpMaxCluster][kMaxTop];  // every block's
  Part in_part[kLpMaxCluster], warp_part[kLpWarps];
  uint32_t in_n[kLpMaxCluster], warp_n[kLpWarps], rank[kMaxTop];
  uint32_t shown[kLpTurns][kLpWarps * kLpTop];         // the warps' largest lane maxima (keys)
};
constexpr int kLpAhead = 2;  // chunks of a warp on their way
template <int VEC>
constexpr uint32_t kLpSmem = sizeof(LpShared) + kLpWarps * kLpAhead * VEC * 512 > sizeof(LpShared) + kLpWarps * kLpKeep * 8
                                 ? sizeof(LpShared) + kLpWarps * kLpAhead * VEC * 512
                                 : sizeof(LpShared) + kLpWarps * kLpKeep * 8;
static_assert(kLpKeep * kLpWarps % kLpThreads == 0 && sizeof(LpShared) % 16 == 0, "chunks are 16-byte aligned");

// 2^x to 2 ulp (results below 2^-126 are 0)
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The k largest of list[0, n), sorted, to sh.best (n <= 4 kLpThreads, the keys differ).  Of many keys first
// those whose value reaches the k-th largest's, up to ten bits behind the bits that all share; then a key's
// place is the number of larger ones, which four lanes count.  `other` has room for n keys.
__device__ __forceinline__ void select_best(LpShared& sh, const unsigned long long* list, unsigned long long* other, uint32_t n,
                                            uint32_t k) {
  const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  if (n > 96 && n > k) {
    uint32_t key[kLpKeep * kLpWarps / kLpThreads], hi = 0, lo = 0xffffffffu;
#pragma unroll
    for (uint32_t u = 0; u < kLpKeep * kLpWarps / kLpThreads; u++) {
      key[u] = tid + u * kLpThreads < n ? (uint32_t)(list[tid + u * kLpThreads] >> 32) : 0;
      hi = max(hi, key[u]);
      if (tid + u * kLpThreads < n) lo = min(lo, key[u]);
    }
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo);
    if (lane == 0) {
      sh.shown[0][warp] = hi;
      sh.shown[0][kLpWarps + warp] = lo;
    }
    if (tid == 0) sh.warp_n[0] = 0;
    __syncthreads();
    for (uint32_t v = 0; v < kLpWarps; v++) {
      hi = max(hi, sh.shown[0][v]);
      lo = min(lo, sh.shown[0][kLpWarps + v]);
    }
    const int same = hi == lo ? 32 : __clz(hi ^ lo), end = max(0, 32 - same - 10);
    uint32_t T = same ? hi & ~(0xffffffffu >> (same - 1) >> 1) : 0, turn = 1;
    for (int b = 31 - same; b >= end; b--, turn = 3 - turn) {  // (counts alternate between two places)
      uint32_t count = 0;
#pragma unroll
      for (uint32_t u = 0; u < kLpKeep * kLpWarps / kLpThreads; u++)
        count += tid + u * kLpThreads < n && key[u] >= (T | 1u << b);
      count = __reduce_add_sync(0xffffffffu, count);
      if (lane == 0) sh.shown[turn][warp] = count;
      __syncthreads();
      count = 0;
#pragma unroll
      for (uint32_t v = 0; v < kLpWarps; v++) count += sh.shown[turn][v];
      if (count >= k) T |= 1u << b;
    }
#pragma unroll
    for (uint32_t u = 0; u < kLpKeep * kLpWarps / kLpThreads; u++)
      if (tid + u * kLpThreads < n && key[u] >= T) other[atomicAdd(&sh.warp_n[0], 1)] = list[tid + u * kLpThreads];
    __syncthreads();
    n = sh.warp_n[0];
    list = other;
  }
  for (uint32_t i0 = 0; i0 < n; i0 += kLpThreads / 4) {
    const uint32_t i = i0 + tid / 4;
    const unsigned long long x = i < n ? list[i] : 0;
    uint32_t above = 0;
#pragma unroll 8
    for (uint32_t j = tid % 4; j < n; j += 4) above += list[j] > x;
    above += __shfl_xor_sync(0xffffffffu, above, 1);
    above += __shfl_xor_sync(0xffffffffu, above, 2);
    if (i < n && above < k && tid % 4 == 0) sh.best[above] = x;
  }
  __syncthreads();
}

// The warp's k largest of kept[0, n), sorted (k < n <= kLpKeep).
__device__ __noinline__ void shrink(unsigned long long* kept, uint32_t n, uint32_t k) {
  const uint32_t lane = threadIdx.x % 32;
  unsigned long long x[kLpKeep / 32];
  uint32_t above[kLpKeep / 32];
#pragma unroll
  for (uint32_t u = 0; u < kLpKeep / 32; u++) {
    x[u] = lane + 32 * u < n ? kept[lane + 32 * u] : 0;
    above[u] = 0;
    if (32 * u < n) {
#pragma unroll 4
      for (uint32_t j = 0; j < n; j++) above[u] += kept[j] > x[u];
    }
  }
  __syncwarp();
#pragma unroll
  for (uint32_t u = 0; u < kLpKeep / 32; u++)
    if (lane + 32 * u < n && above[u] < k) kept[above[u]] = x[u];
  __syncwarp();
}

// VEC 16-byte pieces a lane and chunk.
template <int VEC>
__global__ void __launch_bounds__(kLpThreads, 4) k_logprobs(LogprobArgs a, uint32_t logc) {
  constexpr uint32_t kLpVec = VEC, kLpChunk = 32 * VEC;
  extern __shared__ __align__(16) uint8_t lp_smem[];
  LpShared& sh = *reinterpret_cast<LpShared*>(lp_smem);
  uint8_t* const behind = lp_smem + sizeof(LpShared);
  const uint32_t C = 1u << logc, rank = blockIdx.x & (C - 1), row = blockIdx.x >> logc, tid = threadIdx.x;
  const uint32_t warp = tid / 32, lane = tid % 32, n = a.n, k = a.top;
  lp_cluster_arrive();  // this block runs: it may be written to
  const float* x = a.logits + (uint64_t)(a.src ? a.src[row] : row) * a.stride;
  // 16-byte pieces of the row; piece 0 starts at the boundary at or before x[0]
  const uint32_t shift = (uint32_t)(reinterpret_cast<uintptr_t>(x) / 4 % 4);
  const float4* x4 = reinterpret_cast<const float4*>(x - shift);
  const uint32_t pieces = (n + shift + 3) / 4, per = (pieces + C - 1) / C;
  const uint32_t p0 = min(pieces, rank * per), p1 = min(pieces, p0 + per);

  // Starts copying a chunk from piece `from` on to the warp's buffer of its number; -inf where the row has
  // no values (they add nothing, and ids behind n are no candidates).
  auto fetch = [&](uint32_t from, uint32_t number) {
    uint8_t* const to = behind + ((warp * kLpAhead + number % kLpAhead) * kLpVec * 32 + lane) * 16;
    if (from > 0 && from + kLpChunk <= p1 && (from + kLpChunk) * 4 <= n + shift) {
#pragma unroll
      for (uint32_t j = 0; j < kLpVec; j++)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to + j * 512)),
                     "l"(x4 + from + j * 32 + lane)
                     : "memory");
    } else {
#pragma unroll
      for (uint32_t j = 0; j < kLpVec; j++)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
          const uint32_t p = from + j * 32 + lane, i = p * 4 + e - shift;  // (wraps below 0)
          reinterpret_cast<float*>(to + j * 512)[e] = p < p1 && i < n ? __ldg(x + i) : -INFINITY;
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // (a lane reads what it copied itself)
  auto load = [&](uint32_t number, float (&v)[kLpVec][4]) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kLpAhead - 1) : "memory");
    const uint8_t* const from = behind + ((warp * kLpAhead + number % kLpAhead) * kLpVec * 32 + lane) * 16;
#pragma unroll
    for (uint32_t j = 0; j < kLpVec; j++) {
      const float4 q = *reinterpret_cast<const float4*>(from + j * 512);
      v[j][0] = q.x, v[j][1] = q.y, v[j][2] = q.z, v[j][3] = q.w;
    }
  };
  constexpr float kLog2e = 1.4426950408889634f;
  float cur[kLpVec][4];
  const uint32_t first = p0 + warp * kLpChunk;
  constexpr uint32_t kStep = kLpWarps * kLpChunk;
#pragma unroll
  for (int i = 0; i < kLpAhead; i++) fetch(first + i * kStep, i);
  load(0, cur);
  fetch(first + kLpAhead * kStep, kLpAhead);
  // relative to the warp's maximum m so far: the sum over smaller values, the number of values equal to it,
  // and the sum of exp(d) d, of this lane's values
  float m = -FLT_MAX, l = 0.f, ties = 0.f, t = 0.f;
  uint32_t kept = 0;
  unsigned long long above = 0;  // candidates have larger keys (0: all are)
  unsigned long long* const mine = sh.kept[warp];
  // warps that have values, and the lane maxima each shows: twice k in all where there are that many
  const uint32_t warps = min((uint32_t)kLpWarps, (p1 - p0 + kLpChunk - 1) / kLpChunk);
  const uint32_t show = warps ? min((uint32_t)kLpTop, (2 * k + warps - 1) / warps) : 0;
  uint32_t lane_max = 0;  // (a key)
  // (the block together, its barrier between) raises the threshold to the k-th largest of what the warps show
  auto raise = [&](uint32_t turn) {
    uint32_t rest = lane_max;
    for (uint32_t i = 0; i < show; i++) {
      const uint32_t key = __reduce_max_sync(0xffffffffu, rest), who = __ballot_sync(0xffffffffu, rest == key);
      if (lane == __ffs(who) - 1) rest = 0;
      if (lane == 0 && warp < warps) sh.shown[turn][i * warps + warp] = key;
    }
    __syncthreads();
    const uint32_t shown = show * warps;
    uint32_t key[kLpWarps * kLpTop / 32], T = 0;
#pragma unroll
    for (uint32_t u = 0; u < kLpWarps * kLpTop / 32; u++) key[u] = lane + 32 * u < shown ? sh.shown[turn][lane + 32 * u] : 0;
    uint32_t hi = key[0], lo = lane < shown ? key[0] : 0xffffffffu;
#pragma unroll
    for (uint32_t u = 1; u < kLpWarps * kLpTop / 32; u++) {
      hi = max(hi, key[u]);
      if (lane + 32 * u < shown) lo = min(lo, key[u]);
    }
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo);
    // ten bits behind those that all share (what it misses adds candidates)
    const int same = hi == lo ? 32 : __clz(hi ^ lo), end = max(0, 32 - same - 10);
    T = same ? hi & ~(0xffffffffu >> (same - 1) >> 1) : 0;
    for (int b = 31 - same; b >= end && shown >= k; b--) {
      uint32_t count = 0;
#pragma unroll
      for (uint32_t u = 0; u < kLpWarps * kLpTop / 32; u++)
        if (32 * u < shown) count += __popc(__ballot_sync(0xffffffffu, key[u] >= (T | 1u << b)));
      if (count >= k) T |= 1u << b;
    }
    if (shown < k) T = 0;
    // (at -inf or below some of the maxima were of lanes without values: everything stays a candidate)
    if (T > value_key(-INFINITY)) above = max(above, ((unsigned long long)T << 32) - 1);
  };
  if (k) {
    float mx = -INFINITY;
#pragma unroll
    for (uint32_t j = 0; j < kLpVec; j++)
#pragma unroll
      for (uint32_t e = 0; e < 4; e++) mx = fmaxf(mx, cur[j][e]);
    lane_max = value_key(mx);
    raise(0);
  }
  const uint32_t rounds = (p1 - p0 + kLpWarps * kLpChunk - 1) / (kLpWarps * kLpChunk);  // (all warps take part in all)
  uint32_t base = first;
  for (uint32_t round = 0; round < rounds; round++, base += kStep) {
    float mx = -INFINITY;
#pragma unroll
    for (uint32_t j = 0; j < kLpVec; j++)
#pragma unroll
      for (uint32_t e = 0; e < 4; e++) mx = fmaxf(mx, cur[j][e]);
    const uint32_t key = value_key(mx), top = __reduce_max_sync(0xffffffffu, key);
    const float bm = key_value(top);
    if (bm > m) {  // (the warp together)
      const float d = m - bm, f = pow2(d * kLog2e), mass = l + ties;
      t = f == 0.f ? 0.f : f * fmaf(d, mass, t);
      l = mass * f;
      ties = 0.f;
      m = bm;
    }
    F2 pl2(0.f, 0.f), pt2(0.f, 0.f);
    const F2 minus_m(-m, -m), log2e(kLog2e, kLog2e);
#pragma unroll
    for (uint32_t j = 0; j < kLpVec; j++)
#pragma unroll
      for (uint32_t e = 0; e < 4; e += 2) {
        const F2 d = add2(F2(cur[j][e], cur[j][e + 1]), minus_m);
        const float2 a = mul2(d, log2e).get();
        const F2 ex(pow2(a.x), pow2(a.y));
        pl2 = add2(pl2, ex);
        pt2 = fma2(ex, d, pt2);
      }
    float pl = pl2.get().x + pl2.get().y, pt = pt2.get().x + pt2.get().y;
    if (__any_sync(0xffffffffu, !(pt > -INFINITY))) {  // 0 times -inf: masked ids add nothing
      pt = 0.f;
#pragma unroll
      for (uint32_t j = 0; j < kLpVec; j++)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
          const float d = fmaxf(cur[j][e] - m, -1000.f);
          pt = fmaf(pow2(d * kLog2e), d, pt);
        }
    }
    if (mx == m) {  // this lane has the maximum: its values stay out of the sum
      pl = 0.f;
#pragma unroll
      for (uint32_t j = 0; j < kLpVec; j++)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
          const float d = cur[j][e] - m;
          pl += d == 0.f ? 0.f : pow2(d * kLog2e);
          ties += d == 0.f ? 1.f : 0.f;
        }
    }
    l += pl;
    t += pt;
    if (k) {
      lane_max = max(lane_max, key);
      if (round == 1 || round == 7) raise(round == 1 ? 1 : 2);
      if (top >= (uint32_t)(above >> 32) || above == 0) {
        const float low = above ? key_value((uint32_t)(above >> 32)) : -INFINITY;
#pragma unroll
        for (uint32_t j = 0; j < kLpVec; j++)
#pragma unroll
          for (uint32_t e = 0; e < 4; e++) {
            if (!__any_sync(0xffffffffu, !(cur[j][e] < low))) continue;  // (NaN too: it matters where all count)
            const uint32_t id = (base + j * 32 + lane) * 4 + e - shift;
            const unsigned long long fk = full_key(value_key(cur[j][e]), id);
            const uint32_t who = __ballot_sync(0xffffffffu, fk > above && id < n && base + j * 32 + lane < p1);
            if (kept + __popc(who) > kLpKeep) {
              shrink(mine, kept, k);
              kept = k;
              above = max(above, mine[k - 1]);
            }
            if (who >> lane & 1) mine[kept + __popc(who & ((1u << lane) - 1))] = fk;
            kept += __popc(who);
            __syncwarp();
          }
      }
    }
    if (round + 1 < rounds) {
      load(round + 1, cur);
      fetch(base + (kLpAhead + 1) * kStep, round + 1 + kLpAhead);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");  // (nothing lands where the candidates go)

  // the warps' parts and candidates
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    l += __shfl_xor_sync(0xffffffffu, l, o);
    ties += __shfl_xor_sync(0xffffffffu, ties, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  if (lane == 0) {
    sh.warp_part[warp] = Part{m, l + (ties - 1.f), t};
    sh.warp_n[warp] = kept;
  }
  __syncthreads();
  uint32_t have = 0;
  if (k) {
    uint32_t at = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kLpWarps; w++) {
      if (w == warp) at = all;
      all += sh.warp_n[w];
    }
    unsigned long long* const list = reinterpret_cast<unsigned long long*>(behind);
    for (uint32_t i = lane; i < kept; i += 32) list[at + i] = mine[i];
    __syncthreads();
    select_best(sh, list, sh.kept[0], all, k);  // (the kept keys are all in the list)
    have = min(all, k);
  }
  // the block's, to every block
  lp_cluster_wait();  // (they all run)
  if (tid < C) {
    Part part = sh.warp_part[0];
#pragma unroll
    for (int w = 1; w < kLpWarps; w++) part = join(part, sh.warp_part[w]);
    const uint32_t to = lp_cluster_addr(&sh.in_part[rank], tid);
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(part.m) : "memory");
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(part.l) : "memory");
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(part.t) : "memory");
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(lp_cluster_addr(&sh.in_n[rank], tid)), "r"(have) : "memory");
  }
  for (uint32_t e = tid; e < have << logc; e += kLpThreads) {
    const uint32_t to = e & (C - 1), i = e >> logc;
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(lp_cluster_addr(&sh.in_best[rank][i], to)), "l"(sh.best[i])
                 : "memory");
  }
  if (tid < kMaxTop) sh.rank[tid] = tid;
  lp_cluster_arrive();
  lp_cluster_wait();
  Part all = sh.in_part[0];
  for (uint32_t c = 1; c < C; c++) all = join(all, sh.in_part[c]);
  const float qnan = __int_as_float(0x7fc00000), lg = log1pf(all.l);
  const bool bad = !(all.l >= 0.f);  // NaN, +inf, or nothing above -inf
  auto lp = [&](float v) { return bad ? qnan : (v - all.m) - lg; };
  if (rank == 0) {
    for (uint32_t j = tid; j < a.n_ids; j += kLpThreads) {
      const uint32_t id = a.ids[(uint64_t)row * a.n_ids + j];
      a.logprobs[(uint64_t)row * a.n_ids + j] = id < n ? lp(x[id]) : qnan;
    }
    if (a.entropy && tid == 0) a.entropy[row] = bad ? qnan : lg - all.t / (1.f + all.l);
  }
  // this block's best among everyone's: a key's place is its own plus the larger keys of the others
  for (uint32_t e = tid; e < have << logc; e += kLpThreads) {
    const uint32_t c = e & (C - 1), i = e >> logc;
    if (c == rank) continue;
    const unsigned long long key = sh.best[i];
    uint32_t lo = 0, hi = sh.in_n[c];  // the first of c's keys (falling) that is smaller
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (sh.in_best[c][mid] > key)
        lo = mid + 1;
      else
        hi = mid;
    }
    if (lo) atomicAdd(&sh.rank[i], lo);
  }
  __syncthreads();
  if (tid < have && sh.rank[tid] < k) {
    const unsigned long long key = sh.best[tid];
    const uint64_t at = (uint64_t)row * k + sh.rank[tid];
    a.top_ids[at] = 0xffffffffu - (uint32_t)key;
    a.top_logprobs[at] = lp(key_value((uint32_t)(key >> 32)));
  }
}

}  // namespace

// Once per device, before launch_logprobs.
cudaError_t logprobs_prepare() {
  cudaError_t e = cudaSuccess;
  auto set = [&](void (*f)(LogprobArgs, uint32_t), uint32_t smem) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  };
  set(k_logprobs<1>, kLpSmem<1>);
  set(k_logprobs<4>, kLpSmem<4>);
  return e;
}

// Blocks a row: up to two an SM over all rows, of two chunks a warp at least.  (A block's start and end, its
// thresholds and the exchange, take as long as several chunks: 128 rows of 151,936 values with 5
// alternatives take 28 us with 2 blocks a row, 31 with 4, 40 with 8.)
cudaError_t launch_logprobs(const LogprobArgs& a, cudaStream_t st) {
  uint32_t logc = 0;
  while (logc < 4 && ((uint64_t)a.rows << (logc + 1)) <= 2 * kSMs && a.n > (kLpWarps * 1024u) << logc) logc++;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.rows << logc);
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1u << logc;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const bool few = a.n < kLpWarps * 512u;
  cfg.dynamicSmemBytes = few ? kLpSmem<1> : kLpSmem<4>;
  return cudaLaunchKernelEx(&cfg, few ? k_logprobs<1> : k_logprobs<4>, a, logc);
}

}  // namespace qc
