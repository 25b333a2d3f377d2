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

// ---- attention ---------------------------------------------------------------------------------
// A cluster of C blocks takes one (row, KV head); its warps take 16-position tiles of the sequence in
// turn (tile t goes to warp t mod C W), each with its own running softmax, so a tile needs no block
// barrier.  A warp keeps NS tiles of K and V in flight with 16-byte asynchronous copies, and computes
// per tile, for up to 8 query heads at once (N = 8), on the matrix units:
//   S^T [16 positions x 8 heads] = K q^T          (K rows are the A operand as they lie)
//   O^T [D x 8 heads]           += V^T P^T        (V read transposed; P^T by an 8x8 register transpose)
// The operands keep f32 accuracy: q and p are split into planes of the page type whose sum is exact to
// 2^-22 (f16: two, scaled by a power of two to stay in range) or 2^-24 (bf16: three); f32 pages are
// split themselves, into two tf32 planes.  A tile's products are added to f32 sums outside the matrix
// units, whose accumulators truncate.  Queries of one KV head share K and V; more than 8 heads take
// another turn over the sequence, 8 at a time.
//
// The warps' (maximum, sum, O) are joined in shared memory, the blocks' through the cluster's
// distributed shared memory in a fixed order: no workspace, no atomics, the same bits every time.
// With weights the scores stay in shared memory (512 bytes a tile) until the final maximum and sum are
// known; tiles beyond that room are scored again.

constexpr int kTile = 16;

template <class T, int DP>
struct Att {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kKS = kF32 ? DP / 8 : DP / 16;              // k steps of the score product
  static constexpr int kQP = sizeof(T) == 4 ? 2 : (__is_same(T, __half) ? 2 : 3);  // planes of q and of p
  static constexpr int kRow = DP * (int)sizeof(T) + 16;            // bytes of a tile row: odd multiples of 16 bytes
  static constexpr int kStage = 2 * kTile * kRow;                  //   apart, so 8 rows never share a bank
  static constexpr int kRoom = 112 * 1024;                         // two blocks on an SM
  static constexpr int W = 12 * kStage <= kRoom ? 4 : 2;
  static constexpr int kFit = kRoom / (W * kStage);
  static constexpr int NS = kFit > 4 ? 4 : kFit < 2 ? 2 : kFit;
  static constexpr int kRing = W * NS * kStage;
  static constexpr int kFixed = kRing + 8 * DP * 4 + 128;          // ring, the block's O, maxima, sums, flag
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {  // zeros when not real
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <class T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __half))
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo up to 2^-22 |x|, both with the 11 significant bits of tf32 (hi to nearest, lo cut).
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
// Planes of a pair of values (packed 16-bit): their sum is the pair up to 2^-22 (f16, within its range)
// or 2^-24 (bf16) of it.
template <class T, int P>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&out)[P]) {
#pragma unroll
  for (int p = 0; p < P; p++) {
    if constexpr (__is_same(T, __half)) {
      const __half2 h = __floats2half2_rn(x, y);
      out[p] = *reinterpret_cast<const uint32_t*>(&h);
      x -= __low2float(h);
      y -= __high2float(h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      out[p] = *reinterpret_cast<const uint32_t*>(&h);
      x -= __low2float(h);
      y -= __high2float(h);
    }
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// This block's shared address `a` in block `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// One warp's query operand: the B fragments of q^T for 8 heads, and the factor that undoes q's scaling
// for the two heads whose scores this lane holds.
template <class T, int DP>
struct Query {
  using A = Att<T, DP>;
  uint32_t f[A::kKS][A::kQP][2];
  float undo0, undo1;

  // q: head 0 of the group; heads >= G and values >= D are zero.  factor: scale log2 e.
  __device__ __forceinline__ void load(const float* q, uint32_t D, uint32_t G, float factor) {
    const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane % 4;
    const float* qr = q + (uint64_t)g * D;
    undo0 = undo1 = 1.f;
    if constexpr (A::kF32) {
#pragma unroll
      for (int k = 0; k < A::kKS; k++)
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const uint32_t d = k * 8 + b * 4 + t;
          split_tf32(g < G && d < D ? qr[d] * factor : 0.f, f[k][0][b], f[k][1][b]);
        }
    } else {
      float up = 1.f;
      if constexpr (__is_same(T, __half)) {  // the largest |q| of a head to 2^13..2^14: two planes hold 22 bits
        float mx = 0.f;
        if (g < G)
          for (uint32_t d = t; d < D; d += 4) mx = fmaxf(mx, fabsf(qr[d] * factor));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int e = 13 - ((int)(__float_as_uint(mx) >> 23) - 127);
        e = mx == 0.f || mx > FLT_MAX ? 0 : e > 120 ? 120 : e;
        up = __uint_as_float((uint32_t)(127 + e) << 23);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        undo0 = __shfl_sync(0xffffffffu, down, 8 * t);
        undo1 = __shfl_sync(0xffffffffu, down, 8 * t + 4);
      }
#pragma unroll
      for (int k = 0; k < A::kKS; k++)
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const uint32_t d = k * 16 + b * 8 + 2 * t;
          float2 x = make_float2(0.f, 0.f);
          if (g < G && d < D) x = *reinterpret_cast<const float2*>(qr + d);
          uint32_t pl[A::kQP];
          split_pair<T, A::kQP>(x.x * factor * up, x.y * factor * up, pl);
#pragma unroll
          for (int p = 0; p < A::kQP; p++) f[k][p][b] = pl[p];
        }
    }
  }

  // Scores (times log2 e) of a K tile: s[0], s[1] for position lane / 4 and heads 2 (lane % 4), + 1;
  // s[2], s[3] for position lane / 4 + 8.
  __device__ __forceinline__ void scores(uint32_t ktile, float (&s)[4]) const {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t a0 = ktile + ((lane / 8 % 2) * 8 + lane % 8) * A::kRow + (lane / 16) * 16;
    float c[A::kF32 ? 3 : A::kQP][4];
#pragma unroll
    for (auto& x : c) x[0] = x[1] = x[2] = x[3] = 0.f;
#pragma unroll
    for (int k = 0; k < A::kKS; k++) {
      uint32_t a[4];
      ldsm4(a, a0 + k * 32);
      if constexpr (A::kF32) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split_tf32(__uint_as_float(a[i]), hi[i], lo[i]);
        mma8(c[0], hi, f[k][0][0], f[k][0][1]);
        mma8(c[1], hi, f[k][1][0], f[k][1][1]);
        mma8(c[2], lo, f[k][0][0], f[k][0][1]);
      } else {
#pragma unroll
        for (int p = 0; p < A::kQP; p++) mma16<T>(c[p], a, f[k][p][0], f[k][p][1]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float x = c[0][i];
      if constexpr (A::kF32 || A::kQP == 3)
        x += c[1][i] + c[2][i];
      else
        x += c[1][i];
      s[i] = x * (i % 2 ? undo1 : undo0);
    }
  }
};

// O^T += V^T P^T for one tile; p as Query::scores lays its scores out.
template <class T, int DP>
__device__ __forceinline__ void add_values(uint32_t vtile, const float (&p)[4], float (&o)[DP / 16][4]) {
  using A = Att<T, DP>;
  const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane % 4;
  if constexpr (A::kF32) {
    // k index i of a step of 8 positions stands for position 2 i (i < 4) or 2 (i - 4) + 1: the reads of V
    // then fall on 32 different banks
    uint32_t hi[2][2], lo[2][2];
#pragma unroll
    for (int st = 0; st < 2; st++)
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const uint32_t from = (2 * t + b) * 4 + g / 2;
        const float x = __shfl_sync(0xffffffffu, p[2 * st], from), y = __shfl_sync(0xffffffffu, p[2 * st + 1], from);
        split_tf32(g % 2 ? y : x, hi[st][b], lo[st][b]);
      }
#pragma unroll
    for (int m = 0; m < DP / 16; m++) {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < 2; st++) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float x;
          const uint32_t a = vtile + (st * 8 + 2 * t + i / 2) * A::kRow + (m * 16 + g + (i % 2) * 8) * 4;
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(a) : "memory");
          split_tf32(x, ah[i], al[i]);
        }
        mma8(c, al, hi[st][0], hi[st][1]);
        mma8(c, ah, lo[st][0], lo[st][1]);
        mma8(c, ah, hi[st][0], hi[st][1]);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) o[m][i] += c[i];
    }
  } else {
    uint32_t lo8[A::kQP], hi8[A::kQP];
    const float up = __is_same(T, __half) ? 16384.f : 1.f;  // (undone with the final division)
    split_pair<T, A::kQP>(p[0] * up, p[1] * up, lo8);
    split_pair<T, A::kQP>(p[2] * up, p[3] * up, hi8);
#pragma unroll
    for (int q = 0; q < A::kQP; q++) {
      lo8[q] = transpose8(lo8[q]);
      hi8[q] = transpose8(hi8[q]);
    }
    const uint32_t a0 = vtile + ((lane / 16) * 8 + lane % 8) * A::kRow + (lane / 8 % 2) * 16;
#pragma unroll
    for (int m = 0; m < DP / 16; m++) {
      uint32_t a[4];
      ldsm4_t(a, a0 + m * 32);
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = A::kQP - 1; q >= 0; q--) mma16<T>(c, a, lo8[q], hi8[q]);
#pragma unroll
      for (int i = 0; i < 4; i++) o[m][i] += c[i];
    }
  }
}

template <class T, int DP, bool WEIGHTS>
__global__ void __launch_bounds__(Att<T, DP>::W * 32) k_paged_attention(PagedKV c, PagedRows r, uint32_t score_tiles) {
  using A = Att<T, DP>;
  constexpr int W = A::W, NS = A::NS;
  extern __shared__ __align__(16) uint8_t sm[];
  float* const block_o = reinterpret_cast<float*>(sm + A::kRing);  // [8][DP]
  float* const block_m = block_o + 8 * DP;                         // [8]
  float* const block_l = block_m + 8;                              // [8]
  uint32_t* const block_bad = reinterpret_cast<uint32_t*>(block_l + 8);
  const uint32_t C = cluster_size(), rank = cluster_rank();
  const uint32_t unit = blockIdx.x / C, h = unit % c.kvheads, first = unit / c.kvheads;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane / 4, t = lane % 4;
  const uint32_t D = c.D, G = r.heads / c.kvheads, cap = c.max_pages * c.page, chunks = D * (uint32_t)sizeof(T) / 16;
  uint8_t* const ring = sm + warp * NS * A::kStage;
  const uint32_t ring_a = smem_addr(ring);
  float* const mine = reinterpret_cast<float*>(ring);  // the warp's O [8][DP], maxima and sums, once its tiles are done
  const uint32_t s = r.seq ? r.seq[first] : first;
  if (s >= c.n_seqs) return;  // (the whole cluster)
  if (WEIGHTS && r.seq) {     // the cluster of a sequence's first row takes all its rows, in order
    bool earlier = false;
    for (uint32_t i = tid; i < first; i += W * 32) earlier |= r.seq[i] == s;
    if (__syncthreads_or(earlier)) return;
  }
  const uint32_t* const pages = c.table + (uint64_t)s * c.max_pages;

  for (uint32_t i = first; i < r.rows; i++) {
    if (i > first && !(WEIGHTS && r.seq)) break;
    if (i > first && r.seq[i] != s) continue;
    const uint32_t len = r.len[i];
    const bool too_long = len > cap;
    const uint32_t tiles = too_long ? 0 : (len + kTile - 1) / kTile, gw = rank * W + warp;
    const uint32_t mine_n = tiles > gw ? (tiles - gw + C * W - 1) / (C * W) : 0;  // this warp's tiles
    for (uint32_t g0 = 0; g0 < G; g0 += 8) {
      const uint32_t gn = min(8u, G - g0);
      bool bad = false;
      if (chunks * 16 < DP * sizeof(T)) {  // columns D.. of the tiles are zero (the join below writes over them)
        const uint32_t extra = DP * (uint32_t)sizeof(T) / 16 - chunks;
        for (uint32_t e = lane; e < 2 * NS * kTile * extra; e += 32)
          *reinterpret_cast<uint4*>(ring + (e / extra) * A::kRow + (chunks + e % extra) * 16) = make_uint4(0, 0, 0, 0);
      }
      // The pool row of position lane (< 16) of this warp's n-th tile; kNoSlot: nothing to read.
      auto row_of = [&](uint32_t n) {
        const uint32_t j = (gw + n * C * W) * kTile + lane % kTile;
        if (n >= mine_n || j >= len) return kNoSlot;
        const uint32_t p = pages[j / c.page];
        if (p >= c.n_pages) {
          bad = true;
          return kNoSlot;
        }
        return (p * c.kvheads + h) * c.page + j % c.page;
      };
      auto fetch = [&](uint32_t slot, uint32_t row, bool with_v) {
        const uint32_t dst = ring_a + slot * A::kStage;
        constexpr uint32_t kCh = DP * sizeof(T) / 16;
#pragma unroll 4
        for (uint32_t e = lane; e < kTile * kCh; e += 32) {
          const uint32_t p = e / kCh, ch = e % kCh;
          const uint32_t from = __shfl_sync(0xffffffffu, row, p);
          const uint64_t at = from == kNoSlot ? 0 : (uint64_t)from * D * sizeof(T) + ch * 16;
          if (ch >= chunks) continue;
          copy16(dst + p * A::kRow + ch * 16, static_cast<const uint8_t*>(c.k) + at, from != kNoSlot);
          if (with_v) copy16(dst + (kTile + p) * A::kRow + ch * 16, static_cast<const uint8_t*>(c.v) + at, from != kNoSlot);
        }
      };
#pragma unroll
      for (int n = 0; n < NS; n++) {
        fetch(n, row_of(n), true);
        copy_commit();
      }
      uint32_t next = row_of(NS);
      Query<T, DP> q;
      q.load(r.q + ((uint64_t)i * r.heads + h * G + g0) * D, D, gn, r.scale * 1.4426950408889634f);
      float o[DP / 16][4], m0 = -FLT_MAX, m1 = -FLT_MAX, l0 = 0.f, l1 = 0.f;
#pragma unroll
      for (auto& x : o) x[0] = x[1] = x[2] = x[3] = 0.f;
      float4* const kept_scores = reinterpret_cast<float4*>(sm + A::kFixed) + (uint64_t)warp * score_tiles * 32 + lane;
      auto masked_scores = [&](uint32_t n, uint32_t ktile, float (&x)[4]) {
        q.scores(ktile, x);
        const uint32_t j = (gw + n * C * W) * kTile + g;
        if (j >= len) x[0] = x[1] = -INFINITY;
        if (j + 8 >= len) x[2] = x[3] = -INFINITY;
      };
      for (uint32_t n = 0, slot = 0; n < mine_n; n++, slot = slot + 1 == NS ? 0 : slot + 1) {
        copy_wait<NS - 1>();
        __syncwarp();
        const uint32_t tile_a = ring_a + slot * A::kStage;
        float x[4];
        masked_scores(n, tile_a, x);
        if (WEIGHTS && n < score_tiles) kept_scores[n * 32] = make_float4(x[0], x[1], x[2], x[3]);
        const float t0 = fmaxf(x[0], x[2]), t1 = fmaxf(x[1], x[3]);
        if (__any_sync(0xffffffffu, t0 > m0 || t1 > m1)) {
          float n0 = fmaxf(t0, m0), n1 = fmaxf(t1, m1);
#pragma unroll
          for (int w = 4; w < 32; w *= 2) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, w));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, w));
          }
          const float f0 = exp2f(m0 - n0), f1 = exp2f(m1 - n1);
          m0 = n0;
          m1 = n1;
          l0 *= f0;
          l1 *= f1;
#pragma unroll
          for (auto& y : o) {
            y[0] *= f0;
            y[1] *= f1;
            y[2] *= f0;
            y[3] *= f1;
          }
        }
        const float p[4] = {exp2f(x[0] - m0), exp2f(x[1] - m1), exp2f(x[2] - m0), exp2f(x[3] - m1)};
        l0 += p[0] + p[2];
        l1 += p[1] + p[3];
        add_values<T, DP>(tile_a + kTile * A::kRow, p, o);
        __syncwarp();
        fetch(slot, next, true);
        copy_commit();
        next = row_of(n + NS + 1);
      }
      copy_wait<0>();
      __syncwarp();
      // the warps of the block
#pragma unroll
      for (int w = 4; w < 32; w *= 2) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, w);
        l1 += __shfl_xor_sync(0xffffffffu, l1, w);
      }
#pragma unroll
      for (int m = 0; m < DP / 16; m++)
#pragma unroll
        for (int e = 0; e < 4; e++) mine[(2 * t + e % 2) * DP + m * 16 + g + (e / 2) * 8] = o[m][e];
      if (g == 0) {
        mine[8 * DP + 2 * t] = m0;
        mine[8 * DP + 2 * t + 1] = m1;
        mine[8 * DP + 8 + 2 * t] = l0;
        mine[8 * DP + 8 + 2 * t + 1] = l1;
      }
      bad = __syncthreads_or(bad) || too_long;
      auto part = [&](uint32_t w) { return reinterpret_cast<const float*>(sm + w * NS * A::kStage); };
      for (uint32_t e = tid; e < 8 * DP / 4; e += W * 32) {
        const uint32_t hh = e / (DP / 4);
        float M = -FLT_MAX;
#pragma unroll
        for (int w = 0; w < W; w++) M = fmaxf(M, part(w)[8 * DP + hh]);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; w++) {
          const float f = exp2f(part(w)[8 * DP + hh] - M);
          const float4 y = reinterpret_cast<const float4*>(part(w))[e];
          sum.x = fmaf(y.x, f, sum.x);
          sum.y = fmaf(y.y, f, sum.y);
          sum.z = fmaf(y.z, f, sum.z);
          sum.w = fmaf(y.w, f, sum.w);
        }
        reinterpret_cast<float4*>(block_o)[e] = sum;
        if (e % (DP / 4) == 0) {
          float L = 0.f;
#pragma unroll
          for (int w = 0; w < W; w++) L = fmaf(part(w)[8 * DP + 8 + hh], exp2f(part(w)[8 * DP + hh] - M), L);
          block_m[hh] = M;
          block_l[hh] = L;
        }
      }
      if (tid == 0) *block_bad = bad;
      // the blocks of the cluster: each sums a share of the outputs over all blocks
      cluster_sync();
      const uint32_t o_a = smem_addr(block_o), m_a = smem_addr(block_m), l_a = smem_addr(block_l), b_a = smem_addr(block_bad);
      bad = false;
      for (uint32_t k = 0; k < C; k++) bad |= __float_as_uint(ld_cluster(cluster_addr(b_a, k))) != 0;
      const float qnan = __int_as_float(0x7fc00000);
      const uint64_t row_head = (uint64_t)i * r.heads + h * G + g0;
      for (uint32_t e = rank * W * 32 + tid; e < gn * (DP / 4); e += C * W * 32) {
        const uint32_t hh = e / (DP / 4), d = e % (DP / 4) * 4;
        float M = -FLT_MAX, L = 0.f;
        for (uint32_t k = 0; k < C; k++) M = fmaxf(M, ld_cluster(cluster_addr(m_a + hh * 4, k)));
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t k = 0; k < C; k++) {
          const float f = exp2f(ld_cluster(cluster_addr(m_a + hh * 4, k)) - M);
          const float4 y = ld_cluster4(cluster_addr(o_a + e * 16, k));
          L = fmaf(ld_cluster(cluster_addr(l_a + hh * 4, k)), f, L);
          sum.x = fmaf(y.x, f, sum.x);
          sum.y = fmaf(y.y, f, sum.y);
          sum.z = fmaf(y.z, f, sum.z);
          sum.w = fmaf(y.w, f, sum.w);
        }
        const float inv = bad ? qnan : L == 0.f ? 0.f : (__is_same(T, __half) ? 1.f / 16384.f : 1.f) / L;
        if (d < D)
          *reinterpret_cast<float4*>(r.out + (row_head + hh) * D + d) =
              make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
        if (d == 0 && r.lse) r.lse[row_head + hh] = bad ? qnan : L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
      }
      if (WEIGHTS && !bad) {
        float M[2], inv[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const uint32_t hh = 2 * t + u;
          float L = 0.f;
          M[u] = -FLT_MAX;
          for (uint32_t k = 0; k < C; k++) M[u] = fmaxf(M[u], ld_cluster(cluster_addr(m_a + hh * 4, k)));
          for (uint32_t k = 0; k < C; k++)
            L = fmaf(ld_cluster(cluster_addr(l_a + hh * 4, k)), exp2f(ld_cluster(cluster_addr(m_a + hh * 4, k)) - M[u]), L);
          inv[u] = hh >= gn || L == 0.f ? 0.f : 1.f / L;
        }
        if (mine_n > score_tiles && chunks * 16 < DP * sizeof(T)) {  // (the join has written over the zero columns)
          const uint32_t extra = DP * (uint32_t)sizeof(T) / 16 - chunks;
          __syncwarp();
          for (uint32_t e = lane; e < kTile * extra; e += 32)
            *reinterpret_cast<uint4*>(ring + (e / extra) * A::kRow + (chunks + e % extra) * 16) = make_uint4(0, 0, 0, 0);
        }
        float* const w = r.weights + ((uint64_t)s * c.kvheads + h) * cap;
        for (uint32_t n = 0; n < mine_n; n++) {
          float x[4];
          if (n < score_tiles) {
            const float4 y = kept_scores[n * 32];
            x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
          } else {
            __syncwarp();
            fetch(0, row_of(n), false);
            copy_commit();
            copy_wait<0>();
            __syncwarp();
            masked_scores(n, ring_a, x);
          }
          float w0 = exp2f(x[0] - M[0]) * inv[0] + exp2f(x[1] - M[1]) * inv[1];
          float w8 = exp2f(x[2] - M[0]) * inv[0] + exp2f(x[3] - M[1]) * inv[1];
          w0 += __shfl_xor_sync(0xffffffffu, w0, 1);
          w8 += __shfl_xor_sync(0xffffffffu, w8, 1);
          w0 += __shfl_xor_sync(0xffffffffu, w0, 2);
          w8 += __shfl_xor_sync(0xffffffffu, w8, 2);
          const uint32_t j = (gw + n * C * W) * kTile + g;
          if (t == 0 && j < len) w[j] += w0;
          if (t == 1 && j + 8 < len) w[j + 8] += w8;
        }
      }
      cluster_sync();  // the other blocks have read this one's part
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

namespace {

constexpr int kMaxCluster = 16;
constexpr uint32_t kMaxAttSmem = 220 * 1024;

template <class T, int DP, bool WEIGHTS>
cudaError_t att_prepare() {
  auto* f = k_paged_attention<T, DP, WEIGHTS>;
  cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       WEIGHTS ? (int)kMaxAttSmem : Att<T, DP>::kFixed);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

// Blocks of a cluster: enough that the launch fills the GPU (two blocks an SM) several times over, as the
// sequences' lengths differ and are not known here, as long as a warp keeps two tiles of a full cache.
template <class T, int DP, bool WEIGHTS>
cudaError_t att_launch(const PagedKV& c, const PagedRows& r, cudaStream_t st) {
  using A = Att<T, DP>;
  const uint32_t units = r.rows * c.kvheads, tiles = (uint32_t)(((uint64_t)c.max_pages * c.page + kTile - 1) / kTile);
  uint32_t C = 1;
  while (C < (uint32_t)kMaxCluster && (uint64_t)units * C < 1024 && tiles >= 4 * C * A::W) C *= 2;
  uint32_t keep = 0;
  if (WEIGHTS) {
    const uint32_t room = (kMaxAttSmem - A::kFixed) / (A::W * 512);
    while (C < (uint32_t)kMaxCluster && (tiles + C * A::W - 1) / (C * A::W) > room) C *= 2;
    keep = (tiles + C * A::W - 1) / (C * A::W);
    keep = keep < room ? keep : room;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(units * C);
  cfg.blockDim = dim3(A::W * 32);
  cfg.dynamicSmemBytes = A::kFixed + keep * A::W * 512;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_paged_attention<T, DP, WEIGHTS>, c, r, keep);
}

// Rows are computed at the next of these widths; the columns between are zeros in shared memory.
template <class T, class F>
cudaError_t by_width(uint32_t D, F&& f) {
  if (D <= 32) return f.template operator()<T, 32>();
  if (D <= 64) return f.template operator()<T, 64>();
  if (D <= 96) return f.template operator()<T, 96>();
  if (D <= 128) return f.template operator()<T, 128>();
  if (D <= 192) return f.template operator()<T, 192>();
  return f.template operator()<T, 256>();
}
struct AttLaunch {
  const PagedKV& c;
  const PagedRows& r;
  cudaStream_t st;
  template <class T, int DP>
  cudaError_t operator()() const {
    return r.weights ? att_launch<T, DP, true>(c, r, st) : att_launch<T, DP, false>(c, r, st);
  }
};
struct AttPrepare {
  template <class T, int DP>
  cudaError_t operator()() const {
    const cudaError_t e = att_prepare<T, DP, false>();
    return e == cudaSuccess ? att_prepare<T, DP, true>() : e;
  }
};

}  // namespace

// Once per device, before launch_paged_attention.
cudaError_t paged_prepare() {
  cudaError_t e = cudaSuccess;
  for (uint32_t D : {32u, 64u, 96u, 128u, 192u, 256u}) {
    if (e == cudaSuccess) e = by_width<float>(D, AttPrepare{});
    if (e == cudaSuccess) e = by_width<__half>(D, AttPrepare{});
    if (e == cudaSuccess) e = by_width<__nv_bfloat16>(D, AttPrepare{});
  }
  return e;
}

cudaError_t launch_paged_attention(const PagedKV& c, const PagedRows& r, cudaStream_t st) {
  const AttLaunch f{c, r, st};
  switch (c.kind) {
    case F32: return by_width<float>(c.D, f);
    case F16: return by_width<__half>(c.D, f);
    default: return by_width<__nv_bfloat16>(c.D, f);
  }
}

cudaError_t launch_paged_evict(const PagedKV& c, const PagedEvict& e, cudaStream_t st) {
  k_evict_select<<<c.n_seqs * c.kvheads, 1024, 0, st>>>(c, e);
  QC_BY_KIND(c.kind, (k_evict_move<T><<<dim3(c.n_seqs * c.kvheads, 2), 256, 0, st>>>(c, e)));
  return cudaGetLastError();
}

}  // namespace qc
