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

// Eight values (four of f32) to nearest, as the 16 bytes of a cache row they make.
template <class T>
__device__ __forceinline__ uint4 round16(const float* x) {
  const float4 a = *reinterpret_cast<const float4*>(x);
  uint4 r;
  if constexpr (sizeof(T) == 4) {
    r = *reinterpret_cast<const uint4*>(&a);
  } else {
    const float4 b = *reinterpret_cast<const float4*>(x + 4);
    const T v[8] = {from_float<T>(a.x), from_float<T>(a.y), from_float<T>(a.z), from_float<T>(a.w),
                    from_float<T>(b.x), from_float<T>(b.y), from_float<T>(b.z), from_float<T>(b.w)};
    memcpy(&r, v, 16);
  }
  return r;
}

// Row i's k and v (f32, rounded to nearest) to slot pos[i] of sequence seq[i]; its weights become 0.  A block
// takes a row, a thread 16 bytes of the cache at a time, of k and of v.  A step's rows are bound by latency (the
// row's place, then its values, then the write): 64 rows of 4 x 128 bf16 take 2.1 us; a prompt's by bytes:
// 4500 rows of 8 x 128 f16 take 12.1 us, 4.6 TB/s.
template <class T>
__global__ void __launch_bounds__(256) k_paged_append(PagedKV c, const float* __restrict__ k, const float* __restrict__ v,
                                                       const uint32_t* __restrict__ seq, const uint32_t* __restrict__ pos,
                                                       float* __restrict__ weights) {
  constexpr uint32_t kPer = 16 / sizeof(T);
  const uint32_t i = blockIdx.x, s = seq ? seq[i] : i, j = pos[i], pieces = c.D / kPer;
  if (s >= c.n_seqs || j >= c.max_pages * c.page) return;
  const uint32_t at = j / c.page, in = j - at * c.page, p = c.table[(uint64_t)s * c.max_pages + at];
  if (p >= c.n_pages) return;
  for (uint32_t e = threadIdx.x; e < c.kvheads * pieces; e += blockDim.x) {
    const uint32_t h = e / pieces;
    const uint64_t to = (((uint64_t)p * c.kvheads + h) * c.page + in) * pieces + e % pieces;
    const uint64_t from = ((uint64_t)i * c.kvheads * pieces + e) * kPer;
    const uint4 a = round16<T>(k + from), b = round16<T>(v + from);
    static_cast<uint4*>(c.k)[to] = a;
    static_cast<uint4*>(c.v)[to] = b;
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
// split themselves, into two tf32 planes (2^-22), and the product of the two smaller parts is left out (2^-24 to
// 2^-22 of the product; adding it changed no error).  A tile's products are added to f32 sums outside the matrix
// units, whose accumulators truncate.  Queries of one KV head share K and V; more than 8 heads take
// another turn over the sequence, 8 at a time.
//
// Neighbouring rows of one sequence (prompts) are taken R units of 8 (row, head) columns at a time, their q's
// planes in shared memory: K and V come from L2 once for up to 8 R columns, and a unit's products fill the waits
// of another's.  512 rows of 4096 positions, 32/4 heads of 128 bf16: 362 us, the matrix units busy about half
// the time (48 products a tile and unit); a row at a time 466.  These kernels use all 255 registers, and spill 8 to
// 44 bytes a thread at most widths.
//
// The warps' (maximum, sum, O) are joined in shared memory, the blocks' through the cluster's
// distributed shared memory in a fixed order: no workspace, no atomics, the same bits every time.

constexpr int kTile = 16;
constexpr int kMaxCluster = 16;

template <class T, int DP>
struct Att {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kKS = kF32 ? DP / 8 : DP / 16;              // k steps of the score product
  static constexpr int kQP = sizeof(T) == 4 ? 2 : (__is_same(T, __half) ? 2 : 3);  // planes of q and of p
  static constexpr int kRow = DP * (int)sizeof(T) + 16;            // bytes of a tile row: odd multiples of 16 bytes
  static constexpr int kStage = 2 * kTile * kRow;                  //   apart, so 8 rows never share a bank
  static constexpr int kRoom = 70 * 1024;                          // three blocks on an SM
  static constexpr int W = 8 * kStage <= kRoom ? 4 : 2;
  static constexpr int kFit = kRoom / (W * kStage);
  static constexpr int NS = kFit > 4 ? 4 : kFit < 2 ? 2 : kFit;
  static constexpr int kWide = 200 * 1024 / (NS * kStage) > 8 ? 8 : 200 * 1024 / (NS * kStage);  // one block an SM
  static constexpr int kO = DP + 4;                                // floats between two heads' O in a warp's part
  static constexpr int kShared = DP <= 128 ? 4 : 2;                // units of a block that shares tiles among rows
  static constexpr int kPlanes = kKS * 32 * kQP * 2;               // words of a unit's q
  // this block's share of every block's O; of several units, their q before
  static constexpr int space(int units) {
    const int o = units * (2 * DP + kMaxCluster) * 16, q = units > 1 ? units * kPlanes * 4 : 0;
    return o > q ? o : q;
  }
  // ring of w warps; space; every block's maxima and sums; the warps' maxima; columns' lengths, factors; bad slots
  static constexpr int fixed(int w, int units) {
    return w * NS * kStage + space(units) + units * kMaxCluster * 16 * 4 + w * units * 8 * 4 + (units > 1 ? units * 64 + w * 4 : 0);
  }
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
// x = hi + lo up to 2^-22 |x|, both with the 11 significant bits of tf32 (hi to nearest, ties away from zero; lo
// cut).  What rounds beyond the largest such number is that number, so that finite values have finite parts; of an
// infinity or a NaN lo keeps it.  In integers: 64 sequences of 130..4096 positions 137 us; with
// cvt.rna.tf32 143, and 151 with the bound.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  float h = __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
  asm("min.xorsign.abs.f32 %0, %0, %1;" : "+f"(h) : "f"(__uint_as_float(0x7f7fe000u)));
  hi = __float_as_uint(h);
  lo = __float_as_uint(x - h) & 0xffffe000u;
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

__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();  // (the barrier wants a warp's threads together)
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
// This block's shared address `a` in block `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster(uint32_t a, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster4(uint32_t a, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(a), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
__device__ __forceinline__ uint2 ld_cluster2(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
// 2^x to 2 ulp (results below 2^-126 are 0)
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Scores (times log2 e, and q's scaling) of a K tile and of n <= R units of 8 columns (queries): s[u][0], s[u][1]
// for position lane / 4 and columns 2 (lane % 4), + 1; s[u][2], s[u][3] for position lane / 4 + 8.  frag(u, k, b):
// the planes of q^T of unit u, step k.  All: n = R; without a test at every unit the compiler interleaves their
// products (512 rows of 4096 positions, 32/4 heads of 128 bf16: 361 us against 489).
//
// The matrix units cut their sums at every step, D / 8 of them in f32: there hi x hi goes to H sums in turn and the
// smaller products to L others.  Four and one where rows are computed by themselves: errors of 3e-7 to 6e-7 of the
// outputs, about the plain form's or below it, where one and two give 5e-7 to 1.4e-6 in the same time.  Two and one
// for R units, whose registers hold no more (64 rows of 2048 positions 83 us, with three and one 93), two and two
// for the weights (with one 188 us for those rows, against 181).
template <class T, int DP, int R, bool All, int H, int L, class F>
__device__ __forceinline__ void scores_of(uint32_t ktile, uint32_t n, F&& frag, float (&s)[R][4]) {
  using A = Att<T, DP>;
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t a0 = ktile + ((lane / 8 % 2) * 8 + lane % 8) * A::kRow + (lane / 16) * 16;
  float c[R][A::kF32 ? H + L : A::kQP][4];
#pragma unroll
  for (auto& u : c)
#pragma unroll
    for (auto& x : u) x[0] = x[1] = x[2] = x[3] = 0.f;
#pragma unroll
  for (int k = 0; k < A::kKS; k++) {
    uint32_t a[4], b[A::kQP][2];
    ldsm4(a, a0 + k * 32);
    if constexpr (A::kF32) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; i++) split_tf32(__uint_as_float(a[i]), hi[i], lo[i]);
#pragma unroll
      for (int u = 0; u < R; u++) {
        if (!All && u >= n) break;
        frag(u, k, b);
        mma8(c[u][k % H], hi, b[0][0], b[0][1]);
        mma8(c[u][H], hi, b[1][0], b[1][1]);
        mma8(c[u][H + L - 1], lo, b[0][0], b[0][1]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < R; u++) {
        if (!All && u >= n) break;
        frag(u, k, b);
#pragma unroll
        for (int p = 0; p < A::kQP; p++) mma16<T>(c[u][p], a, b[p][0], b[p][1]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < R; u++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float first = c[u][0][i];
      if constexpr (A::kF32) {
#pragma unroll
        for (int p = 1; p < H; p++) first += c[u][p][i];
        s[u][i] = first + (L == 2 ? c[u][H][i] + c[u][H + L - 1][i] : c[u][H][i]);
      } else {
        // An infinite sum of the first planes is the score: the other planes' may be infinite the other way (keys
        // of the type's lowest value, queries rounded up) or NaN (infinite keys, queries without a second plane).
        float rest = c[u][1][i];
        if constexpr (A::kQP == 3) rest += c[u][2][i];
        s[u][i] = fabsf(first) == INFINITY ? first : first + rest;
      }
    }
}

// One warp's query operand: the B fragments of q^T for 8 heads, and the factor that undoes q's scaling
// for the two heads whose scores this lane holds.
template <class T, int DP>
struct Query {
  using A = Att<T, DP>;
  static constexpr bool kScaled = A::kF32 || __is_same(T, __half);
  float raw[A::kKS][A::kF32 ? 2 : 4];
  uint32_t f[A::kKS][A::kQP][2];
  float undo0, undo1, undo;  // (undo: of column lane / 4)

  // Starts reading q, column lane / 4 at qr; columns that are not real and values >= D are zero.
  __device__ __forceinline__ void fetch(const float* qr, uint32_t D, bool real) {
    const uint32_t t = threadIdx.x & 3;
#pragma unroll
    for (int k = 0; k < A::kKS; k++)
#pragma unroll
      for (int b = 0; b < 2; b++) {
        if constexpr (A::kF32) {
          const uint32_t d = k * 8 + b * 4 + t;
          raw[k][b] = real && d < D ? qr[d] : 0.f;
        } else {
          const uint32_t d = k * 16 + b * 8 + 2 * t;
          float2 x = make_float2(0.f, 0.f);
          if (real && d < D) x = *reinterpret_cast<const float2*>(qr + d);
          raw[k][2 * b] = x.x;
          raw[k][2 * b + 1] = x.y;
        }
      }
  }
  // Splits q times factor (scale log2 e) into planes.
  __device__ __forceinline__ void split(float factor) {
    const uint32_t t = threadIdx.x & 3;
    undo0 = undo1 = undo = 1.f;
    float up = 1.f;
    if constexpr (kScaled) {
      // the largest |q| of a head: f16, to 2^13..2^14, so that two planes hold 22 bits; f32, to 2^-10..2^-9, so that
      // no sum of the parts' products overflows before the score does
      constexpr int kTo = A::kF32 ? -10 : 13;
      float mx = 0.f;
#pragma unroll
      for (int k = 0; k < A::kKS; k++)
#pragma unroll
        for (int b = 0; b < (A::kF32 ? 2 : 4); b++) mx = fmaxf(mx, fabsf(raw[k][b] * factor));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      int e = kTo - ((int)(__float_as_uint(mx) >> 23) - 127);
      e = mx == 0.f || mx > FLT_MAX ? 0 : e > 120 ? 120 : e < -126 ? -126 : e;
      up = __uint_as_float((uint32_t)(127 + e) << 23);
      undo = __uint_as_float((uint32_t)(127 - e) << 23);
      undo0 = __shfl_sync(0xffffffffu, undo, 8 * t);
      undo1 = __shfl_sync(0xffffffffu, undo, 8 * t + 4);
    }
    if constexpr (A::kF32) {
#pragma unroll
      for (int k = 0; k < A::kKS; k++) {
        split_tf32(raw[k][0] * factor * up, f[k][0][0], f[k][1][0]);
        split_tf32(raw[k][1] * factor * up, f[k][0][1], f[k][1][1]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < A::kKS; k++) {
        const float x[4] = {raw[k][0] * factor * up, raw[k][1] * factor * up, raw[k][2] * factor * up,
                            raw[k][3] * factor * up};
        uint32_t lo[A::kQP], hi[A::kQP];
        split_pair<T, A::kQP>(x[0], x[1], lo);
        split_pair<T, A::kQP>(x[2], x[3], hi);
#pragma unroll
        for (int p = 0; p < A::kQP; p++) {
          f[k][p][0] = lo[p];
          f[k][p][1] = hi[p];
        }
      }
    }
  }

  template <int H, int L>
  __device__ __forceinline__ void scores(uint32_t ktile, float (&s)[4]) const {
    float x[1][4];
    scores_of<T, DP, 1, true, H, L>(ktile, 1, [&](int, int k, uint32_t (&b)[A::kQP][2]) {
#pragma unroll
      for (int p = 0; p < A::kQP; p++) {
        b[p][0] = f[k][p][0];
        b[p][1] = f[k][p][1];
      }
    }, x);
#pragma unroll
    for (int i = 0; i < 4; i++) s[i] = x[0][i] * (i % 2 ? undo1 : undo0);
  }
};

// O^T += V^T P^T for one tile and n <= R units; p as scores_of lays its scores out.
template <class T, int DP, int R, bool All>
__device__ __forceinline__ void add_values(uint32_t vtile, uint32_t n, const float (&p)[R][4], float (&o)[R][DP / 16][4]) {
  using A = Att<T, DP>;
  const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane % 4;
  if constexpr (A::kF32) {
    // k index i of a step of 8 positions stands for position 2 i (i < 4) or 2 (i - 4) + 1: the reads of V
    // then fall on 32 different banks
    uint32_t hi[R][2][2], lo[R][2][2];
#pragma unroll
    for (int u = 0; u < R; u++)
#pragma unroll
      for (int st = 0; st < 2; st++)
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const uint32_t from = (2 * t + b) * 4 + g / 2;
          const float x = __shfl_sync(0xffffffffu, p[u][2 * st], from), y = __shfl_sync(0xffffffffu, p[u][2 * st + 1], from);
          split_tf32(g % 2 ? y : x, hi[u][st][b], lo[u][st][b]);
        }
#pragma unroll
    for (int m = 0; m < DP / 16; m++) {
      uint32_t ah[2][4], al[2][4];
#pragma unroll
      for (int st = 0; st < 2; st++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float x;
          const uint32_t a = vtile + (st * 8 + 2 * t + i / 2) * A::kRow + (m * 16 + g + (i % 2) * 8) * 4;
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(a) : "memory");
          split_tf32(x, ah[st][i], al[st][i]);
        }
#pragma unroll
      for (int u = 0; u < R; u++) {
        if (!All && u >= n) break;
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < 2; st++) {
          mma8(c, al[st], hi[u][st][0], hi[u][st][1]);
          mma8(c, ah[st], lo[u][st][0], lo[u][st][1]);
          mma8(c, ah[st], hi[u][st][0], hi[u][st][1]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) o[u][m][i] += c[i];
      }
    }
  } else {
    uint32_t lo8[R][A::kQP], hi8[R][A::kQP];
    const float up = __is_same(T, __half) ? 16384.f : 1.f;  // (undone with the final division)
#pragma unroll
    for (int u = 0; u < R; u++) {
      split_pair<T, A::kQP>(p[u][0] * up, p[u][1] * up, lo8[u]);
      split_pair<T, A::kQP>(p[u][2] * up, p[u][3] * up, hi8[u]);
#pragma unroll
      for (int q = 0; q < A::kQP; q++) {
        lo8[u][q] = transpose8(lo8[u][q]);
        hi8[u][q] = transpose8(hi8[u][q]);
      }
    }
    const uint32_t a0 = vtile + ((lane / 16) * 8 + lane % 8) * A::kRow + (lane / 8 % 2) * 16;
#pragma unroll
    for (int m = 0; m < DP / 16; m++) {
      uint32_t a[4];
      ldsm4_t(a, a0 + m * 32);
#pragma unroll
      for (int u = 0; u < R; u++) {
        if (!All && u >= n) break;
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = A::kQP - 1; q >= 0; q--) mma16<T>(c, a, lo8[u][q], hi8[u][q]);
#pragma unroll
        for (int i = 0; i < 4; i++) o[u][m][i] += c[i];
      }
    }
  }
}

// How a launch splits a sequence: the blocks of a cluster; a warp's next tile lies step_pages pages and
// step_slots slots further; the rows of a group; whether the longest come first.
struct AttSplit {
  uint32_t blocks, step_pages, step_slots, rows;
  bool longest_first;
};
constexpr uint32_t kMaxSorted = 128;  // rows
static_assert(kMaxSorted < kMaxCluster * 16, "lengths are sorted where the maxima and sums come later");

template <class T, int DP, int W, int R>
__global__ void __launch_bounds__(W * 32, R > 1 ? 2 : Att<T, DP>::fixed(W, R) <= 75 * 1024 ? 3 : 1)
    k_paged_attention(PagedKV c, PagedRows r, AttSplit sp) {
  using A = Att<T, DP>;
  constexpr int NS = A::NS;
  constexpr int kPart = 8 * A::kO + 8;  // floats of a unit's O and sums
  static_assert(R * kPart * 4 <= NS * A::kStage, "a warp's part lies in its ring");
  extern __shared__ __align__(16) uint8_t sm[];
  uint8_t* const space = sm + W * NS * A::kStage;
  float* const in_o = reinterpret_cast<float*>(space);                  // [R][C][8 DP / C]: this block's share of every block's O
  uint32_t* const planes = reinterpret_cast<uint32_t*>(space);          // R > 1, before: [R][kPlanes], the units' q
  float* const in_m = reinterpret_cast<float*>(space + A::space(R));    // [R][C][16]: every block's maxima, sums
  float* const warp_m = in_m + R * kMaxCluster * 16;                    // [W][R][8]
  uint32_t* const col_len = reinterpret_cast<uint32_t*>(warp_m + W * R * 8);  // R > 1: [R][8]; kNoSlot: beyond the cache
  float* const col_undo = reinterpret_cast<float*>(col_len + R * 8);          // R > 1: [R][8]
  uint32_t* const warp_bad = col_len + R * 16;                                // R > 1: [W] first slot of an invalid page
  const uint32_t C = sp.blocks, h = blockIdx.y;
  uint32_t rank, first;  // (the row, or the rows' place among the clusters)
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(first));
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane / 4, t = lane % 4;
  const uint32_t D = c.D, G = r.heads / c.kvheads, cap = c.max_pages * c.page, chunks = D * (uint32_t)sizeof(T) / 16;
  uint8_t* const ring = sm + warp * NS * A::kStage;
  const uint32_t ring_a = smem_addr(ring);
  if (R == 1 && sp.longest_first) {  // the row of rank `first` among the lengths
    uint32_t* const lens = reinterpret_cast<uint32_t*>(in_m);
    for (uint32_t k = tid; k < r.rows; k += W * 32) lens[k] = r.len[k];
    __syncthreads();
    for (uint32_t k = tid; k < r.rows; k += W * 32) {
      const uint32_t n = lens[k];
      uint32_t before = 0;
#pragma unroll 8
      for (uint32_t j = 0; j < r.rows; j++) before += lens[j] > n || (lens[j] == n && j < k);
      if (before == first) lens[kMaxSorted] = k;
    }
    __syncthreads();
    first = lens[kMaxSorted];
    __syncthreads();  // (in_m is the cluster's from here on)
  }
  // Rows of a group (sp.rows of them) are computed together where all are of one sequence (R > 1), each by itself
  // where they are not (R = 1); the other kernel's blocks leave.
  const uint32_t i = R > 1 ? first * sp.rows : first, group = R > 1 ? i : i - i % sp.rows;
  const uint32_t nr = R > 1 ? min(sp.rows, r.rows - i) : 1, s = r.seq ? r.seq[i] : i;
  if (s >= c.n_seqs) return;  // (the whole cluster)
  if (sp.rows > 1) {
    const bool other = lane < sp.rows && group + lane < r.rows && (r.seq ? r.seq[group + lane] : group + lane) != s;
    if (__any_sync(0xffffffffu, other) == (R > 1)) return;
  }
  // Where pages hold whole runs of 8 positions a lane copies its part of a run with one address; else every
  // position has its own page and its lanes ask the lane that looked it up.  64 sequences of 4096
  // positions in bf16: 105 us with pages of 16 slots (runs), 108 with pages of 250.
  const bool runs = c.page % 8 == 0;
  const uint32_t step = C * W * kTile, gw = rank * W + warp;
  const uint32_t ahead = runs ? lane / 16 * 8 : lane % kTile;  // the position of a tile this lane looks up
  const uint32_t page0 = (gw * kTile + ahead) / c.page, slot0 = (gw * kTile + ahead) % c.page;
  const uint32_t* const pages = c.table + (uint64_t)s * c.max_pages;
  const uint32_t columns = nr * G;  // column x: row i + x / G, head x % G of the KV head's
  for (uint32_t x0 = 0; x0 < columns; x0 += 8 * R) {
    const uint32_t units = R > 1 ? min((uint32_t)R, (columns - x0 + 7) / 8) : 1;
    auto column = [&](uint32_t x) {  // row of q, out and lse
      return R > 1 ? (uint64_t)(i + x / G) * r.heads + h * G + x % G : (uint64_t)i * r.heads + h * G + x;
    };
    Query<T, DP> q;
    bool bad = false;
    uint32_t first_bad = kNoSlot, len, shortest = 0;
    if constexpr (R == 1) {
      cluster_arrive();  // this block runs, and in_o and in_m may be written
      len = r.len[i];
      q.fetch(r.q + column(x0 + g) * D, D, x0 + g < columns);
      bad = len > cap;
      if (bad) len = 0;
    } else {
      __syncthreads();  // (the last turn's results are read)
      if (tid < R * 8) {
        const uint32_t n = x0 + tid < columns ? r.len[i + (x0 + tid) / G] : 0;
        col_len[tid] = n > cap ? kNoSlot : n;
      }
      __syncthreads();
      uint32_t n = lane < R * 8 ? col_len[lane] : 0;
      if (n == kNoSlot) n = 0;
      len = __reduce_max_sync(0xffffffffu, n);
      shortest = __reduce_min_sync(0xffffffffu, n ? n : kNoSlot);
    }
    const uint32_t tiles = (len + kTile - 1) / kTile;
    const uint32_t mine_n = tiles > gw ? (tiles - gw + C * W - 1) / (C * W) : 0;  // this warp's tiles
    auto clear_columns = [&](uint32_t rows) {  // columns D.. of the tiles are zero (the join writes over them)
      const uint32_t extra = DP * (uint32_t)sizeof(T) / 16 - chunks;
      for (uint32_t e = lane; e < rows * extra; e += 32)
        *reinterpret_cast<uint4*>(ring + (e / extra) * A::kRow + (chunks + e % extra) * 16) = make_uint4(0, 0, 0, 0);
    };
    // The page number of position j, table entry `at`, and its row at slot `in` for the tile from j0 on.
    auto page_at = [&](uint32_t j, uint32_t at) { return j < len ? pages[at] : kNoSlot; };
    auto row_of = [&](uint32_t p, uint32_t in, uint32_t j0) {
      if (p >= c.n_pages) {
        if (R == 1)
          bad |= j0 + ahead < len;
        else if (j0 + ahead < len)
          first_bad = min(first_bad, j0 + ahead);
        return kNoSlot;
      }
      return (p * c.kvheads + h) * c.page + in;
    };
    // Copies the tile of positions j0.. into a ring slot; row: this lane's lookup.
    auto fetch = [&](uint32_t slot, uint32_t row, uint32_t j0) {
      constexpr uint32_t kCh = DP * sizeof(T) / 16;
      const uint32_t dst = ring_a + slot * A::kStage;
      const uint8_t *kp = static_cast<const uint8_t*>(c.k), *vp = static_cast<const uint8_t*>(c.v);
      if (runs) {
        const uint32_t row0 = __shfl_sync(0xffffffffu, row, 0), row1 = __shfl_sync(0xffffffffu, row, 16);
        const uint64_t bytes = D * sizeof(T);
        const uint64_t at0 = row0 == kNoSlot ? 0 : row0 * bytes, at1 = (row1 == kNoSlot ? 0 : row1 * bytes) - 8 * bytes;
        const uint32_t n = j0 < len ? len - j0 : 0, n0 = row0 == kNoSlot ? 0 : n, n1 = row1 == kNoSlot ? 0 : n;
#pragma unroll
        for (uint32_t e0 = 0; e0 < kTile * kCh; e0 += 32) {
          const uint32_t e = e0 + lane, p = e / kCh, ch = e % kCh;
          const bool second = e0 >= 8 * kCh;
          const uint64_t o = (second ? at1 : at0) + (p * chunks + ch) * 16;
          const bool real = p < (second ? n1 : n0);
          if (DP * sizeof(T) != chunks * 16 && ch >= chunks) continue;
          copy16(dst + p * A::kRow + ch * 16, kp + o, real);
          copy16(dst + (kTile + p) * A::kRow + ch * 16, vp + o, real);
        }
      } else {
#pragma unroll 4
        for (uint32_t e = lane; e < kTile * kCh; e += 32) {
          const uint32_t p = e / kCh, ch = e % kCh;
          const uint32_t from = __shfl_sync(0xffffffffu, row, p);
          const uint64_t o = from == kNoSlot ? 0 : (uint64_t)from * D * sizeof(T) + ch * 16;
          if (ch >= chunks) continue;
          copy16(dst + p * A::kRow + ch * 16, kp + o, from != kNoSlot);
          copy16(dst + (kTile + p) * A::kRow + ch * 16, vp + o, from != kNoSlot);
        }
      }
    };
    // this warp's tiles one after the other
    uint32_t j = gw * kTile + ahead, at = page0, in = slot0;
    auto advance = [&] {
      j += step;
      at += sp.step_pages;
      in += sp.step_slots;
      if (in >= c.page) {
        in -= c.page;
        at++;
      }
    };
    uint32_t pg[NS], slots[NS];
#pragma unroll
    for (int n = 0; n < NS; n++) {
      pg[n] = page_at(j, at);
      slots[n] = in;
      advance();
    }
    uint32_t next = page_at(j, at), next_in = in, j0 = gw * kTile;
    if (chunks * 16 < DP * sizeof(T)) clear_columns(2 * NS * kTile);
#pragma unroll
    for (int n = 0; n < NS; n++) {
      fetch(n, row_of(pg[n], slots[n], j0), j0);
      copy_commit();
      j0 += step;
    }
    uint32_t len0[R], len1[R];
    float undo0[R], undo1[R];
    if constexpr (R == 1) {
      q.split(r.scale * 1.4426950408889634f);
      len0[0] = len1[0] = len;
    } else {
      for (uint32_t u = warp; u < units; u += W) {
        const uint32_t x = x0 + u * 8 + g;
        q.fetch(r.q + column(x < columns ? x : 0) * D, D, x < columns);
        q.split(r.scale * 1.4426950408889634f);
#pragma unroll
        for (int k = 0; k < A::kKS; k++)
#pragma unroll
          for (int p = 0; p < A::kQP; p++)
            *reinterpret_cast<uint2*>(planes + ((u * A::kKS + k) * 32 + lane) * A::kQP * 2 + p * 2) =
                make_uint2(q.f[k][p][0], q.f[k][p][1]);
        if (t == 0) col_undo[u * 8 + g] = q.undo;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < R; u++) {
        len0[u] = col_len[u * 8 + 2 * t];
        len1[u] = col_len[u * 8 + 2 * t + 1];
        undo0[u] = Query<T, DP>::kScaled && u < units ? col_undo[u * 8 + 2 * t] : 1.f;
        undo1[u] = Query<T, DP>::kScaled && u < units ? col_undo[u * 8 + 2 * t + 1] : 1.f;
      }
    }
    float o[R][DP / 16][4], m0[R], m1[R], l0[R], l1[R];
#pragma unroll
    for (int u = 0; u < R; u++) {
      m0[u] = m1[u] = -FLT_MAX;
      l0[u] = l1[u] = 0.f;
#pragma unroll
      for (auto& x : o[u]) x[0] = x[1] = x[2] = x[3] = 0.f;
    }
    for (uint32_t n = 0, slot = 0; n < mine_n; n++, slot = slot + 1 == NS ? 0 : slot + 1) {
      copy_wait<NS - 1>();
      __syncwarp();
      const uint32_t tile_a = ring_a + slot * A::kStage, base = gw * kTile + n * step, pos = base + g;
      float x[R][4];
      if constexpr (R == 1) {
        q.template scores<4, 1>(tile_a, x[0]);
      } else {
        auto frag = [&](int u, int k, uint32_t (&b)[A::kQP][2]) {
#pragma unroll
          for (int p = 0; p < A::kQP; p++) {
            const uint2 w = *reinterpret_cast<const uint2*>(planes + ((u * A::kKS + k) * 32 + lane) * A::kQP * 2 + p * 2);
            b[p][0] = w.x;
            b[p][1] = w.y;
          }
        };
        if (units == R)
          scores_of<T, DP, R, true, 2, 1>(tile_a, R, frag, x);
        else
          scores_of<T, DP, R, false, 2, 1>(tile_a, units, frag, x);
#pragma unroll
        for (int u = 0; u < R; u++)
#pragma unroll
          for (int e = 0; e < 4; e++) x[u][e] *= e % 2 ? undo1[u] : undo0[u];
      }
      if (R == 1 || base + kTile > shortest) {
#pragma unroll
        for (int u = 0; u < R; u++) {
          if (pos >= len0[u]) x[u][0] = -INFINITY;
          if (pos >= len1[u]) x[u][1] = -INFINITY;
          if (pos + 8 >= len0[u]) x[u][2] = -INFINITY;
          if (pos + 8 >= len1[u]) x[u][3] = -INFINITY;
        }
        if constexpr (R > 1) {
          // Slots that one row attends to and another does not may hold anything for the latter: a row of V that
          // is not finite becomes zeros, and the columns that attend to it NaN.
          constexpr uint32_t kCh = DP * sizeof(T) / 16;
          uint8_t* const v = ring + slot * A::kStage + kTile * A::kRow;
          uint32_t wild = 0;
          for (uint32_t e = lane; e < kTile * kCh; e += 32) {
            const uint4 y = *reinterpret_cast<const uint4*>(v + (e / kCh) * A::kRow + e % kCh * 16);
            bool any = false;
            const uint32_t ws[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (const uint32_t w : ws) {
              constexpr uint32_t kExp = A::kF32 || !__is_same(T, __half) ? 0x7f800000u : 0x7c000000u;
              any |= (w & kExp) == kExp || (!A::kF32 && (w & kExp >> 16) == kExp >> 16);
            }
            wild |= any ? 1u << e / kCh : 0u;
          }
          wild = __reduce_or_sync(0xffffffffu, wild);
          if (wild) {
            for (uint32_t e = lane; e < kTile * kCh; e += 32)
              if (wild >> e / kCh & 1)
                *reinterpret_cast<uint4*>(v + (e / kCh) * A::kRow + e % kCh * 16) = make_uint4(0, 0, 0, 0);
            __syncwarp();
            const uint32_t same_t = 0x11111111u << t;
#pragma unroll
            for (int u = 0; u < R; u++) {
              const uint32_t b0 = __ballot_sync(0xffffffffu, (wild >> g & 1 && pos < len0[u]) || (wild >> (g + 8) & 1 && pos + 8 < len0[u]));
              const uint32_t b1 = __ballot_sync(0xffffffffu, (wild >> g & 1 && pos < len1[u]) || (wild >> (g + 8) & 1 && pos + 8 < len1[u]));
#pragma unroll
              for (auto& y : o[u]) {
                if (b0 & same_t) y[0] = y[2] = __int_as_float(0x7fc00000);
                if (b1 & same_t) y[1] = y[3] = __int_as_float(0x7fc00000);
              }
            }
          }
        }
      }
      float t0[R], t1[R];
      bool grows = false;
#pragma unroll
      for (int u = 0; u < R; u++) {
        t0[u] = fmaxf(x[u][0], x[u][2]);
        t1[u] = fmaxf(x[u][1], x[u][3]);
        grows |= t0[u] > m0[u] || t1[u] > m1[u];
      }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int u = 0; u < R; u++) {
          float n0 = fmaxf(t0[u], m0[u]), n1 = fmaxf(t1[u], m1[u]);
#pragma unroll
          for (int w = 4; w < 32; w *= 2) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, w));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, w));
          }
          const float f0 = pow2(m0[u] - n0), f1 = pow2(m1[u] - n1);
          m0[u] = n0;
          m1[u] = n1;
          l0[u] *= f0;
          l1[u] *= f1;
#pragma unroll
          for (auto& y : o[u]) {
            y[0] *= f0;
            y[1] *= f1;
            y[2] *= f0;
            y[3] *= f1;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < R; u++) {
        x[u][0] = pow2(x[u][0] - m0[u]);
        x[u][1] = pow2(x[u][1] - m1[u]);
        x[u][2] = pow2(x[u][2] - m0[u]);
        x[u][3] = pow2(x[u][3] - m1[u]);
        l0[u] += x[u][0] + x[u][2];
        l1[u] += x[u][1] + x[u][3];
      }
      if (R == 1 || units == R)
        add_values<T, DP, R, true>(tile_a + kTile * A::kRow, R, x, o);
      else
        add_values<T, DP, R, false>(tile_a + kTile * A::kRow, units, x, o);
      __syncwarp();
      fetch(slot, row_of(next, next_in, j0), j0);
      copy_commit();
      j0 += step;
      advance();
      next = page_at(j, at);
      next_in = in;
    }
    copy_wait<0>();
    // the warps of the block: O and sums relative to the block's maxima, then added up
#pragma unroll
    for (int u = 0; u < R; u++) {
#pragma unroll
      for (int w = 4; w < 32; w *= 2) {
        l0[u] += __shfl_xor_sync(0xffffffffu, l0[u], w);
        l1[u] += __shfl_xor_sync(0xffffffffu, l1[u], w);
      }
      if (g == 0) {
        warp_m[(warp * R + u) * 8 + 2 * t] = m0[u];
        warp_m[(warp * R + u) * 8 + 2 * t + 1] = m1[u];
      }
    }
    if constexpr (R == 1) {
      bad = __syncthreads_or(bad);
    } else {
      first_bad = __reduce_min_sync(0xffffffffu, first_bad);
      if (lane == 0) warp_bad[warp] = first_bad;
      __syncthreads();
      cluster_arrive();  // (q's planes are read, so in_o may be written)
    }
    float* const mine = reinterpret_cast<float*>(ring);  // [R][kPart]
#pragma unroll
    for (int u = 0; u < R; u++) {
      float M0 = m0[u], M1 = m1[u];
#pragma unroll
      for (int w = 0; w < W; w++) {
        M0 = fmaxf(M0, warp_m[(w * R + u) * 8 + 2 * t]);
        M1 = fmaxf(M1, warp_m[(w * R + u) * 8 + 2 * t + 1]);
      }
      const float f0 = pow2(m0[u] - M0), f1 = pow2(m1[u] - M1);
      float* const part = mine + u * kPart;
#pragma unroll
      for (int m = 0; m < DP / 16; m++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          part[(2 * t + e % 2) * A::kO + m * 16 + g + (e / 2) * 8] = o[u][m][e] * (e % 2 ? f1 : f0);
      if (g == 0) {
        part[8 * A::kO + 2 * t] = l0[u] * f0;
        part[8 * A::kO + 2 * t + 1] = l1[u] * f1;
      }
    }
    __syncthreads();
    cluster_wait();  // the other blocks run, and have read what was sent for the previous turn
    // what they add up to goes to the blocks of the cluster: a share of O to each, maxima and sums to all
    auto part = [&](uint32_t w, uint32_t u) { return reinterpret_cast<const float*>(sm + w * NS * A::kStage) + u * kPart; };
    const uint32_t share = (2 * DP + C - 1) / C;  // 16-byte pieces of O of one block (the last may have fewer)
    for (uint32_t ue = tid; ue < units * 2 * DP; ue += W * 32) {
      const uint32_t u = ue / (2 * DP), e = ue % (2 * DP), hh = e / (DP / 4), d = e % (DP / 4) * 4;
      float4 sum = *reinterpret_cast<const float4*>(part(0, u) + hh * A::kO + d);
#pragma unroll
      for (int w = 1; w < W; w++) {
        const float4 y = *reinterpret_cast<const float4*>(part(w, u) + hh * A::kO + d);
        sum.x += y.x;
        sum.y += y.y;
        sum.z += y.z;
        sum.w += y.w;
      }
      const uint32_t to = e / share;
      st_cluster4(cluster_addr(smem_addr(in_o) + ((u * C + rank) * share + e - to * share) * 16, to), sum);
    }
    for (uint32_t e = tid; e < units * C * 8; e += W * 32) {
      const uint32_t hh = e % 8, to = e / 8 % C, u = e / 8 / C;
      float M = warp_m[u * 8 + hh], L = part(0, u)[8 * A::kO + hh];
#pragma unroll
      for (int w = 1; w < W; w++) {
        M = fmaxf(M, warp_m[(w * R + u) * 8 + hh]);
        L += part(w, u)[8 * A::kO + hh];
      }
      if constexpr (R > 1) {
        const uint32_t n = col_len[u * 8 + hh];
        bad = n == kNoSlot;
#pragma unroll
        for (int w = 0; w < W; w++) bad |= warp_bad[w] < n;
      }
      const uint32_t a = cluster_addr(smem_addr(in_m) + (u * kMaxCluster + rank) * 16 * 4, to);
      st_cluster(a + hh * 4, M);
      st_cluster(a + 32 + hh * 4, bad ? __int_as_float(0x7fc00000) : L);
    }
    cluster_sync();
    for (uint32_t ue = tid; ue < units * share; ue += W * 32) {
      const uint32_t u = ue / share, e = ue % share;
      const uint32_t hh = (rank * share + e) / (DP / 4), d = (rank * share + e) % (DP / 4) * 4, x = x0 + u * 8 + hh;
      if (hh >= 8 || x >= columns || d >= D) continue;  // (pieces behind the last belong to column 8)
      const float* const ms = in_m + u * kMaxCluster * 16 + hh;
      // the maximum and the sum of the column over the blocks (bad: NaN)
      float M = -FLT_MAX, L = 0.f;
#pragma unroll 4
      for (uint32_t k = 0; k < C; k++) M = fmaxf(M, ms[k * 16]);
#pragma unroll 4
      for (uint32_t k = 0; k < C; k++) L = fmaf(ms[k * 16 + 8], pow2(ms[k * 16] - M), L);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (uint32_t k = 0; k < C; k++) {
        const float f = pow2(ms[k * 16] - M);
        const float4 y = reinterpret_cast<const float4*>(in_o)[(u * C + k) * share + e];
        sum.x = fmaf(y.x, f, sum.x);
        sum.y = fmaf(y.y, f, sum.y);
        sum.z = fmaf(y.z, f, sum.z);
        sum.w = fmaf(y.w, f, sum.w);
      }
      if (R > 1 && col_len[u * 8 + hh] == 0) {  // (what it holds of the others' tiles means nothing)
        sum = make_float4(0.f, 0.f, 0.f, 0.f);
        L = 0.f;
      }
      const float inv = L == 0.f ? 0.f : (__is_same(T, __half) ? 1.f / 16384.f : 1.f) / L;
      *reinterpret_cast<float4*>(r.out + column(x) * D + d) = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
      if (d == 0 && r.lse) r.lse[column(x)] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
    }
  }
}

// ---- accumulated weights -------------------------------------------------------------------------
// The rows' softmax weights exp(s - lse) (lse is an f32 number, so that they are off by about 2^-22 |lse| of
// themselves), summed over a KV head's heads and a sequence's rows, added to the
// slots: a second pass over K with the lse that the attention has left, so that every slot is added to
// once, whatever rows share a sequence, and the attention need not hold its scores.  A warp takes kTiles
// tiles of 16 positions of a (sequence, KV head) at a time and goes through the sequence's rows in call
// order, scores again, and sums in registers; warps do not wait for one another.  Each block finds the
// sequences that rows name and their longest rows in one pass over seq and len; their spans go to the warps
// in turn.  Where there are fewer spans than warps these are shorter, and a row's q is read while the one
// before is computed: 24 rows of 7001 positions, 4 KV heads, 44 -> 36 us for this pass; 128 rows of 1024, 16
// query heads a KV head, 356 -> 155; 32 rows of 200..2500, 32/4 heads of 128 f16, whose spans stay whole, 43.3 ->
// 44.2 with their attention.  (Keeping the attention's scores in shared memory instead left one block an SM for
// long sequences: 8 of 29,292..35,385 positions, 6 heads of 64 bf16, 113 us against 58 this way; 32 of 200..2500
// 39 against 41.)  Width 256 spills 104 (f16) to 640 bytes (f32) a thread, f32 220 at 192.
template <class T, int DP>
struct Give {
  using A = Att<T, DP>;
  static constexpr int W = 4;
  static constexpr int kTileBytes = kTile * A::kRow;
  static constexpr int kFit = 17600 / kTileBytes;  // (three or four blocks an SM)
  static constexpr int kTiles = kFit > 4 ? 4 : kFit < 1 ? 1 : kFit;
  static constexpr int kSmem = W * kTiles * kTileBytes;  // and a length a sequence
  // Blocks an SM, as many as registers hold: a fourth where only three fit would run its share of the items after
  // the others (32 sequences of 200..2500, 32/4 heads of 64 f16, 38.3 us against 32.4 with their attention; of 32
  // f32 40.9 against 35.3), and one left out is missed (64 of 130..4096, heads of 32 f16, 55.7 against 53.9).
  static constexpr int kBlocks = DP * sizeof(T) <= 64 ? 4 : 3;
};

template <class T, int DP>
__global__ void __launch_bounds__(Give<T, DP>::W * 32, Give<T, DP>::kBlocks) k_paged_weights(PagedKV c, PagedRows r) {
  using A = Att<T, DP>;
  using B = Give<T, DP>;
  constexpr uint32_t W = B::W, kTiles = B::kTiles;
  extern __shared__ __align__(16) uint8_t sm[];
  uint32_t* const longest_of = reinterpret_cast<uint32_t*>(sm + B::kSmem);  // [n_seqs] (rows longer than the cache give none)
  __shared__ unsigned long long s_tiles;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane / 4, t = lane % 4;
  const uint32_t D = c.D, G = r.heads / c.kvheads, cap = c.max_pages * c.page, chunks = D * (uint32_t)sizeof(T) / 16;
  auto seq_of = [&](uint32_t k) { return r.seq ? r.seq[k] : k; };
  for (uint32_t k = tid; k < c.n_seqs; k += W * 32) longest_of[k] = 0;
  if (tid == 0) s_tiles = 0;
  __syncthreads();
  for (uint32_t k = tid; k < r.rows; k += W * 32) {
    const uint32_t s = seq_of(k), n = r.len[k];
    if (s < c.n_seqs && n <= cap) atomicMax(&longest_of[s], n);
  }
  __syncthreads();
  // tiles of an item: kTiles, or fewer where there are not enough for all warps
  unsigned long long sum = 0;
  for (uint32_t k = tid; k < c.n_seqs; k += W * 32) sum += (longest_of[k] + kTile - 1) / kTile;
  if (sum) atomicAdd(&s_tiles, sum * c.kvheads);
  __syncthreads();
  const uint32_t warps = gridDim.x * W, me = warp * gridDim.x + blockIdx.x;
  const unsigned long long each = (s_tiles + warps - 1) / warps;
  const uint32_t tiles = each < kTiles ? (uint32_t)each : kTiles, span = tiles * kTile;
  if (!tiles) return;
  uint8_t* const tile = sm + warp * kTiles * B::kTileBytes;
  const uint32_t tile_a = smem_addr(tile);
  if (chunks * 16 < DP * sizeof(T)) {
    const uint32_t extra = DP * (uint32_t)sizeof(T) / 16 - chunks;
    for (uint32_t e = lane; e < kTiles * kTile * extra; e += 32)
      *reinterpret_cast<uint4*>(tile + (e / extra) * A::kRow + (chunks + e % extra) * 16) = make_uint4(0, 0, 0, 0);
  }
  // Items of a sequence: (KV head, span of positions).  All sequences' items go to the warps in turn; a lane
  // looks at one of 32 sequences.
  uint32_t total = 0;  // items of the sequences before, modulo the warps
  for (uint32_t s0 = 0; s0 < c.n_seqs; s0 += 32) {
    const uint32_t n_lane = s0 + lane < c.n_seqs ? longest_of[s0 + lane] : 0;
    const uint32_t items_lane = (n_lane + span - 1) / span * c.kvheads;
    uint32_t upto = items_lane % warps;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const uint32_t at_lane = (total + upto - items_lane % warps) % warps;  // the warp with the sequence's first item
    const uint32_t mine_lane = me >= at_lane ? me - at_lane : me + warps - at_lane;
    total = (total + __shfl_sync(0xffffffffu, upto, 31)) % warps;
    for (uint32_t bits = __ballot_sync(0xffffffffu, mine_lane < items_lane); bits; bits &= bits - 1) {
      const int from = __ffs(bits) - 1;
      const uint32_t s = s0 + from, longest = __shfl_sync(0xffffffffu, n_lane, from);
      const uint32_t spans = (longest + span - 1) / span, items = spans * c.kvheads;
      const uint32_t* const pages = c.table + (uint64_t)s * c.max_pages;
      for (uint32_t item = __shfl_sync(0xffffffffu, mine_lane, from); item < items; item += warps) {
        const uint32_t h = item / spans, j0 = item % spans * span;
        float* const w = r.weights + ((uint64_t)s * c.kvheads + h) * cap;
        float old[kTiles], w0[kTiles], w8[kTiles];  // sums of positions g and g + 8 of a tile, this lane's heads
        uint32_t row[kTiles];
#pragma unroll
        for (uint32_t u = 0; u < kTiles; u++) {
          const uint32_t j = j0 + u * kTile + lane % kTile, p = u < tiles && j < longest ? pages[j / c.page] : kNoSlot;
          row[u] = p < c.n_pages ? (p * c.kvheads + h) * c.page + j % c.page : kNoSlot;
        }
#pragma unroll
        for (uint32_t u = 0; u < kTiles; u++) {
          constexpr uint32_t kCh = DP * sizeof(T) / 16;
#pragma unroll 4
          for (uint32_t e = lane; e < kTile * kCh; e += 32) {
            const uint32_t pos = e / kCh, ch = e % kCh, src = __shfl_sync(0xffffffffu, row[u], pos);
            if (ch < chunks)
              copy16(tile_a + u * B::kTileBytes + pos * A::kRow + ch * 16,
                     static_cast<const uint8_t*>(c.k) + (src == kNoSlot ? 0 : (uint64_t)src * D * sizeof(T) + ch * 16),
                     src != kNoSlot);
          }
          const uint32_t slot = j0 + u * kTile + g + 8 * t;
          old[u] = t < 2 && u < tiles && slot < longest ? w[slot] : 0.f;
          w0[u] = w8[u] = 0.f;
        }
        copy_commit();
        // the sequence's rows that reach the span, 8 heads at a time; while one is computed the next is read
        uint32_t k0 = 0, rows = 0, g0 = G, i = 0, reach = 0, len_lane = 0;
        auto next = [&] {
          g0 += 8;
          if (g0 < G) return true;
          while (!rows) {
            if (k0 >= r.rows) return false;
            const bool here = k0 + lane < r.rows;
            len_lane = here ? r.len[k0 + lane] : 0;
            rows = __ballot_sync(0xffffffffu, here && len_lane > j0 && len_lane <= cap && seq_of(k0 + lane) == s);
            k0 += 32;
          }
          const int at = __ffs(rows) - 1;
          rows &= rows - 1;
          i = k0 - 32 + at;
          reach = __shfl_sync(0xffffffffu, len_lane, at);
          g0 = 0;
          return true;
        };
        Query<T, DP> q;
        float next0 = INFINITY, next1 = INFINITY;
        auto read = [&] {
          const uint32_t gn = min(8u, G - g0);
          const uint64_t head = (uint64_t)i * r.heads + h * G + g0;
          q.fetch(r.q + (head + g) * D, D, g < gn);
          next0 = 2 * t < gn ? r.lse[head + 2 * t] : INFINITY;
          next1 = 2 * t + 1 < gn ? r.lse[head + 2 * t + 1] : INFINITY;
        };
        bool more = next();
        if (more) read();
        copy_wait<0>();
        __syncwarp();
        while (more) {
          const uint32_t len = min(reach, j0 + span);
          const float lse0 = fabsf(next0) < INFINITY ? next0 * 1.4426950408889634f : INFINITY;  // (inf: no weights)
          const float lse1 = fabsf(next1) < INFINITY ? next1 * 1.4426950408889634f : INFINITY;
          q.split(r.scale * 1.4426950408889634f);
          more = next();
          if (more) read();
#pragma unroll
          for (uint32_t u = 0; u < kTiles; u++) {
            const uint32_t j = j0 + u * kTile;
            if (j >= len) break;
            float x[4];
            q.template scores<2, 2>(tile_a + u * B::kTileBytes, x);
            const bool in0 = j + g < len, in8 = j + g + 8 < len;
            w0[u] += in0 && lse0 < INFINITY ? pow2(x[0] - lse0) : 0.f;
            w8[u] += in8 && lse0 < INFINITY ? pow2(x[2] - lse0) : 0.f;
            w0[u] += in0 && lse1 < INFINITY ? pow2(x[1] - lse1) : 0.f;
            w8[u] += in8 && lse1 < INFINITY ? pow2(x[3] - lse1) : 0.f;
          }
        }
#pragma unroll
        for (uint32_t u = 0; u < kTiles; u++) {
          w0[u] += __shfl_xor_sync(0xffffffffu, w0[u], 1);
          w8[u] += __shfl_xor_sync(0xffffffffu, w8[u], 1);
          w0[u] += __shfl_xor_sync(0xffffffffu, w0[u], 2);
          w8[u] += __shfl_xor_sync(0xffffffffu, w8[u], 2);
          const uint32_t slot = j0 + u * kTile + g + 8 * t;
          if (u < tiles && t < 2 && slot < longest) w[slot] = old[u] + (t ? w8[u] : w0[u]);
        }
        __syncwarp();  // (the tiles are read)
      }
    }
  }
}

// A weight's place in the order of eviction: larger weights have larger keys, NaN the smallest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t b = __float_as_uint(w + 0.f);  // (-0 counts as 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr uint32_t kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr uint32_t kSelHold = 40960;  // slots whose weights a block holds in shared memory
constexpr uint32_t kHists = 4, kBins = 2048, kSelBlocks = 8;
static_assert(kBins == 2 * kSelThreads, "two bins a thread");

// The slots that (sequence, KV head) keeps, ascending, to kept[..][keep]; kNoSlot behind them, and in
// the first place when the sequence's length or pages are invalid.  Their weights to weights_out.
//
// The want-th largest key is found by its first 11, next 11 and last 10 bits: a histogram of the keys that
// share the bits found so far (four, for every fourth lane: the first bits bunch up), then a scan over its
// bins.  Then the slots above it and the first ones at it are numbered: each thread counts its run of
// slots, and knows its place from the counts of those before.  A cluster of 2^logc blocks shares a
// sequence's slots, the histograms and counts through distributed shared memory: one block alone issues
// its instructions for long (a sequence of 20,011 slots, 4 KV heads, with its rows' move: 25.0 us with 1
// block, 19.9 with 8).  The weights are read once, and held in shared memory; of a sequence that does not
// fit they are read again for each turn.
__global__ void __launch_bounds__(kSelThreads) k_evict_select(PagedKV c, PagedEvict e, uint32_t hold, uint32_t logc) {
  extern __shared__ float held[];  // [hold]
  __shared__ __align__(16) uint32_t hist[kHists][kBins];
  __shared__ uint32_t warp_n[2][kSelWarps];
  __shared__ uint32_t s_bin, s_left, s_sums[kSelBlocks][kSelWarps];
  __shared__ __align__(8) uint2 s_total[2], s_bins[kSelBlocks][32];
  const uint32_t C = 1u << logc, rank = blockIdx.x & (C - 1), unit = blockIdx.x >> logc;
  const uint32_t s = unit / c.kvheads, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t n = e.len[s], cap = c.max_pages * c.page, m = min(n, e.keep);
  uint32_t* const kept = e.kept + (uint64_t)unit * e.keep;
  const float* w = e.weights + (uint64_t)unit * cap;
  float* wo = e.weights_out + (uint64_t)unit * cap;
  bool bad = n > cap;
  if (!bad) {
    for (uint32_t p = tid; p < (n + c.page - 1) / c.page; p += kSelThreads)
      bad |= c.table[(uint64_t)s * c.max_pages + p] >= c.n_pages;
    for (uint32_t p = tid; p < (m + c.page - 1) / c.page; p += kSelThreads)
      bad |= e.dst_table[(uint64_t)s * c.max_pages + p] >= c.n_pages;
  }
  // the slots go by chunks that the cluster holds at once, a run of each to a block
  const uint32_t chunk = hold << logc;
  const bool all = n <= e.keep, fits = n <= chunk;
  auto mine = [&](uint32_t first, uint32_t& from, uint32_t& count) {  // this block's run of the chunk at `first`
    const uint32_t in = min(chunk, n - first), per = (in + C - 1) >> logc, at = min(in, rank * per);
    from = first + at;
    count = min(per, in - at);
  };
  auto hold_weights = [&](uint32_t from, uint32_t count) {  // (eight reads on their way at a time)
    for (uint32_t i0 = tid; i0 < count; i0 += 8 * kSelThreads) {
      float x[8];
#pragma unroll
      for (uint32_t u = 0; u < 8; u++) x[u] = i0 + u * kSelThreads < count ? w[from + i0 + u * kSelThreads] : 0.f;
#pragma unroll
      for (uint32_t u = 0; u < 8; u++)
        if (i0 + u * kSelThreads < count) held[i0 + u * kSelThreads] = x[u];
    }
  };
  uint32_t from = 0, count = 0;
  if (!all && fits && n <= cap) {
    mine(0, from, count);
    hold_weights(from, count);
  }
  bad = __syncthreads_or(bad);
  if (bad || all) {  // (the whole cluster)
    for (uint32_t i = rank * kSelThreads + tid; i < e.keep; i += kSelThreads << logc) {
      kept[i] = !bad && i < n ? i : kNoSlot;
      if (!bad && i < n && wo != w) wo[i] = w[i];
    }
    return;
  }
  if (C > 1) cluster_sync();  // (the blocks of the cluster run: they may be written to)
  const uint32_t old = n - e.recent, want = e.keep - e.recent;
  // the sum of a and of b over the warps before this one, and over all (a, b: the same in all lanes)
  auto scan = [&](uint32_t& a, uint32_t& b, uint32_t& all_a, uint32_t& all_b) {
    if (lane == 0) {
      warp_n[0][warp] = a;
      warp_n[1][warp] = b;
    }
    __syncthreads();
    const uint32_t x = warp_n[0][lane], y = warp_n[1][lane];
    a = __reduce_add_sync(0xffffffffu, lane < warp ? x : 0);
    b = __reduce_add_sync(0xffffffffu, lane < warp ? y : 0);
    all_a = __reduce_add_sync(0xffffffffu, x);
    all_b = __reduce_add_sync(0xffffffffu, y);
    __syncthreads();
  };
  uint32_t T = 0, left = want;  // the key's bits so far; how many of the keys that share them stay
  for (int shift = 21; shift >= 0 && want; shift = shift == 21 ? 10 : shift == 10 ? 0 : -1) {
    const uint32_t bits = shift ? 11 : 10;
    for (uint32_t i = tid; i < kHists * kBins; i += kSelThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    auto add = [&](float x) {
      const uint32_t k = weight_key(x);
      if (shift == 21 || (k ^ T) >> (shift + bits) == 0) atomicAdd(&hist[lane % kHists][k >> shift & ((1u << bits) - 1)], 1);
    };
    if (fits) {
#pragma unroll 4
      for (uint32_t i = tid; i < count; i += kSelThreads)
        if (from + i < old) add(held[i]);
    } else {
#pragma unroll 4
      for (uint32_t i = rank * kSelThreads + tid; i < old; i += kSelThreads << logc) add(w[i]);
    }
    __syncthreads();
    // a warp has 64 bins, a lane two of them (b and b - 1), larger keys first.  The blocks exchange the warps'
    // sums, and then the bins of the one warp that has the bin in question.
    const uint32_t b = kBins - 1 - 2 * tid;
    uint32_t c1 = 0, c0 = 0;
#pragma unroll
    for (uint32_t v = 0; v < kHists; v++) {
      const uint2 x = *reinterpret_cast<const uint2*>(&hist[v][b - 1]);
      c0 += x.x;
      c1 += x.y;
    }
    uint32_t total = __reduce_add_sync(0xffffffffu, c0 + c1);
    if (C > 1) {
      if (lane < C) st_cluster(cluster_addr(smem_addr(&s_sums[rank][warp]), lane), __uint_as_float(total));
      cluster_sync();
      total = 0;
      for (uint32_t k = 0; k < C; k++) total += s_sums[k][warp];
    }
    uint32_t before = total, none = 0, u0, u1;
    scan(before, none, u0, u1);
    const bool hit = before < left && before + total >= left;  // (the same warp in all blocks)
    if (C > 1) {
      if (hit)
        for (uint32_t k = 0; k < C; k++) {
          const uint32_t to = cluster_addr(smem_addr(&s_bins[rank][lane]), k);
          st_cluster(to, __uint_as_float(c0));
          st_cluster(to + 4, __uint_as_float(c1));
        }
      cluster_sync();
      if (hit) {
        c0 = c1 = 0;
        for (uint32_t k = 0; k < C; k++) {
          c0 += s_bins[k][lane].x;
          c1 += s_bins[k][lane].y;
        }
      }
    }
    if (hit) {
      uint32_t sum = c1 + c0;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const uint32_t above = before + sum - c1 - c0;  // keys in the bins before these two
      if (above < left && above + c1 + c0 >= left) {
        const bool second = above + c1 < left;
        s_bin = b - second;
        s_left = left - above - (second ? c1 : 0);
      }
    }
    __syncthreads();
    T |= s_bin << shift;
    left = s_left;
  }
  uint32_t base = 0, ties = 0, turn = 0;  // kept so far; slots at T so far
  for (uint32_t first = 0; first < n; first += chunk, turn ^= 1) {
    if (!fits) {
      mine(first, from, count);
      hold_weights(from, count);
      __syncthreads();
    }
    // a thread takes a run of slots (of an odd length: the threads then read from different banks)
    const uint32_t run = (count + kSelThreads - 1) / kSelThreads | 1, r0 = min(count, tid * run), r1 = min(count, r0 + run);
    auto above = [&](uint32_t i, uint32_t k) { return from + i >= old || (want && k > T); };
    auto tie = [&](uint32_t i, uint32_t k) { return from + i < old && want && k == T; };
    uint32_t a = 0, t = 0, all_a, all_t;
    for (uint32_t i = r0; i < r1; i++) {
      const uint32_t k = weight_key(held[i]);
      a += above(i, k);
      t += tie(i, k);
    }
    uint32_t sa = a, st = t;  // up to and with this thread, in the warp
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const uint32_t ya = __shfl_up_sync(0xffffffffu, sa, o), yt = __shfl_up_sync(0xffffffffu, st, o);
      if (lane >= o) {
        sa += ya;
        st += yt;
      }
    }
    uint32_t wa = __shfl_sync(0xffffffffu, sa, 31), wt = __shfl_sync(0xffffffffu, st, 31);
    scan(wa, wt, all_a, all_t);
    // the blocks before this one.  (Past this barrier the whole chunk is read, so its slots may be written:
    // what a chunk writes lies below all that later ones read.)
    if (C > 1) {
      if (tid == 0) s_total[turn] = make_uint2(all_a, all_t);
      cluster_sync();
      all_a = all_t = 0;
      for (uint32_t k = 0; k < C; k++) {
        const uint2 x = ld_cluster2(cluster_addr(smem_addr(&s_total[turn]), k));
        if (k < rank) {
          wa += x.x;
          wt += x.y;
        }
        all_a += x.x;
        all_t += x.y;
      }
    }
    const uint32_t ties_in = min(ties, left);
    uint32_t ties_at = ties + wt + st - t, to = base + wa + sa - a + min(ties_at, left) - ties_in;
    for (uint32_t i = r0; i < r1; i++) {
      const uint32_t k = weight_key(held[i]);
      const bool at_T = tie(i, k);
      // (the ties that stay come among the others in slot order: as many before this one as fit)
      if (above(i, k) || (at_T && ties_at < left)) {
        kept[to] = from + i;
        wo[to] = held[i];
        to++;
      }
      ties_at += at_T;
    }
    base += all_a + min(ties + all_t, left) - ties_in;
    ties += all_t;
    __syncthreads();
  }
  if (C > 1) cluster_sync();  // (the others have read this block's counts)
}

// Rows kept[i] of K or V to slot i, in 16-byte pieces: block (x: sequence and KV head; y:
// K or V, and its share of a row's pieces; z: its share of the rows).  In place a sequence's rows move to
// lower slots, kept[i] >= i ascending, so one block takes them all, tile by tile: a tile is written only
// when the block has read it, and what it writes lies below all that later tiles read.  The rows before the first
// that moves are left alone, up to a 256th of all (64 sequences of 4000 slots of 4 x 128 bf16 within their budget:
// 15 us, 400 with their rows written where they are).  Elsewhere the tiles are spread over the blocks.
constexpr uint32_t kMoveThreads = 256, kMoveRows = 128;  // rows of a tile

template <class T>
__global__ void __launch_bounds__(kMoveThreads) k_evict_move(PagedKV c, PagedEvict e, uint32_t shares) {
  __shared__ uint32_t from_row[2][kMoveRows], to_row[2][kMoveRows];
  const uint32_t s = blockIdx.x / c.kvheads, h = blockIdx.x % c.kvheads, tid = threadIdx.x;
  const uint32_t share = blockIdx.y >> 1;
  const uint32_t* const kept = e.kept + (uint64_t)blockIdx.x * e.keep;
  const uint32_t n = e.len[s], m = min(n, e.keep);
  // (new_len may be len: who reads it after this has the same m)
  if (blockIdx.y == 0 && h == 0 && blockIdx.z == 0 && tid == 0) e.new_len[s] = kept[0] == kNoSlot ? n : m;
  if (kept[0] == kNoSlot) return;  // nothing cached, or an invalid sequence
  const uint32_t pieces = c.D * (uint32_t)sizeof(T) / 16, per = (pieces + shares - 1) / shares;
  const uint32_t c0 = share * per, cn = min(pieces, c0 + per) - min(pieces, c0);
  if (!cn) return;
  uint8_t* const pool = static_cast<uint8_t*>(blockIdx.y & 1 ? c.v : c.k) + c0 * 16;
  constexpr uint32_t kHold = 8;  // pieces a thread holds at once
  const uint32_t step_row = kMoveThreads / cn, step_piece = kMoveThreads % cn;
  uint32_t turn = 0, r0 = blockIdx.z * kMoveRows;
  if (e.dst_table == c.table) {  // (kept[i] - i never falls: who has it 0 at the end of a run has it 0 all through)
    const uint32_t run = (m + kMoveThreads - 1) / kMoveThreads, last = min(m, (tid + 1) * run) - 1;
    r0 = run * __syncthreads_count(tid * run < m && kept[last] == last);
  }
  for (; r0 < m; r0 += gridDim.z * kMoveRows, turn ^= 1) {
    const uint32_t rows = min(kMoveRows, m - r0);
    if (tid < rows) {
      from_row[turn][tid] = (uint32_t)pool_row(c, c.table, s, h, kept[r0 + tid]);
      to_row[turn][tid] = (uint32_t)pool_row(c, e.dst_table, s, h, r0 + tid);
    }
    __syncthreads();
    uint32_t row = tid / cn, piece = tid % cn;
    for (uint32_t done = 0; done < rows * cn; done += kHold * kMoveThreads) {
      uint4 x[kHold];
      uint32_t row2 = row, piece2 = piece;
      auto advance = [&](uint32_t& r, uint32_t& p) {
        r += step_row;
        p += step_piece;
        if (p >= cn) {
          p -= cn;
          r++;
        }
      };
#pragma unroll
      for (uint32_t u = 0; u < kHold; u++) {
        if (row < rows) x[u] = *reinterpret_cast<const uint4*>(pool + ((uint64_t)from_row[turn][row] * pieces + piece) * 16);
        advance(row, piece);
      }
      __syncthreads();  // all of this part is read
#pragma unroll
      for (uint32_t u = 0; u < kHold; u++) {
        if (row2 < rows) *reinterpret_cast<uint4*>(pool + ((uint64_t)to_row[turn][row2] * pieces + piece2) * 16) = x[u];
        advance(row2, piece2);
      }
    }
  }
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
  const uint32_t pieces = c.kvheads * (c.D * (c.kind == F32 ? 4 : 2) / 16), threads = pieces < 256 ? (pieces + 31) / 32 * 32 : 256;
  QC_BY_KIND(c.kind, (k_paged_append<T><<<rows, threads, 0, st>>>(c, k, v, seq, pos, weights)));
  return cudaGetLastError();
}

namespace {


template <class T, int DP, int W, int R>
cudaError_t att_prepare() {
  static_assert(Att<T, DP>::fixed(W, R) <= 227 * 1024, "shared memory of a block");
  auto* f = k_paged_attention<T, DP, W, R>;
  cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, Att<T, DP>::fixed(W, R));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

// A cluster of C blocks of W warps takes a row and KV head, or with R > 1 a group of `rows` rows.
template <class T, int DP, int W, int R>
cudaError_t att_launch(const PagedKV& c, const PagedRows& r, uint32_t C, uint32_t rows, cudaStream_t st) {
  using A = Att<T, DP>;
  AttSplit sp{C, 0, 0, rows, false};
  const uint32_t clusters = R > 1 ? (r.rows + rows - 1) / rows : r.rows;
  // Where the blocks take more than one turn on the GPU (three an SM) and fewer than three, the short rows should be
  // the last: 21 sequences of 0..1531 positions in f32 26.9 -> 24.1 us, 64 of 130..4096 in bf16 63.1 -> 60.2, 96 of
  // them 88.5 -> 84.6.  The lengths are not known here: equal ones lose by the later start (64 of 4096, 103 -> 106;
  // 32 of them 62.6 -> 64.9).  With more turns the end matters less (128 of 130..2048: 62.5 either way).
  const uint32_t blocks = clusters * c.kvheads * C;
  sp.longest_first = R == 1 && r.rows > 1 && r.rows <= kMaxSorted && blocks > 3 * kSMs && blocks <= 8 * kSMs;
  const uint32_t step = W * kTile * C;
  sp.step_pages = step / c.page;
  sp.step_slots = step % c.page;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(clusters * C, c.kvheads);
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = A::fixed(W, R);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_paged_attention<T, DP, W, R>, c, r, sp);
}

// Blocks of a cluster, and warps of a block.  Where the largest clusters leave SMs to spare, as many as there
// are tiles for, and wide blocks (one sequence of 32,768 positions in bf16, 4 KV heads: 41.7 us with 4 warps,
// 26.5 with 8; of 8192, 14.2 and 12.0).  Else enough small blocks to fill the GPU (three an SM) nearly twice, as the
// sequences' lengths differ and are not known here, as long as a warp keeps six tiles of a full cache: 64 of
// 130..4096, 4 KV heads, 80 us with 1 block, 60 with this rule's 4, 75 with 8; 16 of 1000..8192, 46 with 4, 43 with
// 8, 49 with 16.  Large clusters leave parts of a GPC unused; where they would not all find room at once, clusters
// that do are better (8 of 9000..32768: 74 us with 12 blocks, 80 with 16, 87 with 8).
// What the rule misses: equal lengths need no second turn (64 of 4096: 106 us, 90 with 1 block), and next to its
// bounds half the blocks can be better (32 of 130..4096: 41 with 8, 36 with 4; 6 rows of 7001: 36 with 16, 23 with 8).
template <class T, int DP>
cudaError_t att_launch(const PagedKV& c, const PagedRows& r, cudaStream_t st) {
  using A = Att<T, DP>;
  const uint32_t tiles = (uint32_t)(((uint64_t)c.max_pages * c.page + kTile - 1) / kTile);
  cudaError_t e = cudaSuccess;
  uint32_t C = 1, rows = 1;
  if (r.shared) {
    // Groups of neighbouring rows of one sequence, as prompts have them, read every tile once: as many rows as
    // make R units of 8 columns.  512 rows of 4096 positions, 32/4 heads of 128 bf16: 466 us -> 361, 256 rows of
    // 1024 with 8/8 heads of 64 f16 75 -> 18.5; 8 rows of 4096, which fill fewer blocks, 17 -> 23.  Other rows are left
    // to the other kernel.  Where there are many, two kernels take longer than one (60 single rows beside a prompt's
    // 100: 157 us against 120; 30 beside 256: 222 against 211), so the callers ask for groups only where they expect
    // nearly all rows to form them: a batch, which knows its rows, where 15 of 16 neighbours are of one sequence,
    // qc_paged_attention where there are 16 rows for every sequence of the table.  That says nothing about the order:
    // 512 rows of 4 sequences in turn form no group and take 464 us, 455 without the first launch, and 512 rows of one
    // sequence in a table of 64 stay by themselves, 490 us instead of 372.
    const uint32_t G = r.heads / c.kvheads;
    rows = 8 * A::kShared / G;
    if (rows < 2) rows = 1;
    if (rows > 1) {
      const uint32_t units = (r.rows + rows - 1) / rows * c.kvheads;
      while (C < (uint32_t)kMaxCluster && tiles > A::W * C && units * C < kSMs) C *= 2;
      e = att_launch<T, DP, A::W, A::kShared>(c, r, C, rows, st);
      C = 1;
    }
  }
  const uint32_t units = r.rows * c.kvheads;
  while (C < (uint32_t)kMaxCluster && tiles > A::W * C &&
         (units * C < kSMs || (units * C < 700 && tiles >= 12 * A::W * C)))
    C *= 2;
  if (C == (uint32_t)kMaxCluster && units > 384 / C) C = 384 / units > 8 ? 384 / units : 8;
  const bool wide = units * C <= kSMs && tiles > A::W * C;
  if (e == cudaSuccess)
    e = wide ? att_launch<T, DP, A::kWide, 1>(c, r, C, rows, st) : att_launch<T, DP, A::W, 1>(c, r, C, rows, st);
  if (r.weights && e == cudaSuccess) {
    using B = Give<T, DP>;
    const uint32_t smem = B::kSmem + c.n_seqs * 4, per_sm = 225 * 1024 / (smem + 1024), most = B::kBlocks;
    k_paged_weights<T, DP><<<kSMs * (per_sm > most ? most : per_sm), B::W * 32, smem, st>>>(c, r);
    e = cudaGetLastError();
  }
  return e;
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
    return att_launch<T, DP>(c, r, st);
  }
};
struct AttPrepare {
  template <class T, int DP>
  cudaError_t operator()() const {
    using A = Att<T, DP>;
    static_assert(Give<T, DP>::kSmem + (int)kMaxWeightSeqs * 4 <= 227 * 1024, "shared memory of a block");
    cudaError_t e = att_prepare<T, DP, A::W, 1>();
    if (e == cudaSuccess) e = att_prepare<T, DP, A::kWide, 1>();
    if (e == cudaSuccess) e = att_prepare<T, DP, A::W, A::kShared>();
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(k_paged_weights<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               Give<T, DP>::kSmem + (int)kMaxWeightSeqs * 4);
    return e;
  }
};

}  // namespace

// Once per device, before launch_paged_attention.
cudaError_t paged_prepare() {
  cudaError_t e = cudaFuncSetAttribute(k_evict_select, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelHold * 4);
  cudaFuncAttributes loaded;  // (a kernel is loaded when it is first asked about: not in a capture)
  for (uint32_t kind : {(uint32_t)F32, (uint32_t)F16, (uint32_t)BF16}) {
    if (e == cudaSuccess) QC_BY_KIND(kind, e = cudaFuncGetAttributes(&loaded, k_paged_append<T>));
    if (e == cudaSuccess) QC_BY_KIND(kind, e = cudaFuncGetAttributes(&loaded, k_evict_move<T>));
  }
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
  const uint32_t units = c.n_seqs * c.kvheads, pieces = c.D * (c.kind == F32 ? 4 : 2) / 16;
  // blocks a sequence and KV head: to fill the GPU, of 4096 slots at least
  const uint32_t cap = c.max_pages * c.page;
  uint32_t logc = 0;
  while (1u << logc < kSelBlocks && ((uint64_t)units << logc) < kSMs && cap > 4096u << logc) logc++;
  const uint32_t per = (cap + (1u << logc) - 1) >> logc, hold = per < kSelHold ? per : kSelHold;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(units << logc);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = hold * 4;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1u << logc;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t err = cudaLaunchKernelEx(&cfg, k_evict_select, c, e, hold, logc);
  if (err != cudaSuccess) return err;
  // Enough blocks to fill the GPU, where there are few sequences: by rows, or in place by parts of a row
  // (64 bytes at least).
  uint32_t shares = 1, tiles = 1;
  if (e.dst_table == c.table)
    while ((uint64_t)units * 2 * shares < 8 * kSMs && pieces / (shares * 2) >= 4) shares *= 2;
  else
    while ((uint64_t)units * 2 * tiles < 16 * kSMs && tiles * kMoveRows < e.keep) tiles *= 2;
  QC_BY_KIND(c.kind, (k_evict_move<T><<<dim3(units, 2 * shares, tiles), kMoveThreads, 0, st>>>(c, e, shares)));
  return cudaGetLastError();
}

}  // namespace qc
