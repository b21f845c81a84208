// Low-rank updates of many adapters, and their gradients.  A row i of x has the adapter e = ids[i] with factors A_e [rank][in] and B_e [out][rank]:
//
//   forward    h_i = A_e x~_i;   y_i = base_i + s_e B_e h_i                   x~: x, or what dropout leaves of it (philox.cuh)
//   backward   g_i = B_e^T dy_i; dx_i = s_e A_e^T g_i (dropped again);  dA_e = s_e sum_i g_i x~_i^T;  dB_e = s_e sum_i dy_i h_i^T
//
// Both directions of the rows are the same two products: one over a long axis that leaves `rank` values a row, and one from these to a long axis.  Few rows
// (lr_rows_kernel): a cluster of blocks takes one tile of rows of one adapter; each block multiplies its part of the long axis, the parts meet
// over distributed shared memory in one order, and each block writes its part of the columns.  One launch, no atomics; rank values leave the chip only
// where a backward pass wants them.  Many rows: the same kernel stops at the rank values and lr_expand_kernel makes the second product.  The factors'
// gradients (lr_outer_kernel) are sums over an adapter's rows, split over a cluster and joined the same way.
//
// All are bound by memory: 2 rank operations for each value that is read.  So the matrix instructions are mma.sync, whose operands are gathered rows
// from shared memory; tcgen05 would want tiles of 128 rows and does not pay at one operation a byte.  The long product of 16-bit types multiplies them as they are
// (f32 sums); everything that meets the rank values keeps these in two TF32 parts, 22 bits, beside 16-bit operands that TF32 holds exactly.  f32 operands are
// two TF32 parts too, three products of them, added to f32 registers every few steps because the matrix instructions' own sums truncate.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <map>
#include <mutex>
#include <type_traits>
#include <utility>

#include "common.cuh"
#include "philox.cuh"

namespace bonsai {

constexpr int kLrThreads = 256, kLrWarps = 8, kLrSelf = 256;      // kLrSelf: rows that blocks group by themselves
// From so many rows and results on the two products are kernels of their own: each is then a stream over memory with as many blocks as it likes.  bf16, rank 16,
// us in one kernel and in two: 2000 rows 4096 to 4096 19 and 23, 4000 rows 34 and 37, 2000 rows 4096 to 12288 38 and 34, 8000 rows 4096 to 4096 67 and 49,
// to 12288 143 and 94.
constexpr int kLrSplit = 1024;
inline bool lr_split_at(int n, int cols) { return n >= kLrSplit && (long long)n * cols >= 1 << 24; }
constexpr int kLrSmemMost = 227 * 1024 - 2048, kLrSmemHalf = 112 * 1024, kLrSmemThird = 74 * 1024;        // dynamic shared memory of a block, of each of two or three on an SM
constexpr int kLrOuterCols = 128, kLrOuterRows = 64;
enum LrGrouping { LR_ONE = 0, LR_SELF = 1, LR_PLAN = 2 };

struct LrGroups {            // which rows have which adapter
  int mode;
  const void* ids;           // LR_SELF
  int ids_wide;              // int64, else int32
  const int* order;          // LR_PLAN: rows by adapter; behind them those without one, and those whose id names none
  const int* start;          // [adapters + 3]: where each adapter's rows begin in it
  const int4* tiles;         // LR_PLAN where a product is split: tiles of 16 rows: group (-1: none), place, number of rows
  const int* tile_rows;      // and their rows, -1 behind the last
  int n, adapters;
};

// The rank values of a forward or a backward pass, times the adapter's scale, by place in the order: f32 [n][R] (R: the padded rank), of bf16 two parts [2][n][R].  f16 for the second
// product: two parts over a power of two for each row, and that power.
struct LrValues {
  void* values;
  __half* parts;
  float* factors;
};

struct LrRowsArgs {
  LrGroups groups;
  const void* x; long long ldx;          // [n][k]
  const void *w1, *w2;                   // forward: A, B; backward: B, A
  const void* base; long long ld_base;   // [n][cols], may be null
  void* y; long long ldy;                // null: the rank values alone are wanted
  LrValues kept;                         // null where nothing is kept
  const float* scales;                   // of the adapters, or null: scale
  float scale;
  int k, cols, rank;
  int split;                             // two kernels: lr_split_at
  int vec_x, vec_w1, vec_w2, vec_y;      // rows that 16-byte (w2 of the forward pass: 8-byte) accesses may take
  DropoutRule drop;
  int drop_x, drop_y;                    // forward: the rows of x; backward: those of dx
};

struct LrOuterArgs {
  LrGroups groups;
  // two products of one launch: 0: dA [rank][k] from x (dropped) and g, 1: dB [cols][rank] from dy and h
  const void* q[2]; long long ldq[2];
  const void* p[2];                      // `kept` of the rows
  void* out[2];
  int width[2], blocks[2], vec[2];       // columns, blocks of columns
  int rank;
  DropoutRule drop;
  int drop_x;
};

// ---- values ------------------------------------------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float lr_float(T v);
template <> __device__ __forceinline__ float lr_float(float v) { return v; }
template <> __device__ __forceinline__ float lr_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float lr_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T lr_round(float v);
template <> __device__ __forceinline__ float lr_round(float v) { return v; }
template <> __device__ __forceinline__ __half lr_round(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 lr_round(float v) { return __float2bfloat16_rn(v); }
// the two halves of a word of 16-bit values
template <typename T> __device__ __forceinline__ float2 lr_pair(uint32_t w);
template <> __device__ __forceinline__ float2 lr_pair<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 lr_pair<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 lr_pair<float>(uint32_t w) { return make_float2(__uint_as_float(w), 0.0f); }     // not used

// two values rounded into a word
template <typename T> __device__ __forceinline__ uint32_t lr_two(float a, float b);
template <> __device__ __forceinline__ uint32_t lr_two<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t lr_two<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// eight neighbouring values
template <typename T, bool VEC>
__device__ __forceinline__ void lr_load8(const T* p, int n, float* v) {
  if (VEC) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = lr_pair<T>(w[i]);
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? lr_float<T>(p[i]) : 0.0f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void lr_store8(T* p, int n, const float* v) {
  if (VEC) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(lr_two<T>(v[0], v[1]), lr_two<T>(v[2], v[3]), lr_two<T>(v[4], v[5]), lr_two<T>(v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = lr_round<T>(v[i]);
  }
}

// ---- shared memory, matrix instructions --------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t lr_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void lr_copy16(void* dst, const void* src, bool there) {       // zeros where it is not there
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(lr_smem(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void lr_copy16(void* dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(lr_smem(dst)), "l"(src) : "memory"); }
__device__ __forceinline__ void lr_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void lr_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void lr_ldm4(uint32_t* r, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(lr_smem(p)) : "memory");
}
__device__ __forceinline__ void lr_ldm4t(uint32_t* r, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(lr_smem(p)) : "memory");
}
// d = a b + d
#define LR_MMA(name, shape, types)                                                                                                           \
  __device__ __forceinline__ void name(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {                                              \
    asm volatile("mma.sync.aligned." shape ".row.col.f32." types ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"                \
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                                            \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));                                                            \
  }
LR_MMA(lr_mma_f16, "m16n8k16", "f16.f16")
LR_MMA(lr_mma_bf16, "m16n8k16", "bf16.bf16")
LR_MMA(lr_mma8, "m16n8k8", "tf32.tf32")
#undef LR_MMA
template <typename T>
__device__ __forceinline__ void lr_mma16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) lr_mma_f16(d, a, b0, b1);
  else lr_mma_bf16(d, a, b0, b1);
}
__device__ __forceinline__ uint32_t lr_tf32(float v) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return r;
}
// v = hi + lo to 2^-23; an infinity has no second part
__device__ __forceinline__ void lr_split(float v, uint32_t& hi, uint32_t& lo) {
  hi = lr_tf32(v);
  const float h = __uint_as_float(hi);
  lo = fabsf(h) <= 3.4028234e38f ? lr_tf32(v - h) : 0u;
}

// ---- clusters ------------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t lr_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t lr_ranks() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void lr_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void lr_meet() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 lr_remote4(const float* p, uint32_t rank) {
  uint32_t at;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(lr_smem(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

// ---- groups of rows ----------------------------------------------------------------------------------------------------------------------
// adapters: group `adapters` are the rows without one, adapters + 1 those whose id names none
__device__ __forceinline__ int lr_group(const LrGroups& g, int row) {
  const long long id = g.ids_wide ? ((const long long*)g.ids)[row] : (long long)((const int*)g.ids)[row];
  return id < 0 ? g.adapters : id < g.adapters ? (int)id : g.adapters + 1;
}

struct LrTile {
  int group, count, place;   // rows in it, place of its first one in the order
};

// The tile of rows of slot `slot`; rows[i]: its row numbers, -1 behind the last.  Every block of a cluster finds the same one.
template <int M>
__device__ __forceinline__ LrTile lr_tile(const LrGroups& g, int slot, int* rows, int* s) {
  const int t = threadIdx.x;
  LrTile tile = {0, 0, 0};
  if (g.mode == LR_ONE) {
    tile.place = slot * M;
    tile.count = g.n - tile.place < M ? g.n - tile.place : M;
    if (t < M) rows[t] = t < tile.count ? tile.place + t : -1;
  } else if (g.mode == LR_SELF) {
    // Row `slot` leads a tile where the rows of its adapter before it fill whole tiles: it and the next ones are the tile.
    const int mine = lr_group(g, slot), of = t < g.n ? lr_group(g, t) : -1;
    const int before = __syncthreads_count(of == mine && t < slot);
    if (before % M != 0) return tile;
    if (t < M) rows[t] = -1;
    const bool in = of == mine && t >= slot;
    const unsigned b = __ballot_sync(0xffffffffu, in);
    if ((t & 31) == 0) s[t >> 5] = __popc(b);
    __syncthreads();
    int at = __popc(b & ((1u << (t & 31)) - 1u)), all = 0;
    for (int w = 0; w < kLrWarps; ++w) {
      at += w < (t >> 5) ? s[w] : 0;
      all += s[w];
    }
    if (in && at < M) rows[at] = t;
    tile.group = mine;
    tile.count = all < M ? all : M;
  } else {
    for (int e = t; e < g.adapters + 2; e += kLrThreads) {
      const int lo = g.start[e], hi = g.start[e + 1], first = lo / M + e;
      if (slot >= first && slot <= hi / M + e) { s[0] = e; s[1] = lo + (slot - first) * M; s[2] = hi; }
    }
    __syncthreads();
    tile.group = s[0];
    tile.place = s[1];
    const int left = s[2] - tile.place;
    if (left <= 0) return tile;
    tile.count = left < M ? left : M;
    if (t < M) rows[t] = t < tile.count ? g.order[tile.place + t] : -1;
  }
  __syncthreads();
  return tile;
}

// Eight values of a row in shared memory, those that dropout takes set to 0; what stays is scaled behind the sums.  The thread that copied them calls it.
template <typename T>
__device__ __forceinline__ void lr_drop8(T* p, const uint4& words, unsigned limit) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float4 f = reinterpret_cast<float4*>(p)[h];
      f.x = dropout_keeps(words, 4 * h, limit) ? f.x : 0.0f; f.y = dropout_keeps(words, 4 * h + 1, limit) ? f.y : 0.0f;
      f.z = dropout_keeps(words, 4 * h + 2, limit) ? f.z : 0.0f; f.w = dropout_keeps(words, 4 * h + 3, limit) ? f.w : 0.0f;
      reinterpret_cast<float4*>(p)[h] = f;
    }
  } else {
    uint4 w = *reinterpret_cast<uint4*>(p);
    w.x = dropout_pair(w.x, words.x, limit); w.y = dropout_pair(w.y, words.y, limit);
    w.z = dropout_pair(w.z, words.z, limit); w.w = dropout_pair(w.w, words.w, limit);
    *reinterpret_cast<uint4*>(p) = w;
  }
}

// Eight values into shared memory, of which `left` are there, zeros for the others (all of them or none where `vec`).  any: a readable address.
template <typename T>
__device__ __forceinline__ void lr_copy8(T* dst, const T* src, int left, bool vec, const T* any) {
  if (vec) {
    if (left <= 0) src = any;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) lr_copy16(dst + i * (16 / sizeof(T)), src + (left > 0 ? i * (16 / (int)sizeof(T)) : 0), left > 0);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = i < left ? src[i] : lr_round<T>(0.0f);
  }
}

// ---- the second product ------------------------------------------------------------------------------------------------------------------------
// A warp takes 16 rows and 32 columns at a time, four matrix instructions wide.  Column 8 (c / 2) + 2 j + c % 2 is column c of the j-th, so that the eight
// values that a thread has of a row lie side by side.  Of the rank values a thread has 4 t .. 4 t + 3 of every sixteen (f32: 2 t and 2 t + 1 of
// every eight): the axis of a product may be taken in any order, and so its factors lie side by side too.
template <typename T> struct LrStep {
  static constexpr int kStep = sizeof(T) == 4 ? 8 : 16, kEach = kStep / 4;
};

template <typename T, bool BACK>
struct LrFactor {              // w2 of one adapter: forward [cols][rank], backward [rank][cols]
  const T* p;                  // this thread's first value
  int cols, rank, vec, g, t;
  __device__ __forceinline__ LrFactor(const T* w2, int cols, int rank, int vec, int g, int t)
      : p(BACK ? w2 + (long long)(LrStep<T>::kEach * t) * cols + 8 * (g >> 1) : w2 + (long long)(8 * (g >> 1) + (g & 1)) * rank + LrStep<T>::kEach * t),
        cols(cols), rank(rank), vec(vec), g(g), t(t) {}
  // columns 32 b and on, rank values k and on; `at`: first + k of the first (forward), all columns and words there, RANK the rank
  template <int RANK>
  __device__ __forceinline__ static void whole(const T* at, long long cols, int k, int g, int t, uint32_t (*w)[2]) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int kEach = LrStep<T>::kEach;
    const bool there = RANK % LrStep<T>::kStep == 0 ? k < RANK : k + kEach * t < RANK;         // behind the rank lies what is not this adapter's
    if (BACK) {
      uint32_t v[kEach][F32 ? 8 : 4];
#pragma unroll
      for (int i = 0; i < kEach; ++i)
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
          const uint4 u = there ? reinterpret_cast<const uint4*>(at + i * cols)[h] : make_uint4(0, 0, 0, 0);
          v[i][4 * h] = u.x; v[i][4 * h + 1] = u.y; v[i][4 * h + 2] = u.z; v[i][4 * h + 3] = u.w;
        }
      pick(v, g, w);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint2 u = there ? *reinterpret_cast<const uint2*>(at + 2 * j * RANK) : make_uint2(0, 0);
        w[j][0] = u.x; w[j][1] = u.y;
      }
    }
  }
  template <typename V>
  __device__ __forceinline__ static void pick(const V& v, int g, uint32_t (*w)[2]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        w[j][0] = g & 1 ? v[0][2 * j + 1] : v[0][2 * j];
        w[j][1] = g & 1 ? v[1][2 * j + 1] : v[1][2 * j];
      } else {
        const unsigned half = g & 1 ? 0x7632u : 0x5410u;        // the upper or the lower halves of two words
        w[j][0] = __byte_perm(v[0][j], v[1][j], half);
        w[j][1] = __byte_perm(v[LrStep<T>::kEach - 2][j], v[LrStep<T>::kEach - 1][j], half);
      }
    }
  }
  // as they are, with everything checked
  __device__ __forceinline__ void load(int b, int k, uint32_t (*w)[2]) const {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int kEach = LrStep<T>::kEach;
    const int wc = b * 32 + 8 * (g >> 1), kk = k + kEach * t;      // eight columns, of which this thread takes every second
    if (BACK) {
      uint32_t v[kEach][F32 ? 8 : 4];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const T* q = p + (long long)(k + i) * cols + b * 32;
        const bool there = kk + i < rank && wc < cols;
        if (vec) {
#pragma unroll
          for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
            const uint4 u = there ? reinterpret_cast<const uint4*>(q)[h] : make_uint4(0, 0, 0, 0);
            v[i][4 * h] = u.x; v[i][4 * h + 1] = u.y; v[i][4 * h + 2] = u.z; v[i][4 * h + 3] = u.w;
          }
        } else {
          __align__(16) T e[8];
#pragma unroll
          for (int h = 0; h < 8; ++h) e[h] = there && wc + h < cols ? q[h] : lr_round<T>(0.0f);
#pragma unroll
          for (int h = 0; h < (F32 ? 8 : 4); ++h) v[i][h] = reinterpret_cast<const uint32_t*>(e)[h];
        }
      }
      pick(v, g, w);
    } else {
      const T* first = p + (long long)b * 32 * rank + k;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int cc = wc + 2 * j + (g & 1);
        const T* q = first + 2 * j * rank;
        if (vec) {
          const uint2 u = cc < cols && kk < rank ? *reinterpret_cast<const uint2*>(q) : make_uint2(0, 0);
          w[j][0] = u.x; w[j][1] = u.y;
        } else {
          __align__(8) T e[kEach];
#pragma unroll
          for (int h = 0; h < kEach; ++h) e[h] = cc < cols && kk + h < rank ? q[h] : lr_round<T>(0.0f);
          w[j][0] = reinterpret_cast<const uint32_t*>(e)[0];
          w[j][1] = reinterpret_cast<const uint32_t*>(e)[1];
        }
      }
    }
  }
};

// acc += the rank values of 16 rows (two parts) times the factors of 32 columns
template <typename T>
__device__ __forceinline__ void lr_multiply(float (*acc)[4], const uint32_t* hi, const uint32_t* lo, const uint32_t (*w)[2]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      uint32_t h0, l0, h1, l1;
      lr_split(__uint_as_float(w[j][0]), h0, l0);
      lr_split(__uint_as_float(w[j][1]), h1, l1);
      lr_mma8(acc[j], lo, h0, h1);
      lr_mma8(acc[j], hi, l0, l1);
      lr_mma8(acc[j], hi, h0, h1);
    } else {
      lr_mma16<T>(acc[j], lo, w[j][0], w[j][1]);
      lr_mma16<T>(acc[j], hi, w[j][0], w[j][1]);
    }
  }
}

// What the sums of a block start from.  bf16: base itself, so that the matrix instructions add it; a last bit of f32 that they cut off is far below bf16's.
// f32 would lose that bit, f16 has its rows over a power of two: zeros, and base is added behind.
template <typename T> struct LrStart {
  static constexpr bool kBase = std::is_same<T, __nv_bfloat16>::value;
};
// the eight values of row g + 8 h that a thread has in the sums
template <typename T>
__device__ __forceinline__ void lr_set(float (*acc)[4], int h, const float* v) {
#pragma unroll
  for (int q = 0; q < 8; ++q) acc[q >> 1][2 * h + (q & 1)] = v[q];
}
template <typename T>
__device__ __forceinline__ void lr_get(float (*acc)[4], int h, float up, const float* base, float* v) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float d = acc[q >> 1][2 * h + (q & 1)];
    v[q] = LrStart<T>::kBase ? d : std::is_same<T, __half>::value ? fmaf(d, up, base[q]) : d + base[q];
  }
}
__device__ __forceinline__ void lr_drop(float* v, const uint4& words, unsigned limit) {
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = dropout_keeps(words, q, limit) ? v[q] : 0.0f;
}

// f16: the power of two that brings a row's largest rank value between 2^13 and 2^14, and one over it; 1 for zeros, infinities and what is next to them
__device__ __forceinline__ float lr_power(float top, float& down) {
  const int e = (int)(__float_as_uint(top) >> 23 & 255u) - 127 - 13;
  const bool scaled = top > 1e-30f && top < 1e30f;
  down = scaled ? __uint_as_float((unsigned)(127 - e) << 23) : 1.0f;
  return scaled ? __uint_as_float((unsigned)(127 + e) << 23) : 1.0f;
}
template <typename T>
__device__ __forceinline__ void lr_parts(const float* f, T* hi, T* lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi[i] = lr_round<T>(f[i]);
    const float h = lr_float<T>(hi[i]);
    lo[i] = lr_round<T>(fabsf(h) <= 3.4028234e38f ? f[i] - h : 0.0f);
  }
}

// ---- the rows ------------------------------------------------------------------------------------------------------------------------------
template <typename T, int M> struct LrShape {
  static constexpr int kM16 = M / 16, kParts = kLrWarps / kM16;       // warps over rows, and over the long axis
  static constexpr int kChunk = M == 64 && sizeof(T) == 4 ? 64 : 128, kWarpK = kChunk / kParts;
};

// SPLIT: the rank values are all that is made.  Else they wait for the second product in two parts, each of the inputs' 16-bit type (f16 over a power of two for
// each row, so that neither large nor small ones are lost) or TF32, and tiles have 16 rows.
template <typename T, int R, int M, bool BACK, bool SPLIT> struct LrSmem {
  static constexpr int kPad = 16 / sizeof(T);
  static constexpr int kChunk = LrShape<T, M>::kChunk;
  static constexpr int kPitchX = kChunk + kPad, kPitchW = BACK ? R + 8 : kChunk + kPad, kRowsW = BACK ? kChunk : R;
  static constexpr int kStage = (M * kPitchX + kRowsW * kPitchW) * (int)sizeof(T);
  static constexpr int kJoin = LrShape<T, M>::kParts * M * R * 4;         // the warps' parts, over the stages
  static constexpr int kPart = M * R * 4, kPitchH = R + 8, kH = SPLIT ? 0 : 2 * M * kPitchH * (int)sizeof(T);
  // what of base is on its way: each lane's own 16 bytes, `kDepth` steps of a warp
  static constexpr int kDepth = sizeof(T) == 4 ? 2 : 4, kPieces = (int)sizeof(T);
  static constexpr int kBase = BACK || SPLIT ? 0 : kLrWarps * kDepth * kPieces * 512;
  // as many stages as leave room for two blocks on an SM (three that make rank values of 16-bit types), or one where the rank is large
  static constexpr int kMost = SPLIT && R == 16 && sizeof(T) == 2 ? kLrSmemThird : R <= 32 ? kLrSmemHalf : kLrSmemMost;
  static constexpr int ring(int stages) { return stages * kStage > kJoin ? stages * kStage : kJoin; }
  static constexpr int bytes(int stages) { return ring(stages) + kPart + kH + kBase; }
  static constexpr int kStages = bytes(4) <= kMost ? 4 : bytes(3) <= kMost ? 3 : 2, kRing = ring(kStages), kBytes = bytes(kStages);
};

template <typename T, int R, int M, bool BACK, bool SPLIT>
__global__ void __launch_bounds__(kLrThreads, SPLIT && R == 16 && sizeof(T) == 2 ? 3 : R <= 32 ? 2 : 1) lr_rows_kernel(const __grid_constant__ LrRowsArgs a) {
  using S = LrShape<T, M>;
  using L = LrSmem<T, R, M, BACK, SPLIT>;
  static_assert(SPLIT || M == 16, "tiles of 16 rows");
  constexpr bool F32 = sizeof(T) == 4, F16 = std::is_same<T, __half>::value, BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kStep = LrStep<T>::kStep, kEach = LrStep<T>::kEach;
  extern __shared__ __align__(16) unsigned char lr_dynamic[];
  __shared__ int rows[M];
  __shared__ float factors[M];
  __shared__ int scratch[kLrWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  unsigned char* behind = lr_dynamic + L::kRing;
  float* join = reinterpret_cast<float*>(lr_dynamic);
  float* part = reinterpret_cast<float*>(behind);
  T* hs = reinterpret_cast<T*>(behind + L::kPart);                   // first parts, then second parts
  const uint32_t rank = lr_rank(), ranks = lr_ranks();
  const LrTile tile = lr_tile<M>(a.groups, blockIdx.x / ranks, rows, scratch);
  if (tile.count == 0) return;                        // the whole cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool has = tile.group < a.groups.adapters;
  if (SPLIT && !has) return;
  const uint2 key = a.drop_x || a.drop_y ? philox_key(a.drop) : make_uint2(0, 0);

  const int all = (a.cols + 31) / 32;
  const int b0 = (int)((long long)all * rank / ranks), b1 = !SPLIT && a.y != nullptr ? (int)((long long)all * (rank + 1) / ranks) : b0;
  const int row_of[2] = {SPLIT ? -1 : rows[g], SPLIT ? -1 : rows[g + 8]};
  uint4* ahead = reinterpret_cast<uint4*>(behind + L::kPart + L::kH) + warp * L::kDepth * L::kPieces * 32 + lane;
  const bool fetched = !BACK && !SPLIT && a.base != nullptr && a.vec_y;
  auto request = [&](int i) {           // base of this warp's i-th step
    if constexpr (!BACK && !SPLIT) {
      const int b = b0 + warp + i * kLrWarps, col = b * 32 + 8 * t;
      if (fetched && b < b1 && col < a.cols) {
        uint4* to = ahead + i % L::kDepth * L::kPieces * 32;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int v = 0; v < (int)sizeof(T) / 2; ++v)
            if (row_of[h] >= 0) lr_copy16(to + (h * ((int)sizeof(T) / 2) + v) * 32, (const T*)a.base + row_of[h] * a.ld_base + col + v * (16 / (int)sizeof(T)));
      }
    }
  };

  if (has) {
    const T* w1 = (const T*)a.w1 + (long long)tile.group * a.k * a.rank;
    const int chunks = (a.k + S::kChunk - 1) / S::kChunk;
    const int c0 = (int)((long long)chunks * rank / ranks), c1 = (int)((long long)chunks * (rank + 1) / ranks);
    auto stage = [&](int i) { return reinterpret_cast<T*>(lr_dynamic + i * L::kStage); };
    // The eights that this thread copies of every chunk: their rows and columns stay the same.
    constexpr int kAcrossX = S::kChunk / 8, kX = M * kAcrossX / kLrThreads, kRowStep = kLrThreads / kAcrossX;
    constexpr int kAcrossW = BACK ? R / 8 : kAcrossX, kUnitsW = L::kRowsW * kAcrossW, kW = (kUnitsW + kLrThreads - 1) / kLrThreads, kStepW = kLrThreads / kAcrossW;
    static_assert(M * kAcrossX % kLrThreads == 0 && kLrThreads % kAcrossX == 0 && kLrThreads % kAcrossW == 0, "whole rows of threads");
    const int xr = threadIdx.x / kAcrossX, xc = threadIdx.x % kAcrossX * 8, wr = threadIdx.x / kAcrossW, wc = threadIdx.x % kAcrossW * 8;
    const T* from[kX];
    int from_row[kX];             // -1: none
#pragma unroll
    for (int i = 0; i < kX; ++i) {
      from_row[i] = rows[xr + i * kRowStep];
      from[i] = (const T*)a.x + (from_row[i] < 0 ? rows[0] : from_row[i]) * a.ldx + xc;        // rows behind the last: any, their results go nowhere
    }
    auto fetch = [&](int c, int slot) {
      T* xs = stage(slot);
      T* ws = xs + M * L::kPitchX;
      const int k0 = c * S::kChunk;
      if (a.vec_x && k0 + S::kChunk <= a.k) {
#pragma unroll
        for (int i = 0; i < kX; ++i)
#pragma unroll
          for (int v = 0; v < (int)sizeof(T) / 2; ++v)
            lr_copy16(xs + (xr + i * kRowStep) * L::kPitchX + xc + v * (16 / (int)sizeof(T)), from[i] + k0 + v * (16 / (int)sizeof(T)));
      } else {
#pragma unroll 1
        for (int i = 0; i < kX; ++i) lr_copy8<T>(xs + (xr + i * kRowStep) * L::kPitchX + xc, from[i] + k0, a.k - k0 - xc, a.vec_x, (const T*)a.x);
      }
      if (a.vec_w1 && a.rank == R && k0 + S::kChunk <= a.k) {
        const T* src = BACK ? w1 + (long long)(k0 + wr) * R + wc : w1 + (long long)wr * a.k + k0 + wc;
#pragma unroll
        for (int i = 0; i < kW; ++i) {
          const int r = wr + i * kStepW;
          if (kUnitsW % kLrThreads != 0 && r >= L::kRowsW) break;
#pragma unroll
          for (int v = 0; v < (int)sizeof(T) / 2; ++v)
            lr_copy16(ws + r * L::kPitchW + wc + v * (16 / (int)sizeof(T)), src + (BACK ? i * kStepW * R : (long long)i * kStepW * a.k) + v * (16 / (int)sizeof(T)));
        }
        return;
      }
#pragma unroll 1
      for (int i = 0; i < kW; ++i) {
        const int r = wr + i * kStepW;
        if (kUnitsW % kLrThreads != 0 && r >= L::kRowsW) break;
        if (BACK) lr_copy8<T>(ws + r * L::kPitchW + wc, w1 + (long long)(k0 + r) * a.rank + wc, k0 + r < a.k ? a.rank - wc : 0, a.vec_w1, w1);
        else lr_copy8<T>(ws + r * L::kPitchW + wc, w1 + (long long)r * a.k + k0 + wc, r < a.rank ? a.k - k0 - wc : 0, a.vec_w1, w1);
      }
    };
    float acc[R / 8][4];
#pragma unroll
    for (int j = 0; j < R / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
    const int m0 = warp % S::kM16 * 16, kp = warp / S::kM16 * S::kWarpK;
    for (int i = 0; i < L::kStages - 1; ++i) {
      if (c0 + i < c1) fetch(c0 + i, i);
      if (i == L::kStages - 2) {
#pragma unroll
        for (int d = 0; d < L::kDepth; ++d) request(d);
      }
      lr_commit();
    }
    int slot = 0;
    for (int c = c0; c < c1; ++c) {
      lr_wait<L::kStages - 2>();
      T* xs = stage(slot);
      if (a.drop_x) {
#pragma unroll
        for (int i = 0; i < kX; ++i)
          if (from_row[i] >= 0)
            lr_drop8<T>(xs + (xr + i * kRowStep) * L::kPitchX + xc, dropout_words((unsigned)(c * S::kChunk + xc) >> 3, from_row[i], key), a.drop.limit);
      }
      __syncthreads();
      if (c + L::kStages - 1 < c1) fetch(c + L::kStages - 1, slot == 0 ? L::kStages - 1 : slot - 1);
      lr_commit();
      const T* ws = xs + M * L::kPitchX;
      if constexpr (!F32) {
#pragma unroll
        for (int k = 0; k < S::kWarpK; k += 16) {
          uint32_t x[4];
          lr_ldm4(x, xs + (m0 + (lane & 15)) * L::kPitchX + kp + k + (lane >> 4) * 8);
#pragma unroll
          for (int j = 0; j < R / 16; ++j) {
            uint32_t w[4];
            if (BACK) lr_ldm4t(w, ws + (kp + k + (lane & 15)) * L::kPitchW + j * 16 + (lane >> 4) * 8);
            else lr_ldm4(w, ws + (j * 16 + (lane & 7) + (lane >> 4) * 8) * L::kPitchW + kp + k + (lane >> 3 & 1) * 8);
            lr_mma16<T>(acc[2 * j], x, w[0], w[1]);
            lr_mma16<T>(acc[2 * j + 1], x, w[2], w[3]);
          }
        }
      } else {
        float sum[R / 8][4];
#pragma unroll
        for (int j = 0; j < R / 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[j][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < S::kWarpK; k += 8) {
          uint32_t hi[4], lo[4];
          const float* xp = (const float*)xs + (m0 + g) * L::kPitchX + kp + k + t;
          lr_split(xp[0], hi[0], lo[0]);
          lr_split(xp[8 * L::kPitchX], hi[1], lo[1]);
          lr_split(xp[4], hi[2], lo[2]);
          lr_split(xp[8 * L::kPitchX + 4], hi[3], lo[3]);
#pragma unroll
          for (int j = 0; j < R / 8; ++j) {
            const float* wp = BACK ? (const float*)ws + (kp + k + t) * L::kPitchW + j * 8 + g : (const float*)ws + (j * 8 + g) * L::kPitchW + kp + k + t;
            uint32_t h0, l0, h1, l1;
            lr_split(wp[0], h0, l0);
            lr_split(wp[BACK ? 4 * L::kPitchW : 4], h1, l1);
            lr_mma8(sum[j], lo, h0, h1);
            lr_mma8(sum[j], hi, l0, l1);
            lr_mma8(sum[j], hi, h0, h1);
          }
        }
#pragma unroll
        for (int j = 0; j < R / 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[j][i] += sum[j][i];
      }
      slot = slot + 1 == L::kStages ? 0 : slot + 1;
    }
    lr_wait<0>();
    __syncthreads();                                   // the stages are read: the warps' parts go over them
    float* mine = join + (warp / S::kM16 * M + m0) * R;
#pragma unroll
    for (int j = 0; j < R / 8; ++j) {
      *reinterpret_cast<float2*>(mine + g * R + j * 8 + 2 * t) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * R + j * 8 + 2 * t) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    for (int u = threadIdx.x; u < M * R / 4; u += kLrThreads) {
      float4 v = reinterpret_cast<const float4*>(join)[u];
#pragma unroll
      for (int p = 1; p < S::kParts; ++p) {
        const float4 w = reinterpret_cast<const float4*>(join)[p * (M * R / 4) + u];
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
      reinterpret_cast<float4*>(part)[u] = v;
    }
    lr_arrive();
    lr_meet();
    const float by = (a.scales != nullptr ? a.scales[tile.group] : a.scale) * (a.drop_x || a.drop_y ? a.drop.share : 1.0f);
    constexpr int kUnits = M * R / 4, kLanes = R / 4;              // of a row: neighbouring lanes
#pragma unroll 1
    for (int u = threadIdx.x; u < kUnits; u += kLrThreads) {       // a multiple of 32: whole warps
      float4 v = lr_remote4(part + 4 * u, 0);
      for (uint32_t r = 1; r < ranks; ++r) {
        const float4 w = lr_remote4(part + 4 * u, r);
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
      const int row = u / kLanes, col = u % kLanes * 4;
      // behind the rank there is nothing, also beside an infinity, whose product with the zeros there is none
      float f[4] = {col < a.rank ? v.x * by : 0.0f, col + 1 < a.rank ? v.y * by : 0.0f, col + 2 < a.rank ? v.z * by : 0.0f, col + 3 < a.rank ? v.w * by : 0.0f};
      const bool keeps = a.kept.values != nullptr && rank == 0 && row < tile.count;
      const long long place = (long long)(tile.place + row) * R + col, second = (long long)a.groups.n * R;
      if (!BF16 && keeps) *reinterpret_cast<float4*>((float*)a.kept.values + place) = make_float4(f[0], f[1], f[2], f[3]);
      if constexpr (F16) {
        float top = fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3]))), down;
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float up = lr_power(top, down);
        if (col == 0) {
          factors[row] = up;
          if (keeps && a.kept.factors != nullptr) a.kept.factors[tile.place + row] = up;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] *= down;
      }
      if constexpr (F32) {
        if constexpr (!SPLIT) {
          uint4 hi, lo;
          lr_split(f[0], hi.x, lo.x);
          lr_split(f[1], hi.y, lo.y);
          lr_split(f[2], hi.z, lo.z);
          lr_split(f[3], hi.w, lo.w);
          *reinterpret_cast<uint4*>(hs + row * L::kPitchH + col) = hi;
          *reinterpret_cast<uint4*>(hs + (M + row) * L::kPitchH + col) = lo;
        }
      } else {
        __align__(8) T hi[4], lo[4];
        lr_parts<T>(f, hi, lo);
        if constexpr (!SPLIT) {
          *reinterpret_cast<uint2*>(hs + row * L::kPitchH + col) = *reinterpret_cast<const uint2*>(hi);
          *reinterpret_cast<uint2*>(hs + (M + row) * L::kPitchH + col) = *reinterpret_cast<const uint2*>(lo);
        }
        T* to = BF16 ? (T*)a.kept.values : (T*)a.kept.parts;
        if (keeps && to != nullptr) {
          *reinterpret_cast<uint2*>(to + place) = *reinterpret_cast<const uint2*>(hi);
          *reinterpret_cast<uint2*>(to + second + place) = *reinterpret_cast<const uint2*>(lo);
        }
      }
    }
    __syncwarp();
    lr_arrive();                                       // this block has read the others' parts; it leaves when they have read its own
    __syncthreads();
  } else {
#pragma unroll
    for (int d = 0; d < L::kDepth; ++d) request(d);
    lr_commit();
    lr_wait<0>();
  }

  if constexpr (!SPLIT) {              // y = base + s W2 h
    const LrFactor<T, BACK> w2((const T*)a.w2 + (has ? (long long)tile.group * a.cols * a.rank : 0), a.cols, a.rank, a.vec_w2, g, t);
    auto load_h = [&](int k, int part, uint32_t* h) {
      const T* p = hs + (part * M + g) * L::kPitchH + k + kEach * t;
      const uint2 u = *reinterpret_cast<const uint2*>(p), v = *reinterpret_cast<const uint2*>(p + 8 * L::kPitchH);
      h[0] = u.x; h[1] = v.x; h[2] = u.y; h[3] = v.y;
    };
    const float up[2] = {F16 && has ? factors[g] : 1.0f, F16 && has ? factors[g + 8] : 1.0f};
    constexpr bool kHold = R == 16;                                  // the rank values and the next factors stay in registers
    constexpr int kSteps = kHold ? R / kStep : 1;
    uint32_t held[kSteps][2][4], next[kSteps][4][2];
    int b = b0 + warp;
    if (kHold && has) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        load_h(k * kStep, 0, held[k][0]);
        load_h(k * kStep, 1, held[k][1]);
        if (b < b1) w2.load(b, k * kStep, next[k]);
      }
    }
    for (int i = 0; b < b1; b += kLrWarps, ++i) {
      const int col = b * 32 + 8 * t, left = a.cols - col;         // may be negative
      float acc[4][4], from[2][8];
      if (!BACK) lr_wait<L::kDepth - 1>();
      const uint4* here = ahead + i % L::kDepth * L::kPieces * 32;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int q = 0; q < 8; ++q) from[h][q] = 0.0f;
        if (!BACK && a.base != nullptr && row_of[h] >= 0 && left > 0) {
          if (a.vec_y) {
            __align__(16) T e[8];
#pragma unroll
            for (int q = 0; q < (int)sizeof(T) / 2; ++q) reinterpret_cast<uint4*>(e)[q] = here[(h * ((int)sizeof(T) / 2) + q) * 32];
            lr_load8<T, true>(e, 8, from[h]);
          } else {
            lr_load8<T, false>((const T*)a.base + row_of[h] * a.ld_base + col, left, from[h]);
          }
        }
        const float zeros[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        lr_set<T>(acc, h, LrStart<T>::kBase ? from[h] : zeros);
      }
      if (has) {
        if constexpr (kHold) {
          uint32_t w[kSteps][4][2];
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
#pragma unroll
            for (int j = 0; j < 4; ++j) { w[k][j][0] = next[k][j][0]; w[k][j][1] = next[k][j][1]; }
            if (b + kLrWarps < b1) w2.load(b + kLrWarps, k * kStep, next[k]);
          }
#pragma unroll
          for (int k = 0; k < kSteps; ++k) lr_multiply<T>(acc, held[k][0], held[k][1], w[k]);
        } else {
#pragma unroll 2
          for (int k = 0; k < R; k += kStep) {
            if (k >= a.rank) break;
            uint32_t w[4][2], hi[4], lo[4];
            w2.load(b, k, w);
            load_h(k, 0, hi);
            load_h(k, 1, lo);
            lr_multiply<T>(acc, hi, lo, w);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (row_of[h] < 0 || left <= 0) continue;
        float v[8];
        lr_get<T>(acc, h, up[h], from[h], v);
        if (BACK && a.drop_y && has) lr_drop(v, dropout_words((unsigned)col >> 3, row_of[h], key), a.drop.limit);
        if (tile.group > a.groups.adapters) {
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = __uint_as_float(0x7fc00000u);
        }
        T* p = (T*)a.y + row_of[h] * a.ldy + col;
        if (a.vec_y) lr_store8<T, true>(p, 8, v);
        else lr_store8<T, false>(p, left, v);
      }
      request(i + L::kDepth);
      if (!BACK) lr_commit();
    }
    lr_wait<0>();
  }
  __syncwarp();
  if (has) lr_meet();
}

// ---- the second product of many rows ---------------------------------------------------------------------------------------------------------
// y = base + s W2 h, h by place.  A warp takes 16 rows of one adapter and walks over blocks of columns, its own lanes' pieces of base two blocks ahead in shared
// memory; warps do not wait for one another.
template <typename T, int R, bool BACK> struct LrExpand {
  static constexpr int kGroups = sizeof(T) == 4 ? 2 : 4, kCols = 32 * kGroups;         // of a block of columns
  static constexpr int kStages = 2, kPieces = 8, kBytes = BACK ? 0 : kLrWarps * kStages * kPieces * 512;
  static constexpr bool kHold = R <= 32 || (R == 64 && sizeof(T) == 2);
  static constexpr int kWays = R == 64 ? 1 : 2;                                          // groups of factors in registers
  static_assert(kWays - 1 <= kGroups && kGroups % kWays == 0, "a block's groups take turns");
  static constexpr int kBlocks = R == 16 && sizeof(T) == 2 && !BACK ? 3 : 2;            // on an SM
};

template <typename T, int R, bool BACK>
__global__ void __launch_bounds__(kLrThreads, LrExpand<T, R, BACK>::kBlocks) lr_expand_kernel(const __grid_constant__ LrRowsArgs a, int tiles, int row_blocks, int per) {
  using X = LrExpand<T, R, BACK>;
  constexpr bool F32 = sizeof(T) == 4, F16 = std::is_same<T, __half>::value, BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kStep = LrStep<T>::kStep, kEach = LrStep<T>::kEach, kSize = (int)sizeof(T) / 2;
  extern __shared__ __align__(16) unsigned char lr_dynamic[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int index = blockIdx.x % row_blocks * kLrWarps + warp;
  if (index >= tiles) return;
  int group = 0, place = index * 16, count = a.groups.n - place < 16 ? a.groups.n - place : 16;
  int row_of[2] = {g < count ? place + g : -1, g + 8 < count ? place + g + 8 : -1};
  if (a.groups.mode == LR_PLAN) {
    const int4 tile = a.groups.tiles[index];
    row_of[0] = a.groups.tile_rows[index * 16ll + g];
    row_of[1] = a.groups.tile_rows[index * 16ll + g + 8];
    group = tile.x; place = tile.y; count = tile.z;
    if (group < 0) return;
  }
  const bool has = group < a.groups.adapters;
  const int blocks = (a.cols + X::kCols - 1) / X::kCols, c0 = blockIdx.x / row_blocks * per, c1 = c0 + per < blocks ? c0 + per : blocks;
  const bool fetched = !BACK && a.base != nullptr && a.vec_y, full = fetched && count == 16;
  const T* from[2] = {(const T*)a.base + (row_of[0] < 0 ? 0 : row_of[0]) * a.ld_base + 8 * t, (const T*)a.base + (row_of[1] < 0 ? 0 : row_of[1]) * a.ld_base + 8 * t};
  T* to[2] = {(T*)a.y + (row_of[0] < 0 ? 0 : row_of[0]) * a.ldy + 8 * t, (T*)a.y + (row_of[1] < 0 ? 0 : row_of[1]) * a.ldy + 8 * t};
  uint4* ring = reinterpret_cast<uint4*>(lr_dynamic) + warp * X::kStages * X::kPieces * 32 + lane;
  auto request = [&](int c, int stage) {
    if constexpr (!BACK) {
      if (full && c < c1 && (c + 1) * X::kCols <= a.cols) {
#pragma unroll
        for (int q = 0; q < X::kGroups; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int v = 0; v < kSize; ++v)
              lr_copy16(ring + ((stage * X::kGroups + q) * 2 * kSize + h * kSize + v) * 32, from[h] + c * X::kCols + q * 32 + v * (8 / kSize));
      } else if (fetched && c < c1) {
#pragma unroll 1
        for (int q = 0; q < X::kGroups; ++q)
          if (c * X::kCols + q * 32 + 8 * t < a.cols) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int v = 0; v < kSize; ++v)
                if (row_of[h] >= 0) lr_copy16(ring + ((stage * X::kGroups + q) * 2 * kSize + h * kSize + v) * 32, from[h] + c * X::kCols + q * 32 + v * (8 / kSize));
          }
      }
      lr_commit();
    }
  };
  request(c0, 0);
  request(c0 + 1, 1);
  const uint2 key = a.drop_y ? philox_key(a.drop) : make_uint2(0, 0);
  const LrFactor<T, BACK> w2((const T*)a.w2 + (has ? (long long)group * a.cols * a.rank : 0), a.cols, a.rank, a.vec_w2, g, t);
  // two parts of the rank values; rows behind the last have those of the first one, which go nowhere
  const long long at[2] = {(long long)(place + (g < count ? g : 0)) * R + kEach * t, (long long)(place + (g + 8 < count ? g + 8 : 0)) * R + kEach * t};
  auto load_h = [&](int k, uint32_t* hi, uint32_t* lo) {
    if constexpr (F32) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 f = *reinterpret_cast<const float2*>((const float*)a.kept.values + at[h] + k);
        lr_split(f.x, hi[h], lo[h]);
        lr_split(f.y, hi[2 + h], lo[2 + h]);
      }
    } else {
      const T* p = BF16 ? (const T*)a.kept.values : (const T*)a.kept.parts;
      const long long second = (long long)a.groups.n * R;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint2 u = *reinterpret_cast<const uint2*>(p + at[h] + k), v = *reinterpret_cast<const uint2*>(p + second + at[h] + k);
        hi[h] = u.x; hi[2 + h] = u.y;
        lo[h] = v.x; lo[2 + h] = v.y;
      }
    }
  };
  float up[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) up[h] = F16 && has ? a.kept.factors[place + (g + 8 * h < count ? g + 8 * h : 0)] : 1.0f;
  constexpr int kSteps = X::kHold ? R / kStep : 1;
  uint32_t held[kSteps][2][4];
  if (X::kHold && has) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) load_h(k * kStep, held[k][0], held[k][1]);
  }
  int c = c0, stage = 0;
  // Whole blocks: 16 rows, all columns and their factors in whole accesses, the rank known.  Nothing is checked, and the next factors are on their way.
  auto walk = [&](auto known) {
    constexpr int RANK = decltype(known)::value;
    const long long step = BACK ? 32 : 32 * RANK;
    const T* at = w2.p + c * X::kGroups * step;
    uint32_t w[X::kWays][kSteps][4][2];             // the factors of a group of columns and of the next ones
    const int last = c1 < a.cols / X::kCols ? c1 : a.cols / X::kCols;
    if (c >= last) return;
    auto ask = [&](int q) {                         // of the group at `at`
#pragma unroll
      for (int k = 0; k < kSteps; ++k) LrFactor<T, BACK>::template whole<RANK>(at + k * kStep * (BACK ? a.cols : 1), a.cols, k * kStep, g, t, w[q % X::kWays][k]);
      at += step;
    };
#pragma unroll
    for (int q = 0; q < X::kWays - 1; ++q) ask(q);  // a block has as many groups
    T* y[2] = {to[0] + c * X::kCols, to[1] + c * X::kCols};
    for (; c < last; ++c, stage ^= 1) {
      if (!BACK) lr_wait<1>();
      const uint4* here = ring + stage * X::kPieces * 32;
#pragma unroll
      for (int q = 0; q < X::kGroups; ++q) {
        float acc[4][4], base[2][8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int i = 0; i < 8; ++i) base[h][i] = 0.0f;
          if (!BACK) {
            __align__(16) T e[8];
#pragma unroll
            for (int i = 0; i < kSize; ++i) reinterpret_cast<uint4*>(e)[i] = here[(q * 2 * kSize + h * kSize + i) * 32];
            lr_load8<T, true>(e, 8, base[h]);
          }
          const float zeros[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
          lr_set<T>(acc, h, LrStart<T>::kBase ? base[h] : zeros);
        }
        if (q + X::kWays - 1 < X::kGroups || c + 1 < last) ask(q + X::kWays - 1);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) lr_multiply<T>(acc, held[k][0], held[k][1], w[q % X::kWays][k]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[8];
          lr_get<T>(acc, h, up[h], base[h], v);
          if (BACK && a.drop_y) lr_drop(v, dropout_words((unsigned)((c * X::kGroups + q) * 32 + 8 * t) >> 3, row_of[h], key), a.drop.limit);
          lr_store8<T, true>(y[h] + q * 32, 8, v);
        }
      }
      y[0] += X::kCols;
      y[1] += X::kCols;
      request(c + 2, stage);
    }
  };
  // The backward factors lie by rank value: 64 columns at a time, column 8 n + j for column n of the j-th of eight instructions, so that all of a thread's
  // 16 bytes of a rank value's row are its own; of a row it has 16 neighbouring results.  (32 columns as above use half of what they load: 52 us of
  // 8192 rows to 4096 values at rank 32.)
  auto walk_back = [&](auto known) {
    constexpr int RANK = decltype(known)::value;
    const int last = c1 < a.cols / X::kCols ? c1 : a.cols / X::kCols;
    if (c >= last) return;
    const T* at = (const T*)a.w2 + (long long)group * a.cols * a.rank + (long long)(4 * t) * a.cols + 8 * g + c * X::kCols;
    constexpr int kNext = kSteps <= 2 ? kSteps : 1;
    uint4 next[kNext][4];
    auto ask = [&](int k, uint4* v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = 16 * k + 4 * t < RANK ? *reinterpret_cast<const uint4*>(at + (long long)(16 * k + i) * a.cols) : make_uint4(0, 0, 0, 0);
    };
    if constexpr (kSteps <= 2) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) ask(k, next[k]);
    }
    T* y[2] = {to[0] + c * X::kCols + 8 * t, to[1] + c * X::kCols + 8 * t};       // 16 t: `to` has 8 t
    for (int b = 2 * c; b < 2 * last; ++b) {
      float acc[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
      auto multiply = [&](int k, const uint4* v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned half = j & 1 ? 0x7632u : 0x5410u;
          auto word = [&](int i) { return j < 2 ? v[i].x : j < 4 ? v[i].y : j < 6 ? v[i].z : v[i].w; };
          const uint32_t w0 = __byte_perm(word(0), word(1), half), w1 = __byte_perm(word(2), word(3), half);
          lr_mma16<T>(acc[j], held[k][1], w0, w1);
          lr_mma16<T>(acc[j], held[k][0], w0, w1);
        }
      };
      if constexpr (kSteps <= 2) {
        uint4 now[kNext][4];
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) now[k][i] = next[k][i];
        at += 64;
        if (b + 1 < 2 * last) {
#pragma unroll
          for (int k = 0; k < kSteps; ++k) ask(k, next[k]);
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k) multiply(k, now[k]);
      } else {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint4 now[4];
          ask(k, now);
          multiply(k, now);
        }
        at += 64;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = F16 ? acc[j][2 * h + i] * up[h] : acc[j][2 * h + i];
          if (a.drop_y) lr_drop(v, dropout_words((unsigned)(8 * b + 2 * t + i), row_of[h], key), a.drop.limit);
          lr_store8<T, true>(y[h] + 8 * i, 8, v);
        }
      y[0] += 64;
      y[1] += 64;
    }
    c = last;
  };
  if constexpr (X::kHold) {
    if (has && count == 16 && a.vec_y && a.vec_w2 && (BACK || a.base != nullptr)) {
      if constexpr (BACK && !F32) {
        if (a.rank == R) walk_back(std::integral_constant<int, R>());
        else if (R == 16 && a.rank == 8) walk_back(std::integral_constant<int, 8>());
      } else {
        if (a.rank == R) walk(std::integral_constant<int, R>());
        else if (R == 16 && a.rank == 8) walk(std::integral_constant<int, 8>());
      }
    }
  }
  for (; c < c1; ++c, stage ^= 1) {                 // anything else
    if (!BACK) lr_wait<1>();
#pragma unroll 1
    for (int q = 0; q < X::kGroups; ++q) {
      const int b = c * X::kGroups + q, left = a.cols - b * 32 - 8 * t;         // may be negative
      float acc[4][4], base[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 8; ++i) base[h][i] = 0.0f;
        if (!BACK && a.base != nullptr && row_of[h] >= 0 && left > 0) {
          if (a.vec_y) {
            __align__(16) T e[8];
#pragma unroll
            for (int i = 0; i < kSize; ++i) reinterpret_cast<uint4*>(e)[i] = ring[((stage * X::kGroups + q) * 2 * kSize + h * kSize + i) * 32];
            lr_load8<T, true>(e, 8, base[h]);
          } else {
            lr_load8<T, false>(from[h] + b * 32, left, base[h]);
          }
        }
        const float zeros[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        lr_set<T>(acc, h, LrStart<T>::kBase ? base[h] : zeros);
      }
      if (has) {
        if constexpr (X::kHold) {
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            uint32_t w[4][2];
            w2.load(b, k * kStep, w);
            lr_multiply<T>(acc, held[k][0], held[k][1], w);
          }
        } else {
#pragma unroll 2
          for (int k = 0; k < R; k += kStep) {
            if (k >= a.rank) break;
            uint32_t w[4][2], hi[4], lo[4];
            w2.load(b, k, w);
            load_h(k, hi, lo);
            lr_multiply<T>(acc, hi, lo, w);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (row_of[h] < 0 || left <= 0) continue;
        float v[8];
        lr_get<T>(acc, h, up[h], base[h], v);
        if (BACK && a.drop_y && has) lr_drop(v, dropout_words((unsigned)(b * 32 + 8 * t) >> 3, row_of[h], key), a.drop.limit);
        if (group > a.groups.adapters) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(0x7fc00000u);
        }
        if (a.vec_y) lr_store8<T, true>(to[h] + b * 32, 8, v);
        else lr_store8<T, false>(to[h] + b * 32, left, v);
      }
    }
    request(c + 2, stage);
  }
  if (!BACK) lr_wait<0>();
}

// ---- the factors' gradients --------------------------------------------------------------------------------------------------------------
// out[r][c] (or [c][r]) = sum over the adapter's rows of p[row][r] q[row][c]; the rank values p have the scales in them.  A cluster takes 128 columns of one adapter and one product, its blocks
// split the rows.  bf16: the rank values' two parts times q, both as ldmatrix turns them.  f16 and f32: TF32, where f16 is exact (its range would lose small rank
// values); the two rows 2 t and 2 t + 1 of every eight are then what a thread has of a matrix instruction's axis of eight, which is how
// ldmatrix hands out 16-bit values of q; p follows.
template <typename T, int R> struct LrOuterSmem {
  static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  static constexpr int kPitchQ = kLrOuterCols + (sizeof(T) == 4 ? 4 : 8), kPitchP = kBf16 ? R + 8 : R + 4;
  static constexpr int kSizeP = kBf16 ? 2 : 4, kP = kLrOuterRows * kPitchP * kSizeP;            // one part
  static constexpr int kStage = kLrOuterRows * kPitchQ * (int)sizeof(T) + 2 * kP;
  static constexpr int kSum = R * kLrOuterCols * 4;
  static constexpr int kStages = 3 * kStage <= kLrSmemMost ? 3 : 2;
  static constexpr int kBytes = kStages * kStage > kSum ? kStages * kStage : kSum;
  static_assert(kBytes <= kLrSmemMost, "shared memory");
};

template <typename T, int R>
__global__ void __launch_bounds__(kLrThreads, R <= 32 ? 3 : 1) lr_outer_kernel(const __grid_constant__ LrOuterArgs a) {
  using L = LrOuterSmem<T, R>;
  constexpr bool F32 = sizeof(T) == 4, BF16 = L::kBf16;
  extern __shared__ __align__(16) unsigned char lr_dynamic[];
  __shared__ int rows[4][kLrOuterRows];
  __shared__ long long places[4][kLrOuterRows];          // of the rows in q
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t rank = lr_rank(), ranks = lr_ranks();
  const int cluster = blockIdx.x / ranks, per = a.blocks[0] + a.blocks[1], adapter = cluster / per, within = cluster % per;
  const int which = within < a.blocks[0] ? 0 : 1, width = a.width[which], col0 = (within - (which ? a.blocks[0] : 0)) * kLrOuterCols;
  int first = 0, last = a.groups.n;
  if (a.groups.mode == LR_PLAN) { first = a.groups.start[adapter]; last = a.groups.start[adapter + 1]; }
  const int steps = (last - first + kLrOuterRows - 1) / kLrOuterRows;
  const int s0 = (int)((long long)steps * rank / ranks), s1 = (int)((long long)steps * (rank + 1) / ranks);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const T* q = (const T*)a.q[which];
  const bool drop = which == 0 && a.drop_x, inside = a.vec[which] && col0 + kLrOuterCols <= width;
  const uint2 key = drop ? philox_key(a.drop) : make_uint2(0, 0);
  auto list = [&](int s) {          // row numbers of a step, four steps side by side
    if (threadIdx.x < kLrOuterRows) {
      const int place = first + s * kLrOuterRows + threadIdx.x;
      const int row = place < last ? (a.groups.mode == LR_PLAN ? a.groups.order[place] : place) : -1;
      rows[s % 4][threadIdx.x] = row;
      places[s % 4][threadIdx.x] = (row < 0 ? 0 : row) * a.ldq[which];
    }
  };
  auto qs = [&](int i) { return reinterpret_cast<T*>(lr_dynamic + i * L::kStage); };
  auto ps = [&](int i) { return lr_dynamic + i * L::kStage + kLrOuterRows * L::kPitchQ * sizeof(T); };
  auto fetch = [&](int s, int slot) {
    const int from = first + s * kLrOuterRows;
    constexpr int kAcross = kLrOuterCols / 8, kRows = kLrThreads / kAcross;
    const int r0 = threadIdx.x / kAcross, c0 = threadIdx.x % kAcross * 8;
    T* to = qs(slot) + r0 * L::kPitchQ + c0;
    if (inside && from + kLrOuterRows <= last) {
#pragma unroll
      for (int r = 0; r < kLrOuterRows; r += kRows) {
        const T* src = q + places[s % 4][r0 + r] + col0 + c0;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) lr_copy16(to + r * L::kPitchQ + i * (16 / sizeof(T)), src + i * (16 / sizeof(T)));
      }
    } else {
#pragma unroll 1
      for (int r = 0; r < kLrOuterRows; r += kRows)
        lr_copy8<T>(to + r * L::kPitchQ, q + places[s % 4][r0 + r] + col0 + c0, from + r0 + r < last ? width - col0 - c0 : 0, a.vec[which], q);
    }
    // rank values: eights of the rows side by side, of bf16 both parts
    using P = typename std::conditional<BF16, T, float>::type;
    constexpr int kOne = kLrOuterRows * (R / 8), kAll = BF16 ? 2 * kOne : kOne;
    const P* p = (const P*)a.p[which] + (long long)from * R;
#pragma unroll
    for (int u0 = 0; u0 < kAll; u0 += kLrThreads) {
      const int u = u0 + threadIdx.x;
      if (kAll % kLrThreads != 0 && u >= kAll) break;
      const int part = u / kOne, r = u % kOne / (R / 8), c = u % (R / 8) * 8;
      const P* src = p + part * (long long)a.groups.n * R + r * R + c;
      lr_copy8<P>((P*)(ps(slot) + part * L::kP) + r * L::kPitchP + c, src, from + r < last ? 8 : 0, true, (const P*)a.p[which]);
    }
  };
  float acc[R / 16][2][4];
#pragma unroll
  for (int i = 0; i < R / 16; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][j][k] = 0.0f;
  // a ring of stages that is full but for the one that is multiplied; the rows of the step behind it are listed meanwhile
  constexpr int kAhead = L::kStages - 1;
  for (int s = s0; s <= s0 + kAhead && s < s1; ++s) list(s);
  __syncthreads();
  for (int s = s0; s < s0 + kAhead; ++s) {
    if (s < s1) fetch(s, s - s0);
    lr_commit();
  }
  int slot = 0;
  for (int s = s0; s < s1; ++s, slot = slot == kAhead ? 0 : slot + 1) {
    lr_wait<kAhead - 1>();
    if (drop) {                     // the eights that this thread copied
      const int* list = rows[s % 4];
#pragma unroll 2
      for (int u = threadIdx.x; u < kLrOuterRows * (kLrOuterCols / 8); u += kLrThreads) {
        const int r = u / (kLrOuterCols / 8), c = u % (kLrOuterCols / 8) * 8;
        if (list[r] >= 0) lr_drop8<T>(qs(slot) + r * L::kPitchQ + c, dropout_words((unsigned)(col0 + c) >> 3, list[r], key), a.drop.limit);
      }
    }
    if constexpr (!BF16) {          // and its rank values into two parts
      for (int u = threadIdx.x; u < kLrOuterRows * (R / 8); u += kLrThreads) {
        uint4* hi = reinterpret_cast<uint4*>(ps(slot) + (u / (R / 8) * L::kPitchP + u % (R / 8) * 8) * 4);
        uint4* lo = reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(hi) + L::kP);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 f = reinterpret_cast<const float4*>(hi)[h];
          uint4 x, y;
          lr_split(f.x, x.x, y.x);
          lr_split(f.y, x.y, y.y);
          lr_split(f.z, x.z, y.z);
          lr_split(f.w, x.w, y.w);
          hi[h] = x;
          lo[h] = y;
        }
      }
    }
    __syncthreads();
    if (s + kAhead < s1) fetch(s + kAhead, slot == 0 ? kAhead : slot - 1);
    lr_commit();
    if (s + kAhead + 1 < s1) list(s + kAhead + 1);
    const T* qp = qs(slot) + warp * 16;
    if constexpr (BF16) {
      const T* pp = (const T*)ps(slot);
#pragma unroll
      for (int k = 0; k < kLrOuterRows; k += 16) {
        uint32_t w[4];
        lr_ldm4t(w, qp + (k + (lane & 15)) * L::kPitchQ + (lane >> 4) * 8);
#pragma unroll
        for (int i = 0; i < R / 16; ++i) {
          uint32_t hi[4], lo[4];
          const T* p = pp + (k + (lane & 7) + (lane >> 4) * 8) * L::kPitchP + i * 16 + (lane >> 3 & 1) * 8;
          lr_ldm4t(lo, p + L::kP / 2);
          lr_ldm4t(hi, p);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            lr_mma16<T>(acc[i][j], lo, w[2 * j], w[2 * j + 1]);
            lr_mma16<T>(acc[i][j], hi, w[2 * j], w[2 * j + 1]);
          }
        }
      }
    } else {
      const uint32_t* pp = (const uint32_t*)ps(slot);
      float sum[R / 16][2][4];
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < R / 16; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[i][j][k] = 0.0f;
      }
#pragma unroll
      for (int k = 0; k < kLrOuterRows; k += 16) {
        float v[2][2][2];             // of the first and the second eight rows: product j, rows 2 t and 2 t + 1
        if constexpr (F32) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int i = 0; i < 2; ++i) v[h][j][i] = ((const float*)qp)[(k + 8 * h + 2 * t + i) * L::kPitchQ + j * 8 + g];
        } else {
          uint32_t w[4];
          lr_ldm4t(w, qp + (k + (lane & 15)) * L::kPitchQ + (lane >> 4) * 8);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2 f = lr_pair<T>(w[2 * j + h]);
              v[h][j][0] = f.x; v[h][j][1] = f.y;
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t vh[2][2], vl[2][2];
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if constexpr (F32) lr_split(v[h][j][i], vh[j][i], vl[j][i]);
              else vh[j][i] = __float_as_uint(v[h][j][i]);
            }
#pragma unroll
          for (int i = 0; i < R / 16; ++i) {
            const uint32_t* p = pp + (k + 8 * h + 2 * t) * L::kPitchP + i * 16 + g;
            const uint32_t hi[4] = {p[0], p[8], p[L::kPitchP], p[L::kPitchP + 8]};
            p += L::kP / 4;
            const uint32_t lo[4] = {p[0], p[8], p[L::kPitchP], p[L::kPitchP + 8]};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float* d = F32 ? sum[i][j] : acc[i][j];
              lr_mma8(d, lo, vh[j][0], vh[j][1]);
              if constexpr (F32) lr_mma8(d, hi, vl[j][0], vl[j][1]);
              lr_mma8(d, hi, vh[j][0], vh[j][1]);
            }
          }
        }
      }
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < R / 16; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[i][j][k] += sum[i][j][k];
      }
    }
  }
  lr_wait<0>();
  __syncthreads();
  float* part = reinterpret_cast<float*>(lr_dynamic);            // [R][128]
#pragma unroll
  for (int i = 0; i < R / 16; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float* p = part + (i * 16 + g) * kLrOuterCols + warp * 16 + j * 8 + 2 * t;
      *reinterpret_cast<float2*>(p) = make_float2(acc[i][j][0], acc[i][j][1]);
      *reinterpret_cast<float2*>(p + 8 * kLrOuterCols) = make_float2(acc[i][j][2], acc[i][j][3]);
    }
  lr_arrive();
  lr_meet();
  T* out = (T*)a.out[which] + (long long)adapter * a.rank * width;
  // each block adds and writes its share of the tile: along the rank for dB, whose rank values lie side by side
  for (int u = threadIdx.x + rank * kLrThreads; u < R * kLrOuterCols / 4; u += kLrThreads * ranks) {
    const int r = u / (kLrOuterCols / 4), c = u % (kLrOuterCols / 4) * 4;
    if (r >= a.rank || col0 + c >= width) continue;
    float4 v = lr_remote4(part + 4 * u, 0);
    for (uint32_t k = 1; k < ranks; ++k) {
      const float4 w = lr_remote4(part + 4 * u, k);
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col0 + c + i < width) out[which ? (long long)(col0 + c + i) * a.rank + r : (long long)r * width + col0 + c + i] = lr_round<T>(f[i]);
  }
  __syncwarp();
  lr_arrive();
  lr_meet();
}

// ---- launches ------------------------------------------------------------------------------------------------------------------------------
template <typename Kern, typename... Args>
static cudaError_t lr_launch(Kern kernel, long long clusters, int ranks, int smem, cudaStream_t st, const Args&... args) {
  if (clusters * ranks >= 1ll << 31) return cudaErrorInvalidValue;
  if (smem > 48 * 1024) {          // once for each kernel and device: it costs the host a microsecond
    static std::mutex guard;
    static std::map<std::pair<const void*, int>, int> allowed;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> hold(guard);
    int& have = allowed[{(const void*)kernel, device}];
    if (have < smem) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
      have = smem;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * ranks));
  cfg.blockDim = dim3(kLrThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Blocks of a cluster that divide `units` of work among them: what ends first where `resident` blocks run at once and a block's start and end cost as
// much as `ends` units.
inline int lr_ranks_for(long long clusters, long long units, int resident, int ends) {
  int best = 1;
  double least = 1e300;
  for (int r = 1; r <= 8 && r <= units; ++r) {
    const double cost = (double)((clusters * r + resident - 1) / resident) * ((double)units / r + ends);
    if (cost < least * 0.999) { least = cost; best = r; }
  }
  return best;
}
// Tiles of M rows, the empty ones among them.
inline long long lr_slots(const LrGroups& g, int M) { return g.mode == LR_ONE ? (g.n + M - 1) / M : g.mode == LR_SELF ? g.n : g.n / M + g.adapters + 2; }

template <typename T, int R, int M, bool BACK, bool SPLIT>
static cudaError_t lr_rows_as(const LrRowsArgs& a, cudaStream_t st) {
  using L = LrSmem<T, R, M, BACK, SPLIT>;
  static_assert(L::kBytes <= kLrSmemMost, "shared memory");
  const LrGroups& g = a.groups;
  const long long slots = lr_slots(g, M), busy = g.mode == LR_ONE ? slots : g.n / M + (g.n < g.adapters ? g.n : g.adapters);
  const int chunks = (a.k + L::kChunk - 1) / L::kChunk;
  const int resident = 148 * (SPLIT && R == 16 && sizeof(T) == 2 ? 3 : R <= 32 ? 2 : 1);
  return lr_launch(lr_rows_kernel<T, R, M, BACK, SPLIT>, slots, lr_ranks_for(busy < 1 ? 1 : busy, chunks, resident, 4), L::kBytes, st, a);
}

template <typename T, int R, bool BACK>
static cudaError_t lr_expand_as(const LrRowsArgs& a, cudaStream_t st) {
  using X = LrExpand<T, R, BACK>;
  const int tiles = (int)lr_slots(a.groups, 16), row_blocks = (tiles + kLrWarps - 1) / kLrWarps, blocks = (a.cols + X::kCols - 1) / X::kCols;
  // blocks of columns for a block: what leaves the last wave fullest, where a block's start costs about as much as one of them
  const int resident = 148 * X::kBlocks;
  int per = 1;
  double least = 1e30;
  for (int p = 1; p <= 16 && p <= blocks; ++p) {
    const long long grid = (long long)row_blocks * ((blocks + p - 1) / p);
    const double cost = (double)((grid + resident - 1) / resident) * (p + 1);
    if (cost < least) { least = cost; per = p; }
  }
  const long long grid = (long long)row_blocks * ((blocks + per - 1) / per);
  return lr_launch(lr_expand_kernel<T, R, BACK>, grid, 1, X::kBytes, st, a, tiles, row_blocks, per);
}

template <typename T, int R, bool BACK>
static cudaError_t lr_rows_r(const LrRowsArgs& a, cudaStream_t st) {
  const LrGroups& g = a.groups;
  if (!a.split) return lr_rows_as<T, R, 16, BACK, false>(a, st);
  // Tiles of 64 rows where adapters fill them; 16 rows keep more clusters busy and waste less of the tiles
  cudaError_t e;
  if (g.n / g.adapters >= 48) e = lr_rows_as<T, R, 64, BACK, true>(a, st);
  else e = lr_rows_as<T, R, 16, BACK, true>(a, st);
  return e == cudaSuccess && a.y != nullptr ? lr_expand_as<T, R, BACK>(a, st) : e;
}

template <typename T, int R>
static cudaError_t lr_outer_r(const LrOuterArgs& a, cudaStream_t st) {
  using L = LrOuterSmem<T, R>;
  const long long clusters = (long long)(a.blocks[0] + a.blocks[1]) * a.groups.adapters;
  const long long steps = (a.groups.n / a.groups.adapters + kLrOuterRows - 1) / kLrOuterRows;
  // How the rows are split goes by both products, wanted or not: a gradient has the same bits alone and beside the other.  Columns that are dropped take twice
  // the others' time: many short blocks then even out.
  const long long both = ((a.width[0] + kLrOuterCols - 1) / kLrOuterCols + (a.width[1] + kLrOuterCols - 1) / kLrOuterCols) * (long long)a.groups.adapters;
  const int ranks = a.drop_x && steps >= 32 ? 8 : lr_ranks_for(both, steps, 148 * (R <= 32 ? (L::kBytes <= kLrSmemThird ? 3 : 2) : 1), 4);
  return lr_launch(lr_outer_kernel<T, R>, clusters, ranks, L::kBytes, st, a);
}

inline int lr_padded(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

// Instances by type, each in a file of its own.
template <typename T> cudaError_t lr_rows(const LrRowsArgs& a, bool back, cudaStream_t st);
template <typename T> cudaError_t lr_outer(const LrOuterArgs& a, cudaStream_t st);

template <typename T>
cudaError_t lr_rows_of(const LrRowsArgs& a, bool back, cudaStream_t st) {
  switch (lr_padded(a.rank)) {
    case 16: return back ? lr_rows_r<T, 16, true>(a, st) : lr_rows_r<T, 16, false>(a, st);
    case 32: return back ? lr_rows_r<T, 32, true>(a, st) : lr_rows_r<T, 32, false>(a, st);
    case 64: return back ? lr_rows_r<T, 64, true>(a, st) : lr_rows_r<T, 64, false>(a, st);
    default: return back ? lr_rows_r<T, 128, true>(a, st) : lr_rows_r<T, 128, false>(a, st);
  }
}
template <typename T>
cudaError_t lr_outer_of(const LrOuterArgs& a, cudaStream_t st) {
  switch (lr_padded(a.rank)) {
    case 16: return lr_outer_r<T, 16>(a, st);
    case 32: return lr_outer_r<T, 32>(a, st);
    case 64: return lr_outer_r<T, 64>(a, st);
    default: return lr_outer_r<T, 128>(a, st);
  }
}

}  // namespace bonsai
