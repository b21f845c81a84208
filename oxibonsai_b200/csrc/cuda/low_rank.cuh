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
// from shared memory; tcgen05 would want tiles of 128 rows of one adapter and does not pay at a few operations a byte.  The long product of 16-bit types
// multiplies them as they are.  The rank values are kept in parts, so that nothing is rounded to 16 bits between the products: three bf16
// parts hold the 24 bits of f32 (two would hold 16: one result in 256 then rounds to the other neighbour than f32's); two f16 parts 22, over a power of two for each
// row in the second product, since f16's range would lose small gradients; f16 in the sums over rows and f32 everywhere have two TF32 parts, 22 bits (f16 itself
// is exact in TF32).  f32 operands are two TF32 parts too, three products of them.  Matrix instructions cut their sums off instead of rounding them: the long
// product and the sums over rows start from zero for each 16 to 64 terms and are added to f32 registers (8192 rows, bf16: one value in 4000 of the factors'
// gradients is not the exact one rounded, one in 800 of f32 products by a library).
//
// Measured on one B200, rank 16, bf16, in a graph (copy rate 6.54 TB/s): 1 row 4096 to 4096 6.3 us, 64 rows over 48 adapters 4096 to 12288 15 us (f16); 8192 rows 4096 to
// 12288 without dropout 96 us forward (470 MB: 4.9 TB/s), 82 us for dx (268 MB), 68 us for both factors' gradients (270 MB: 4.0 TB/s); dropout adds 15, 5 and 21.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "philox.cuh"

namespace bonsai {

constexpr int kLrThreads = 256, kLrWarps = 8, kLrSelf = 256;      // kLrSelf: rows that blocks group by themselves
// From so many rows and results on the two products are kernels of their own: each is then a stream over memory with as many blocks as it likes.  Forward, us in
// one kernel and in two, of rows with 4096 values:
//                  1100 to 4096   2000 to 4096   4000 to 4096   2000 to 12288   8000 to 4096
//   bf16 rank 16      12    16       17    20       32    34       37    32        66    48
//   f16 rank 16       13    16       17    20       33    34       38    32        66    49
//   bf16 rank 64      22    31       38    37       74    51       82    66       136    91
//   bf16 rank 128     42    64       76    72      157   133      199   174       287   252
//   f32 rank 16       27    33       45    42       85    78       86    80       162   143
//   f32 rank 128     129   162      260   203      520   391      559   404       904   767
// The border, 2^24 results, is that of 16-bit types at rank 16; larger ranks and f32 would have theirs at 2^23.
constexpr int kLrSplit = 1024;
inline bool lr_split_at(int n, int cols) { return n >= kLrSplit && (long long)n * cols >= 1 << 24; }
// dynamic shared memory of a block, of each of two or three on an SM
constexpr int kLrSmemMost = 227 * 1024 - 2048, kLrSmemHalf = 112 * 1024, kLrSmemThird = 74 * 1024;
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

// The rank values of a forward or a backward pass, times the adapter's scale, by place in the order: f32 [n][R] (R: the padded rank), of bf16 three parts
// [3][n][R].  f16 for the second product: two parts over a power of two for each row, and that power.
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

// Parts of a rank value in the products.
template <typename T> struct LrParts {
  static constexpr int kCount = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
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
__device__ __forceinline__ void lr_copy4(void* dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(lr_smem(dst)), "l"(src), "r"(there ? 4 : 0) : "memory");
}
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

// Rows at odd addresses into shared memory: C columns of rows r < ROWS from `from(r)` (null: zeros), `left` of them there (`any`: an address that is).  A warp takes
// a row at a time, so that neighbouring lanes take neighbouring values; only those of f32 are wide enough for cp.async.  8000 rows 4095 to 4097 values, bf16, rank 16:
// with eights to a thread 286 us forward and 348 backward, with this and the rows of lr_expand_kernel 183 and 244, calls timed one behind another; in a graph 156 and 229 (of
// 4096 values 48 and 92).
template <typename T, int ROWS, int C, typename From>
__device__ __forceinline__ void lr_copy_rows(T* to, int pitch, int left, const T* any, From from) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll 2
  for (int r = warp; r < ROWS; r += kLrWarps) {
    const T* src = from(r);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < C / 32; ++i) {
        const bool there = src != nullptr && i * 32 + lane < left;
        lr_copy4(to + r * pitch + i * 32 + lane, there ? src + i * 32 + lane : any, there);
      }
    } else {
      T v[C / 32];
#pragma unroll
      for (int i = 0; i < C / 32; ++i) v[i] = src != nullptr && i * 32 + lane < left ? src[i * 32 + lane] : lr_round<T>(0.0f);
#pragma unroll
      for (int i = 0; i < C / 32; ++i) to[r * pitch + i * 32 + lane] = v[i];
    }
  }
}

// ---- the kernels' launches ----------------------------------------------------------------------------------------------------------------
inline int lr_padded(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

// Instances by type, each in a file of its own.
template <typename T> cudaError_t lr_rows(const LrRowsArgs& a, bool back, cudaStream_t st);
template <typename T> cudaError_t lr_outer(const LrOuterArgs& a, cudaStream_t st);

}  // namespace bonsai
