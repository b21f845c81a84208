// The two products of the rows of a low-rank update (low_rank.cuh has the formulas): in one kernel for few rows, in two for many.
#pragma once
#include "low_rank.cuh"

namespace bonsai {

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

// acc += the rank values of 16 rows (their parts, the largest first) times the factors of 32 columns
template <typename T>
__device__ __forceinline__ void lr_multiply(float (*acc)[4], const uint32_t (*h)[4], const uint32_t (*w)[2]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      uint32_t h0, l0, h1, l1;
      lr_split(__uint_as_float(w[j][0]), h0, l0);
      lr_split(__uint_as_float(w[j][1]), h1, l1);
      lr_mma8(acc[j], h[1], h0, h1);
      lr_mma8(acc[j], h[0], l0, l1);
      lr_mma8(acc[j], h[0], h0, h1);
    } else {
#pragma unroll
      for (int p = LrParts<T>::kCount - 1; p >= 0; --p) lr_mma16<T>(acc[j], h[p], w[j][0], w[j][1]);
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
// `has`: the row has an adapter; without one it is base as it is, where an addition of zeros would lose the sign of -0
template <typename T>
__device__ __forceinline__ void lr_get(float (*acc)[4], int h, float up, const float* base, bool has, float* v) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float d = acc[q >> 1][2 * h + (q & 1)];
    v[q] = LrStart<T>::kBase ? d : !has ? base[q] : std::is_same<T, __half>::value ? fmaf(d, up, base[q]) : d + base[q];
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
__device__ __forceinline__ void lr_parts(const float* f, T (*part)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float left = f[i];
#pragma unroll
    for (int p = 0; p < LrParts<T>::kCount; ++p) {
      part[p][i] = lr_round<T>(left);
      const float h = lr_float<T>(part[p][i]);
      left = fabsf(h) <= 3.4028234e38f ? left - h : 0.0f;          // an infinity has no other parts
    }
  }
}

// ---- the rows ------------------------------------------------------------------------------------------------------------------------------
template <typename T, int M> struct LrShape {
  static constexpr int kM16 = M / 16, kParts = kLrWarps / kM16;       // warps over rows, and over the long axis
  static constexpr int kChunk = M == 64 && sizeof(T) == 4 ? 64 : 128, kWarpK = kChunk / kParts;
};

// SPLIT: the rank values are all that is made.  Else they wait for the second product in their parts, each of the inputs' 16-bit type (f16 over a power of two
// for each row, so that neither large nor small ones are lost) or TF32, and tiles have 16 rows.
template <typename T, int R, int M, bool BACK, bool SPLIT> struct LrSmem {
  static constexpr int kPad = 16 / sizeof(T);
  static constexpr int kChunk = LrShape<T, M>::kChunk;
  static constexpr int kPitchX = kChunk + kPad, kPitchW = BACK ? R + 8 : kChunk + kPad, kRowsW = BACK ? kChunk : R;
  static constexpr int kStage = (M * kPitchX + kRowsW * kPitchW) * (int)sizeof(T);
  static constexpr int kJoin = LrShape<T, M>::kParts * M * R * 4;         // the warps' parts, over the stages
  static constexpr int kPart = M * R * 4, kPitchH = R + 8, kH = SPLIT ? 0 : LrParts<T>::kCount * M * kPitchH * (int)sizeof(T);
  // what of base is on its way: each lane's own 16 bytes, `kDepth` steps of a warp
  static constexpr int kDepth = sizeof(T) == 4 ? 2 : 4, kPieces = (int)sizeof(T);
  static constexpr int kBase = BACK || SPLIT ? 0 : kLrWarps * kDepth * kPieces * 512;
  static constexpr int kBlocks = SPLIT && R == 16 && sizeof(T) == 2 ? 3 : R <= 32 || (R == 64 && sizeof(T) == 2) ? 2 : 1;      // on an SM
  static constexpr int kMost = kBlocks == 3 ? kLrSmemThird : kBlocks == 2 ? kLrSmemHalf : kLrSmemMost;
  static constexpr int ring(int stages) { return stages * kStage > kJoin ? stages * kStage : kJoin; }
  static constexpr int bytes(int stages) { return ring(stages) + kPart + kH + kBase; }
  // as many stages as leave room for these blocks
  static constexpr int kStages = bytes(4) <= kMost ? 4 : bytes(3) <= kMost ? 3 : 2, kRing = ring(kStages), kBytes = bytes(kStages);
};

template <typename T, int R, int M, bool BACK, bool SPLIT>
__global__ void __launch_bounds__(kLrThreads, LrSmem<T, R, M, BACK, SPLIT>::kBlocks) lr_rows_kernel(const __grid_constant__ LrRowsArgs a) {
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
  T* hs = reinterpret_cast<T*>(behind + L::kPart);                   // first parts, then second ones, then third ones
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
      } else if (a.vec_x) {
#pragma unroll
        for (int i = 0; i < kX; ++i) lr_copy8<T>(xs + (xr + i * kRowStep) * L::kPitchX + xc, from[i] + k0, a.k - k0 - xc, true, (const T*)a.x);
      } else {
        lr_copy_rows<T, M, S::kChunk>(xs, L::kPitchX, a.k - k0, (const T*)a.x, [&](int r) { return rows[r] < 0 ? (const T*)nullptr : (const T*)a.x + rows[r] * a.ldx + k0; });
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
      if (!BACK && !a.vec_w1) {
        lr_copy_rows<T, R, S::kChunk>(ws, L::kPitchW, a.k - k0, w1, [&](int r) { return r < a.rank ? w1 + (long long)r * a.k + k0 : (const T*)nullptr; });
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
        if (!a.vec_x) __syncthreads();                 // others have copied this thread's eights
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
        uint32_t x[S::kWarpK / 16][4];
#pragma unroll
        for (int k = 0; k < S::kWarpK; k += 16) lr_ldm4(x[k / 16], xs + (m0 + (lane & 15)) * L::kPitchX + kp + k + (lane >> 4) * 8);
#pragma unroll
        for (int j = 0; j < R / 16; ++j) {
          float sum[2][4] = {};
#pragma unroll
          for (int k = 0; k < S::kWarpK; k += 16) {
            uint32_t w[4];
            if (BACK) lr_ldm4t(w, ws + (kp + k + (lane & 15)) * L::kPitchW + j * 16 + (lane >> 4) * 8);
            else lr_ldm4(w, ws + (j * 16 + (lane & 7) + (lane >> 4) * 8) * L::kPitchW + kp + k + (lane >> 3 & 1) * 8);
            lr_mma16<T>(sum[0], x[k / 16], w[0], w[1]);
            lr_mma16<T>(sum[1], x[k / 16], w[2], w[3]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[2 * j][i] += sum[0][i];
            acc[2 * j + 1][i] += sum[1][i];
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
      const long long place = (long long)(tile.place + row) * R + col, next = (long long)a.groups.n * R;
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
        __align__(8) T part_of[LrParts<T>::kCount][4];
        lr_parts<T>(f, part_of);
        T* to = BF16 ? (T*)a.kept.values : (T*)a.kept.parts;
#pragma unroll
        for (int p = 0; p < LrParts<T>::kCount; ++p) {
          const uint2 four = *reinterpret_cast<const uint2*>(part_of[p]);
          if constexpr (!SPLIT) *reinterpret_cast<uint2*>(hs + (p * M + row) * L::kPitchH + col) = four;
          if (keeps && to != nullptr) *reinterpret_cast<uint2*>(to + p * next + place) = four;
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
    uint32_t held[kSteps][LrParts<T>::kCount][4], next[kSteps][4][2];
    int b = b0 + warp;
    if (kHold && has) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
#pragma unroll
        for (int p = 0; p < LrParts<T>::kCount; ++p) load_h(k * kStep, p, held[k][p]);
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
          for (int k = 0; k < kSteps; ++k) lr_multiply<T>(acc, held[k], w[k]);
        } else {
#pragma unroll 2
          for (int k = 0; k < R; k += kStep) {
            if (k >= a.rank) break;
            uint32_t w[4][2], h[LrParts<T>::kCount][4];
            w2.load(b, k, w);
#pragma unroll
            for (int p = 0; p < LrParts<T>::kCount; ++p) load_h(k, p, h[p]);
            lr_multiply<T>(acc, h, w);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (row_of[h] < 0 || left <= 0) continue;
        float v[8];
        lr_get<T>(acc, h, up[h], from[h], has, v);
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
// memory; warps do not wait for one another.  8192 rows to 12288 values, rank 16, bf16: 402 MB in 79 us, 5.1 TB/s, 19 % of the issue slots (41 M
// instructions with everything checked took 95 us, 12.5 M in whole blocks of known rank 74, 13.6 M with the third part of the rank values 79).  The next kernel is not let in early, as in dropout.cu (a training step of
// 8192 rows: 327 us, 289 without).
template <typename T, int R, bool BACK> struct LrExpand {
  static constexpr int kGroups = sizeof(T) == 4 ? 2 : 4, kCols = 32 * kGroups;         // of a block of columns
  static constexpr int kStages = 2, kPieces = 8, kRing = BACK ? 0 : kLrWarps * kStages * kPieces * 512;
  // results of rows at odd addresses pass through shared memory, 16 rows of a block, so that lanes write neighbouring values (f32, 8000 rows 4095 to 4097 values,
  // rank 16: 255 us forward and 446 backward with eights to a lane, 198 and 353 so)
  static constexpr int kPitch = kCols + 16 / (int)sizeof(T), kTile = 16 * kPitch * (int)sizeof(T);
  static constexpr int bytes(bool vec) { return vec ? kRing : kRing > kLrWarps * kTile ? kRing : kLrWarps * kTile; }
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
  // the rank values' parts; rows behind the last have those of the first one, which go nowhere
  const long long at[2] = {(long long)(place + (g < count ? g : 0)) * R + kEach * t, (long long)(place + (g + 8 < count ? g + 8 : 0)) * R + kEach * t};
  auto load_h = [&](int k, uint32_t (*part)[4]) {
    if constexpr (F32) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 f = *reinterpret_cast<const float2*>((const float*)a.kept.values + at[h] + k);
        lr_split(f.x, part[0][h], part[1][h]);
        lr_split(f.y, part[0][2 + h], part[1][2 + h]);
      }
    } else {
      const T* p = BF16 ? (const T*)a.kept.values : (const T*)a.kept.parts;
      const long long next = (long long)a.groups.n * R;
#pragma unroll
      for (int i = 0; i < LrParts<T>::kCount; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint2 u = *reinterpret_cast<const uint2*>(p + i * next + at[h] + k);
          part[i][h] = u.x; part[i][2 + h] = u.y;
        }
    }
  };
  float up[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) up[h] = F16 && has ? a.kept.factors[place + (g + 8 * h < count ? g + 8 * h : 0)] : 1.0f;
  constexpr int kSteps = X::kHold ? R / kStep : 1;
  uint32_t held[kSteps][LrParts<T>::kCount][4];
  if (X::kHold && has) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) load_h(k * kStep, held[k]);
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
        for (int k = 0; k < kSteps; ++k) lr_multiply<T>(acc, held[k], w[q % X::kWays][k]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[8];
          lr_get<T>(acc, h, up[h], base[h], true, v);
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
#pragma unroll
          for (int p = LrParts<T>::kCount - 1; p >= 0; --p) lr_mma16<T>(acc[j], held[k][p], w0, w1);
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
  T* tile = reinterpret_cast<T*>(lr_dynamic + warp * X::kTile);
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
            lr_multiply<T>(acc, held[k], w);
          }
        } else {
#pragma unroll 2
          for (int k = 0; k < R; k += kStep) {
            if (k >= a.rank) break;
            uint32_t w[4][2], h[LrParts<T>::kCount][4];
            w2.load(b, k, w);
            load_h(k, h);
            lr_multiply<T>(acc, h, w);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (row_of[h] < 0 || left <= 0) continue;
        float v[8];
        lr_get<T>(acc, h, up[h], base[h], has, v);
        if (BACK && a.drop_y && has) lr_drop(v, dropout_words((unsigned)(b * 32 + 8 * t) >> 3, row_of[h], key), a.drop.limit);
        if (group > a.groups.adapters) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(0x7fc00000u);
        }
        lr_store8<T, true>(a.vec_y ? to[h] + b * 32 : tile + (g + 8 * h) * X::kPitch + q * 32 + 8 * t, 8, v);
      }
    }
    if (!a.vec_y) {
      __syncwarp();
      T* p = (T*)a.y + c * X::kCols + lane;
#pragma unroll 2
      for (int r = 0; r < 16; ++r) {
        const int row = __shfl_sync(0xffffffffu, r < 8 ? row_of[0] : row_of[1], (r & 7) * 4);
        if (row < 0) continue;
#pragma unroll
        for (int q = 0; q < X::kGroups; ++q)
          if (c * X::kCols + q * 32 + lane < a.cols) p[row * a.ldy + q * 32] = tile[r * X::kPitch + q * 32 + lane];
      }
      __syncwarp();
    }
    request(c + 2, stage);
  }
  if (!BACK) lr_wait<0>();
}

}  // namespace bonsai
