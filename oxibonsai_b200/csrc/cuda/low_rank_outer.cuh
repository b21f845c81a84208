// The gradients of the factors of a low-rank update (low_rank.cuh has the formulas).
#pragma once
#include "low_rank.cuh"

namespace bonsai {

// ---- the factors' gradients --------------------------------------------------------------------------------------------------------------
// out[r][c] (or [c][r]) = sum over the adapter's rows of p[row][r] q[row][c]; the rank values p have the scales in them.  A cluster takes 128 columns of one adapter and one product, its blocks
// split the rows.  bf16: the rank values' three parts times q, both as ldmatrix turns them.  f16 and f32: TF32, where f16 is exact (its range would lose small rank
// values); the two rows 2 t and 2 t + 1 of every eight are then what a thread has of a matrix instruction's axis of eight, which is how
// ldmatrix hands out 16-bit values of q; p follows.  8192 rows, 4096 and 12288 columns, rank 16, bf16: 270 MB in 68 us, 4.0 TB/s, with dropout of
// the 4096 columns 89.
template <typename T, int R> struct LrOuterSmem {
  static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  // bf16: a row's three parts side by side, whose pitch spreads eight rows over all banks; else the first parts and, kP bytes on, the second ones
  static constexpr int kPitchQ = kLrOuterCols + (sizeof(T) == 4 ? 4 : 8), kPitchP = kBf16 ? 3 * R + 8 : R + 4;
  static constexpr int kP = kLrOuterRows * kPitchP * (kBf16 ? 2 : 4);
  static constexpr int kStage = kLrOuterRows * kPitchQ * (int)sizeof(T) + (kBf16 ? 1 : 2) * kP;
  static constexpr int kSum = R * kLrOuterCols * 4;
  // bf16 of rank 64 takes two stages, which leave room for a second block: 8192 rows to 12288 columns in 198 us, with three stages and one block 221
  static constexpr int kStages = 3 * kStage <= (kBf16 && R == 64 ? kLrSmemHalf : kLrSmemMost) ? 3 : 2;
  static constexpr int kBytes = kStages * kStage > kSum ? kStages * kStage : kSum;
  static constexpr int kBlocks = kBytes <= kLrSmemThird && R <= 32 ? 3 : kBytes <= kLrSmemHalf && R <= 64 ? 2 : 1;            // on an SM
  static_assert(kBytes <= kLrSmemMost, "shared memory");
};

template <typename T, int R>
__global__ void __launch_bounds__(kLrThreads, LrOuterSmem<T, R>::kBlocks) lr_outer_kernel(const __grid_constant__ LrOuterArgs a) {
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
    } else if (a.vec[which]) {
#pragma unroll 1
      for (int r = 0; r < kLrOuterRows; r += kRows)
        lr_copy8<T>(to + r * L::kPitchQ, q + places[s % 4][r0 + r] + col0 + c0, from + r0 + r < last ? width - col0 - c0 : 0, true, q);
    } else {
      lr_copy_rows<T, kLrOuterRows, kLrOuterCols>(qs(slot), L::kPitchQ, width - col0, q, [&](int r) { return from + r < last ? q + places[s % 4][r] + col0 : (const T*)nullptr; });
    }
    // rank values: eights of the rows side by side, of bf16 all parts
    using P = typename std::conditional<BF16, T, float>::type;
    constexpr int kOne = kLrOuterRows * (R / 8), kAll = BF16 ? 3 * kOne : kOne;
    const P* p = (const P*)a.p[which] + (long long)from * R;
#pragma unroll
    for (int u0 = 0; u0 < kAll; u0 += kLrThreads) {
      const int u = u0 + threadIdx.x;
      if (kAll % kLrThreads != 0 && u >= kAll) break;
      const int part = u / kOne, r = u % kOne / (R / 8), c = u % (R / 8) * 8;
      const P* src = p + part * (long long)a.groups.n * R + r * R + c;
      lr_copy8<P>((P*)ps(slot) + r * L::kPitchP + part * R + c, src, from + r < last ? 8 : 0, true, (const P*)a.p[which]);
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
      if (!a.vec[which]) __syncthreads();          // others have copied them
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
      uint32_t w[kLrOuterRows / 16][4];
#pragma unroll
      for (int k = 0; k < kLrOuterRows; k += 16) lr_ldm4t(w[k / 16], qp + (k + (lane & 15)) * L::kPitchQ + (lane >> 4) * 8);
#pragma unroll
      for (int i = 0; i < R / 16; ++i) {
        float sum[2][4] = {};
#pragma unroll
        for (int k = 0; k < kLrOuterRows; k += 16) {
          const T* p = pp + (k + (lane & 7) + (lane >> 4) * 8) * L::kPitchP + i * 16 + (lane >> 3 & 1) * 8;
#pragma unroll
          for (int part = 2; part >= 0; --part) {
            uint32_t v[4];
            lr_ldm4t(v, p + part * R);
#pragma unroll
            for (int j = 0; j < 2; ++j) lr_mma16<T>(sum[j], v, w[k / 16][2 * j], w[k / 16][2 * j + 1]);
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[i][j][k] += sum[j][k];
      }
    } else {
      const uint32_t* pp = (const uint32_t*)ps(slot);
      float sum[R / 16][2][4];
#pragma unroll
      for (int i = 0; i < R / 16; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) sum[i][j][k] = 0.0f;
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
              lr_mma8(sum[i][j], lo, vh[j][0], vh[j][1]);
              if constexpr (F32) lr_mma8(sum[i][j], hi, vl[j][0], vl[j][1]);
              lr_mma8(sum[i][j], hi, vh[j][0], vh[j][1]);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < R / 16; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[i][j][k] += sum[i][j][k];
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

}  // namespace bonsai
