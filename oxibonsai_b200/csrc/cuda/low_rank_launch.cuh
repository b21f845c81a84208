// Which kernel a low-rank update takes, and how many blocks.
#pragma once
#include <atomic>

#include "low_rank_outer.cuh"
#include "low_rank_rows.cuh"

namespace bonsai {

template <auto KERNEL, typename... Args>
static cudaError_t lr_launch(long long clusters, int ranks, int smem, cudaStream_t st, const Args&... args) {
  if (clusters * ranks >= 1ll << 31) return cudaErrorInvalidValue;
  if (smem > 48 * 1024) {          // allowed once for each kernel and device: it costs the host a microsecond.  A kernel's size above 48 KB is always the same
    static std::atomic<unsigned long long> allowed{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if ((allowed.load(std::memory_order_relaxed) & bit) == 0) {
      e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
      allowed.fetch_or(bit, std::memory_order_relaxed);
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
  return cudaLaunchKernelEx(&cfg, KERNEL, args...);
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
  return lr_launch<lr_rows_kernel<T, R, M, BACK, SPLIT>>(slots, lr_ranks_for(busy < 1 ? 1 : busy, chunks, 148 * L::kBlocks, 4), L::kBytes, st, a);
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
  return lr_launch<lr_expand_kernel<T, R, BACK>>(grid, 1, X::bytes(a.vec_y), st, a, tiles, row_blocks, per);
}

template <typename T, int R, bool BACK>
static cudaError_t lr_rows_r(const LrRowsArgs& a, cudaStream_t st) {
  const LrGroups& g = a.groups;
  if (!a.split) return lr_rows_as<T, R, 16, BACK, false>(a, st);
  // Tiles of 64 rows where adapters fill them; 16 rows keep more clusters busy and waste less of the tiles.  8192 rows, 4096 to 12288, rank 16, forward, us in tiles of
  // 64 and of 16: bf16 680 rows an adapter 139 and 152, 205 rows 147 and 154, 82 rows 152 and 150, 41 rows 164 and 160, 20 rows 220 and 205; f32 309 and 319, 360
  // and 355, 402 and 374, 419 and 407, 550 and 468
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
  // How the rows are split goes by both products, wanted or not: a gradient has the same bits alone and beside the other.  Dropped columns, which take longer, have no
  // rule of their own: clusters of eight from 2048 rows on, which was one, took 176 us where this takes 179 (all gradients of 8192 rows, 4096 to 12288,
  // rank 16, bf16), but 101 and 95 of 4096 rows, 220 and 206 of three adapters, 721 and 578 of three in f32.
  const long long both = ((a.width[0] + kLrOuterCols - 1) / kLrOuterCols + (a.width[1] + kLrOuterCols - 1) / kLrOuterCols) * (long long)a.groups.adapters;
  const int ranks = lr_ranks_for(both, steps, 148 * L::kBlocks, 4);
  return lr_launch<lr_outer_kernel<T, R>>(clusters, ranks, L::kBytes, st, a);
}

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
