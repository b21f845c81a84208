// Entry points of the low-rank updates (low_rank.cuh), and the order of rows by adapter that their tiles go by.
#include "low_rank.cuh"

namespace bonsai {

constexpr int kPlanThreads = 512, kPlanEach = 8;

// order: the rows by adapter, in their own order within each; start[e]: where adapter e's begin.  A block makes one adapter's list on its own: it counts
// the ids below its own, which is where the list begins, and goes through the ids once more.  Nothing is shared between blocks, no atomics.
__global__ void __launch_bounds__(kPlanThreads) lr_plan_kernel(LrGroups g, int* order, int* start) {
  __shared__ int warps[kPlanThreads / 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int e = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int per = kPlanThreads * kPlanEach;
  auto block_scan = [&](int v, int& all) {            // how many before this thread's
    int up = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += w;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = up;
    __syncthreads();
    int before = 0;
    all = 0;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      before += w < warp ? warps[w] : 0;
      all += warps[w];
    }
    return before + up - v;
  };
  int below = 0;
  for (long long row = t; row < g.n; row += kPlanThreads) below += lr_group(g, (int)row) < e;
  int place;
  block_scan(below, place);
  if (t == 0) {
    start[e] = place;
    if (e == g.adapters + 1) start[e + 1] = g.n;
  }
  for (long long first = 0; first < g.n; first += per) {
    const long long row = first + (long long)t * kPlanEach;
    unsigned mine = 0;
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i)
      if (row + i < g.n && lr_group(g, (int)(row + i)) == e) mine |= 1u << i;
    int all;
    int at = place + block_scan(__popc(mine), all);
    for (unsigned m = mine; m != 0; m &= m - 1) order[at++] = (int)row + __ffs(m) - 1;
    place += all;
  }
}

static bool lr_good(int n, int k, int cols, int rank, int adapters, int type) {
  constexpr int kMost = 1 << 30;
  return n >= 1 && n < kMost && k >= 1 && k < kMost && cols >= 1 && cols < kMost && rank >= 1 && rank <= 128 && adapters >= 1 && adapters <= 65536 && type >= 0 &&
         type <= 2;
}
static bool lr_groups_good(const LrGroups& g) {
  return g.mode == LR_ONE ? g.adapters == 1 : g.mode == LR_SELF ? g.ids != nullptr && g.n <= kLrSelf : g.mode == LR_PLAN && g.order != nullptr && g.start != nullptr;
}
// rows of `width` values at distances of ld that begin at multiples of 16 bytes and hold whole eights
static int lr_vec(const void* p, long long ld, long long width, int size) { return width % 8 == 0 && ((uintptr_t)p | (uintptr_t)(ld * size)) % 16 == 0; }
}  // namespace bonsai

extern "C" {

// Rank values of a row in `kept`.
int bonsai_lr_padded(int rank) { return bonsai::lr_padded(rank); }

// Rows that may be grouped without a plan (mode 1).
int bonsai_lr_self_rows() { return bonsai::kLrSelf; }

// order: int [n], start: int [adapters + 3]; ids: int32, or int64 where wide, negative for rows without an adapter.
int bonsai_lr_plan(const void* ids, int wide, int n, int adapters, int* order, int* start, cudaStream_t st) {
  using namespace bonsai;
  if (ids == nullptr || order == nullptr || start == nullptr || !lr_good(n, 1, 1, 1, adapters, 0)) return BONSAI_CUDA_BAD_ARG;
  const LrGroups g = {LR_PLAN, ids, wide, nullptr, nullptr, n, adapters};
  const cudaError_t e = launch_pdl(lr_plan_kernel, dim3(adapters + 2), dim3(kPlanThreads), 0, st, g, order, start);
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

// back = 0: y [n][cols] = base + s w2 (w1 x), w1 [adapters][rank][k], w2 [adapters][cols][rank], x dropped by `steps` of 65536.
// back = 1: y [n][cols] = s w2^T (w1^T x) dropped, w1 [adapters][k][rank], w2 [adapters][rank][cols].
// mode: 0 one adapter, 1 ids of at most bonsai_lr_self_rows() rows, 2 order and start of bonsai_lr_plan.  kept (may be null; not with mode 1): the rank
// values, [n][bonsai_lr_padded(rank)] of 4 bytes by place in the order, for bonsai_lr_outer.  base may be null, or y itself;
// y may be null where the rank values alone are wanted.
int bonsai_lr_rows(const void* x, long long ldx, const void* w1, const void* w2, const void* base, long long ld_base, void* y, long long ldy, void* kept,
                   const float* scales, float scale, int n, int k, int cols, int rank, int adapters, int type, int back, int mode, const void* ids, int ids_wide,
                   const int* order, const int* start, unsigned long long seed, const long long* seed_dev, int steps, cudaStream_t st) {
  using namespace bonsai;
  const LrGroups g = {mode, ids, ids_wide, order, start, n, adapters};
  if (x == nullptr || w1 == nullptr || w2 == nullptr || (y == nullptr && kept == nullptr) || !lr_good(n, k, cols, rank, adapters, type) || !lr_groups_good(g) || steps < 0 ||
      steps > 65536 || (kept != nullptr && mode == LR_SELF))
    return BONSAI_CUDA_BAD_ARG;
  const int size = type == 0 ? 4 : 2, drop = steps < 65536;
  LrRowsArgs a = {g, x, ldx, w1, w2, base, ld_base, y, ldy, kept, scales, scale, k, cols, rank, 0};
  a.vec_x = lr_vec(x, ldx, k, size);
  a.vec_w1 = back ? lr_vec(w1, rank, rank, size) : lr_vec(w1, k, k, size);
  // forward: rank values of a column as words of 8 bytes
  a.vec_w2 = back ? lr_vec(w2, cols, cols, size) : rank % (8 / size) == 0 && (uintptr_t)w2 % 8 == 0;
  a.vec_y = lr_vec(y, ldy, cols, size) && (base == nullptr || lr_vec(base, ld_base, cols, size));
  a.drop = dropout_rule(seed, seed_dev, steps);
  a.drop_x = drop && !back;
  a.drop_y = drop && back;
  const cudaError_t e = type == 0 ? lr_rows<float>(a, back, st) : type == 1 ? lr_rows<__half>(a, back, st) : lr_rows<__nv_bfloat16>(a, back, st);
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

// da [adapters][rank][d] = s sum g x^T (x dropped), db [adapters][out][rank] = s sum dy h^T over each adapter's rows; either may be null.  g, h: `kept`
// of the two directions.  Adapters without rows get zeros.
int bonsai_lr_outer(const void* x, long long ldx, const void* g, void* da, int d, const void* dy, long long lddy, const void* h, void* db, int out,
                    const float* scales, float scale, int n, int rank, int adapters, int type, int mode, const int* order, const int* start,
                    unsigned long long seed, const long long* seed_dev, int steps, cudaStream_t st) {
  using namespace bonsai;
  const LrGroups groups = {mode, nullptr, 0, order, start, n, adapters};
  if (!lr_good(n, d, out, rank, adapters, type) || mode == LR_SELF || !lr_groups_good(groups) || steps < 0 || steps > 65536 || (da == nullptr && db == nullptr) ||
      (da != nullptr && (x == nullptr || g == nullptr)) || (db != nullptr && (dy == nullptr || h == nullptr)))
    return BONSAI_CUDA_BAD_ARG;
  const int size = type == 0 ? 4 : 2;
  LrOuterArgs a = {groups, {x, dy}, {ldx, lddy}, {g, h}, {da, db}, {d, out}};
  a.blocks[0] = da != nullptr ? (d + kLrOuterCols - 1) / kLrOuterCols : 0;
  a.blocks[1] = db != nullptr ? (out + kLrOuterCols - 1) / kLrOuterCols : 0;
  a.vec[0] = lr_vec(x, ldx, d, size);
  a.vec[1] = lr_vec(dy, lddy, out, size);
  a.rank = rank;
  a.scales = scales;
  a.scale = scale;
  a.drop = dropout_rule(seed, seed_dev, steps);
  a.drop_x = steps < 65536;
  const cudaError_t e = type == 0 ? lr_outer<float>(a, st) : type == 1 ? lr_outer<__half>(a, st) : lr_outer<__nv_bfloat16>(a, st);
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

}  // extern "C"
