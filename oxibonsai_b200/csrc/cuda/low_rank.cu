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
// rows of `width` values at distances of ld that begin at multiples of 16 bytes and hold whole eights
static int lr_vec(const void* p, long long ld, long long width, int size) { return width % 8 == 0 && ((uintptr_t)p | (uintptr_t)(ld * size)) % 16 == 0; }

// What a forward pass leaves for the backward one: the rank values, the order of rows and where each adapter's rows begin in it.
struct LrKept {
  long long order, start, bytes;
};
static LrKept lr_kept(int n, int rank, int adapters, bool grouped, bool values) {
  LrKept k;
  k.order = values ? 4ll * n * lr_padded(rank) : 0;
  k.start = k.order + (grouped ? (4ll * n + 15) / 16 * 16 : 0);
  k.bytes = k.start + (grouped ? 4ll * (adapters + 3) : 0);
  return k;
}

template <typename Args>
static cudaError_t lr_rows_by(int type, const Args& a, bool back, cudaStream_t st) {
  return type == 0 ? lr_rows<float>(a, back, st) : type == 1 ? lr_rows<__half>(a, back, st) : lr_rows<__nv_bfloat16>(a, back, st);
}

}  // namespace bonsai

extern "C" {

// Rows of ids that a forward pass groups without `kept`, where no backward pass follows.
int bonsai_lr_self_rows() { return bonsai::kLrSelf; }

// Bytes of `kept` for a forward pass (values: the rank values are wanted behind it; grouped: ids are given), and of the workspace of the backward pass
// (values alone).  Negative for sizes that are refused.
long long bonsai_lr_bytes(int n, int rank, int adapters, int grouped, int values) {
  using namespace bonsai;
  return lr_good(n, 1, 1, rank, adapters, 0) ? lr_kept(n, rank, adapters, grouped, values).bytes : BONSAI_CUDA_BAD_ARG;
}

// y [n][out] = base + s b (a x) by rows: a [adapters][rank][d], b [adapters][out][rank], rows of x, base and y at distances of their ld; base may be null, or y
// itself.  ids (int32, or int64 where wide; negative: a row without an adapter) may be null with one adapter.  scales [adapters], or scale.  x is dropped
// where steps < 65536.  kept: bonsai_lr_bytes of this call, null where nothing is kept and ids are absent or at most bonsai_lr_self_rows.
int bonsai_lr_forward(const void* x, long long ldx, const void* a, const void* b, const void* base, long long ld_base, void* y, long long ldy,
                      const float* scales, float scale, int n, int d, int out, int rank, int adapters, int type, const void* ids, int ids_wide, void* kept,
                      long long kept_bytes, int values, unsigned long long seed, const long long* seed_dev, int steps, cudaStream_t st) {
  using namespace bonsai;
  if (x == nullptr || a == nullptr || b == nullptr || y == nullptr || !lr_good(n, d, out, rank, adapters, type) || steps < 0 || steps > 65536 ||
      (ids == nullptr && adapters != 1) || (values && kept == nullptr) || (ids != nullptr && kept == nullptr && n > kLrSelf))
    return BONSAI_CUDA_BAD_ARG;
  const LrKept at = lr_kept(n, rank, adapters, ids != nullptr, values);
  if (kept != nullptr && kept_bytes < at.bytes) return BONSAI_CUDA_BAD_ARG;
  char* room = (char*)kept;
  LrGroups g = {LR_ONE, ids, ids_wide, nullptr, nullptr, n, adapters};
  cudaError_t e = cudaSuccess;
  if (ids != nullptr) {
    g.mode = kept == nullptr ? LR_SELF : LR_PLAN;
    if (g.mode == LR_PLAN) {
      g.order = (const int*)(room + at.order);
      g.start = (const int*)(room + at.start);
      e = launch_pdl(lr_plan_kernel, dim3(adapters + 2), dim3(kPlanThreads), 0, st, g, (int*)(room + at.order), (int*)(room + at.start));
    }
  }
  if (e != cudaSuccess) return BONSAI_CUDA_LAUNCH_FAILED;
  const int size = type == 0 ? 4 : 2;
  LrRowsArgs r = {g, x, ldx, a, b, base, ld_base, y, ldy, values ? kept : nullptr, scales, scale, d, out, rank};
  r.vec_x = lr_vec(x, ldx, d, size);
  r.vec_w1 = lr_vec(a, d, d, size);
  r.vec_w2 = rank % (8 / size) == 0 && (uintptr_t)b % 8 == 0;         // rank values of a column as words of 8 bytes
  r.vec_y = lr_vec(y, ldy, out, size) && (base == nullptr || lr_vec(base, ld_base, out, size));
  r.drop = dropout_rule(seed, seed_dev, steps);
  r.drop_x = steps < 65536;
  return lr_rows_by(type, r, false, st) == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

// Gradients of bonsai_lr_forward: dx [n][d], da, db (like a and b; zeros of adapters without rows), each may be null.  kept: of the forward pass, with the
// values where db is wanted (values: whether it has them).  ws: bonsai_lr_bytes(n, rank, adapters, 0, 1) where da is wanted.
int bonsai_lr_backward(const void* x, long long ldx, const void* dy, long long lddy, const void* a, const void* b, void* dx, void* da, void* db,
                       const float* scales, float scale, int n, int d, int out, int rank, int adapters, int type, int grouped, const void* kept,
                       long long kept_bytes, int values, void* ws, long long ws_bytes, unsigned long long seed, const long long* seed_dev, int steps,
                       cudaStream_t st) {
  using namespace bonsai;
  if (dy == nullptr || b == nullptr || !lr_good(n, d, out, rank, adapters, type) || steps < 0 || steps > 65536 || (!grouped && adapters != 1) ||
      (dx != nullptr && a == nullptr) || (da != nullptr && (x == nullptr || ws == nullptr)) || (db != nullptr && !values) || ((grouped || db != nullptr) && kept == nullptr))
    return BONSAI_CUDA_BAD_ARG;
  const LrKept at = lr_kept(n, rank, adapters, grouped, values);
  if ((kept != nullptr && kept_bytes < at.bytes) || (da != nullptr && ws_bytes < lr_kept(n, rank, adapters, false, true).bytes)) return BONSAI_CUDA_BAD_ARG;
  const char* room = (const char*)kept;
  LrGroups g = {LR_ONE, nullptr, 0, nullptr, nullptr, n, adapters};
  if (grouped) {
    g.mode = LR_PLAN;
    g.order = (const int*)(room + at.order);
    g.start = (const int*)(room + at.start);
  }
  const int size = type == 0 ? 4 : 2;
  const DropoutRule rule = dropout_rule(seed, seed_dev, steps);
  cudaError_t e = cudaSuccess;
  if (dx != nullptr || da != nullptr) {
    LrRowsArgs r = {g, dy, lddy, b, a, nullptr, 0, dx, d, da != nullptr ? ws : nullptr, scales, scale, out, d, rank};
    r.vec_x = lr_vec(dy, lddy, out, size);
    r.vec_w1 = lr_vec(b, rank, rank, size);
    r.vec_w2 = lr_vec(a, d, d, size);
    r.vec_y = lr_vec(dx, d, d, size);
    r.drop = rule;
    r.drop_y = steps < 65536;
    e = lr_rows_by(type, r, true, st);
  }
  if (e == cudaSuccess && (da != nullptr || db != nullptr)) {
    LrOuterArgs o = {g, {x, dy}, {ldx, lddy}, {ws, kept}, {da, db}, {d, out}};
    o.blocks[0] = da != nullptr ? (d + kLrOuterCols - 1) / kLrOuterCols : 0;
    o.blocks[1] = db != nullptr ? (out + kLrOuterCols - 1) / kLrOuterCols : 0;
    o.vec[0] = lr_vec(x, ldx, d, size);
    o.vec[1] = lr_vec(dy, lddy, out, size);
    o.rank = rank;
    o.scales = scales;
    o.scale = scale;
    o.drop = rule;
    o.drop_x = steps < 65536;
    e = type == 0 ? lr_outer<float>(o, st) : type == 1 ? lr_outer<__half>(o, st) : lr_outer<__nv_bfloat16>(o, st);
  }
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

}  // extern "C"
