// Entry points of the low-rank updates (low_rank.cuh), and the order of rows by adapter that their tiles go by.
#include "low_rank.cuh"

namespace bonsai {

constexpr int kPlanThreads = 512, kPlanEach = 8;

// order: the rows by adapter, in their own order within each; start[e]: where adapter e's begin.  A block makes one adapter's list on its own: it counts
// the ids below its own, which is where the list begins, and goes through the ids once more.  Nothing is shared between blocks, no atomics.
// tiles and their rows (may be null): of 16 rows, those of adapter e in places start[e] / 16 + e to start[e + 1] / 16 + e, which are enough for all and lie
// apart.
__global__ void __launch_bounds__(kPlanThreads) lr_plan_kernel(LrGroups g, int* order, int* start, int4* tiles, int* tile_rows) {
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
  // bit i: the thread's i-th id of the sweep is this adapter's; below: how many are smaller ones
  auto sweep = [&](long long first, int& below) {
    const long long row = first + (long long)t * kPlanEach;
    unsigned mine = 0;
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i)
      if (row + i < g.n) {
        const int of = lr_group(g, (int)(row + i));
        mine |= (of == e ? 1u : 0u) << i;
        below += of < e;
      }
    return mine;
  };
  int below = 0, place, skip = 0;
  unsigned mine = sweep(0, below);
  for (long long first = per; first < g.n; first += per) sweep(first, below);
  block_scan(below, place);
  if (t == 0) {
    start[e] = place;
    if (e == g.adapters + 1) start[e + 1] = g.n;
  }
  const int begin = place;
  for (long long first = 0; first < g.n; first += per) {
    if (first > 0) mine = sweep(first, skip);
    int all;
    int at = place + block_scan(__popc(mine), all);
    for (unsigned m = mine; m != 0; m &= m - 1, ++at) {
      const int row = (int)(first + (long long)t * kPlanEach) + __ffs(m) - 1;
      order[at] = row;
      if (tiles != nullptr) tile_rows[(begin / 16 + e) * 16ll + at - begin] = row;
    }
    place += all;
  }
  if (tiles != nullptr)
    for (int i = t; i <= place / 16 - begin / 16; i += kPlanThreads) {
      const int at = begin + 16 * i, left = place - at;
      tiles[begin / 16 + e + i] = left > 0 ? make_int4(e, at, left < 16 ? left : 16, 0) : make_int4(-1, 0, 0, 0);
      for (int r = left > 0 ? left : 0; r < 16; ++r) tile_rows[(begin / 16 + e + i) * 16ll + r] = -1;
    }
}

static bool lr_good(int n, int k, int cols, int rank, int adapters, int type) {
  constexpr int kMost = 1 << 30;
  return n >= 1 && n < kMost && k >= 1 && k < kMost && cols >= 1 && cols < kMost && rank >= 1 && rank <= 128 && adapters >= 1 && adapters <= 4096 && type >= 0 &&
         type <= 2;
}
// rows of `width` values at distances of ld that begin at multiples of 16 bytes and hold whole eights
static int lr_vec(const void* p, long long ld, long long width, int size) { return width % 8 == 0 && ((uintptr_t)p | (uintptr_t)(ld * size)) % 16 == 0; }

// What a forward pass leaves for the backward one, and what the backward pass works with: the rank values (of bf16 three parts; of f16 also their two parts where the second product is a
// kernel of its own), the order of rows, where each adapter's rows begin in it, the tiles of 16 rows.
struct LrRoom {
  bool values;
  long long parts, factors, order, start, tiles, tile_rows, bytes;
};
static LrRoom lr_room(int n, int rank, int adapters, int type, bool grouped, bool values, bool split, bool tiles) {
  LrRoom k;
  k.values = values || split;
  auto up = [](long long b) { return (b + 15) / 16 * 16; };
  const long long all = (type == 2 ? 6ll : 4ll) * n * lr_padded(rank), slots = grouped && tiles ? n / 16 + adapters + 2 : 0;
  k.parts = k.values ? all : 0;
  k.factors = k.parts + (split && type == 1 ? all : 0);
  k.order = k.factors + (split && type == 1 ? up(4ll * n) : 0);
  k.start = k.order + (grouped ? up(4ll * n) : 0);
  k.tiles = k.start + (grouped ? up(4ll * (adapters + 3)) : 0);
  k.tile_rows = k.tiles + 16 * slots;
  k.bytes = k.tile_rows + 64 * slots;
  return k;
}
// Of a forward pass (tiles are for its own second product or that of the backward one), and the workspace of the backward one.
static LrRoom lr_room_of(int n, int d, int out, int rank, int adapters, int type, bool grouped, bool values, bool back) {
  return back ? lr_room(n, rank, adapters, type, false, true, lr_split_at(n, d), false)
              : lr_room(n, rank, adapters, type, grouped, values, lr_split_at(n, out), lr_split_at(n, out) || lr_split_at(n, d));
}
static LrValues lr_values(void* room, const LrRoom& k) {
  char* p = (char*)room;
  const bool parts = k.factors > k.parts;
  return {k.values ? p : nullptr, parts ? (__half*)(p + k.parts) : nullptr, parts ? (float*)(p + k.factors) : nullptr};
}
static void lr_grouped(LrGroups& g, void* room, const LrRoom& k) {
  char* p = (char*)room;
  g.mode = LR_PLAN;
  g.order = (const int*)(p + k.order);
  g.start = (const int*)(p + k.start);
  const bool tiles = k.tile_rows > k.tiles;
  g.tiles = tiles ? (const int4*)(p + k.tiles) : nullptr;
  g.tile_rows = tiles ? (const int*)(p + k.tile_rows) : nullptr;
}

template <typename Args>
static cudaError_t lr_rows_by(int type, const Args& a, bool back, cudaStream_t st) {
  return type == 0 ? lr_rows<float>(a, back, st) : type == 1 ? lr_rows<__half>(a, back, st) : lr_rows<__nv_bfloat16>(a, back, st);
}

}  // namespace bonsai

extern "C" {

// Rows of ids that a forward pass groups without `kept`, where no backward pass follows.
int bonsai_lr_self_rows() { return bonsai::kLrSelf; }

// Bytes of `kept` for a forward pass (values: the rank values are wanted behind it; grouped: ids are given), or of the workspace of the backward pass (back).
// 0: none is needed.  Negative for sizes that are refused.
long long bonsai_lr_bytes(int n, int d, int out, int rank, int adapters, int type, int grouped, int values, int back) {
  using namespace bonsai;
  return lr_good(n, d, out, rank, adapters, type) ? lr_room_of(n, d, out, rank, adapters, type, grouped, values, back).bytes : BONSAI_CUDA_BAD_ARG;
}

// y [n][out] = base + s b (a x) by rows: a [adapters][rank][d], b [adapters][out][rank], rows of x, base and y at distances of their ld; base may be null, or y
// itself.  ids (int32, or int64 where wide; negative: a row without an adapter) may be null with one adapter.  scales [adapters], or scale.  x is dropped
// where steps < 65536.  kept: bonsai_lr_bytes of this call; null where nothing is kept and there are at most bonsai_lr_self_rows ids.
int bonsai_lr_forward(const void* x, long long ldx, const void* a, const void* b, const void* base, long long ld_base, void* y, long long ldy,
                      const float* scales, float scale, int n, int d, int out, int rank, int adapters, int type, const void* ids, int ids_wide, void* kept,
                      long long kept_bytes, int values, unsigned long long seed, const long long* seed_dev, int steps, cudaStream_t st) {
  using namespace bonsai;
  if (x == nullptr || a == nullptr || b == nullptr || y == nullptr || !lr_good(n, d, out, rank, adapters, type) || steps < 0 || steps > 65536 ||
      (ids == nullptr && adapters != 1))
    return BONSAI_CUDA_BAD_ARG;
  const bool self = ids != nullptr && kept == nullptr && !values && n <= kLrSelf;
  const LrRoom at = lr_room_of(n, d, out, rank, adapters, type, ids != nullptr, values, false);
  if (!self && at.bytes > 0 && (kept == nullptr || kept_bytes < at.bytes)) return BONSAI_CUDA_BAD_ARG;
  LrGroups g = {LR_ONE, ids, ids_wide, nullptr, nullptr, nullptr, nullptr, n, adapters};
  cudaError_t e = cudaSuccess;
  if (ids != nullptr) {
    g.mode = LR_SELF;
    if (!self) {
      lr_grouped(g, kept, at);
      e = launch_pdl(lr_plan_kernel, dim3(adapters + 2), dim3(kPlanThreads), 0, st, g, (int*)g.order, (int*)g.start, (int4*)g.tiles, (int*)g.tile_rows);
    }
  }
  if (e != cudaSuccess) return BONSAI_CUDA_LAUNCH_FAILED;
  const int size = type == 0 ? 4 : 2;
  LrRowsArgs r = {g, x, ldx, a, b, base, ld_base, y, ldy, self ? LrValues{} : lr_values(kept, at), scales, scale, d, out, rank, lr_split_at(n, out)};
  // a single row may have any stride
  r.vec_x = lr_vec(x, n > 1 ? ldx : 0, d, size);
  r.vec_w1 = lr_vec(a, d, d, size);
  r.vec_w2 = rank % (8 / size) == 0 && (uintptr_t)b % 8 == 0;         // rank values of a column as words of 8 bytes
  r.vec_y = lr_vec(y, n > 1 ? ldy : 0, out, size) && (base == nullptr || lr_vec(base, n > 1 ? ld_base : 0, out, size));
  r.drop = dropout_rule(seed, seed_dev, steps);
  r.drop_x = steps < 65536;
  return lr_rows_by(type, r, false, st) == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

// Gradients of bonsai_lr_forward: dx [n][d], da, db (like a and b; zeros of adapters without rows), each may be null.  kept: of the forward pass, with the
// values where db is wanted (values, grouped: as there).  ws: bonsai_lr_bytes of the backward pass where dx or da is wanted.
int bonsai_lr_backward(const void* x, long long ldx, const void* dy, long long lddy, const void* a, const void* b, void* dx, void* da, void* db,
                       const float* scales, float scale, int n, int d, int out, int rank, int adapters, int type, int grouped, const void* kept,
                       long long kept_bytes, int values, void* ws, long long ws_bytes, unsigned long long seed, const long long* seed_dev, int steps,
                       cudaStream_t st) {
  using namespace bonsai;
  if (dy == nullptr || b == nullptr || !lr_good(n, d, out, rank, adapters, type) || steps < 0 || steps > 65536 || (!grouped && adapters != 1) ||
      (dx != nullptr && a == nullptr) || (da != nullptr && x == nullptr) || (db != nullptr && !values))
    return BONSAI_CUDA_BAD_ARG;
  const bool rows = dx != nullptr || da != nullptr;
  const LrRoom at = lr_room_of(n, d, out, rank, adapters, type, grouped, values, false), of = lr_room_of(n, d, out, rank, adapters, type, grouped, values, true);
  if ((at.bytes > 0 && (kept == nullptr || kept_bytes < at.bytes)) || (rows && (ws == nullptr || ws_bytes < of.bytes))) return BONSAI_CUDA_BAD_ARG;
  LrGroups g = {LR_ONE, nullptr, 0, nullptr, nullptr, nullptr, nullptr, n, adapters};
  if (grouped) lr_grouped(g, (void*)kept, at);
  const int size = type == 0 ? 4 : 2;
  const DropoutRule rule = dropout_rule(seed, seed_dev, steps);
  cudaError_t e = cudaSuccess;
  if (rows) {
    LrRowsArgs r = {g, dy, lddy, b, a, nullptr, 0, dx, d, lr_values(ws, of), scales, scale, out, d, rank, lr_split_at(n, d)};
    r.vec_x = lr_vec(dy, n > 1 ? lddy : 0, out, size);
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
    o.vec[0] = lr_vec(x, n > 1 ? ldx : 0, d, size);
    o.vec[1] = lr_vec(dy, n > 1 ? lddy : 0, out, size);
    o.rank = rank;
    o.drop = rule;
    o.drop_x = steps < 65536;
    e = type == 0 ? lr_outer<float>(o, st) : type == 1 ? lr_outer<__half>(o, st) : lr_outer<__nv_bfloat16>(o, st);
  }
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

}  // extern "C"
