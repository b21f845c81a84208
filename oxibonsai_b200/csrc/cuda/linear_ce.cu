// Softmax cross entropy of a linear head, in pieces of the vocabulary, without the logits, and its gradients.
//
//   z_iv = h_i . w_v,   lse_i = log sum_v exp z_iv,   q_iv = (1 - a) [v = t_i] + a / V
//   loss_i = lse_i - sum_v q_iv z_iv
//   dz_iv = u_i (exp(z_iv - lse_i) - q_iv),   dh = dz W,   dW = dz^T h
//
// Rows whose target is the ignored one are left out before anything is multiplied: the kernels work on the list of live rows, whose length
// stays on the device.  A target outside the vocabulary makes its row's loss and gradients NaN.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace bonsai {

constexpr int kCeTile = 64, kCeK = 16, kCeThreads = 256;
enum CeType { CE_F32 = 0, CE_F16 = 1, CE_BF16 = 2 };
enum CeReduce { CE_MEAN = 0, CE_SUM = 1, CE_NONE = 2 };

struct CeRows {         // the live rows, in order: filled by ce_rows_kernel
  int* count;           // [4]: live rows
  int* index;           // [N] row of the hidden states
  int* target;          // [N] its target, -1 outside the vocabulary
  float* lse;           // [N]
};

__device__ __forceinline__ float ce_f32(float x) { return x; }
__device__ __forceinline__ float ce_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float ce_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void ce_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void ce_put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void ce_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// One block walks the targets and lists the live rows in order.  `zero_loss`: where the loss of ignored rows goes (reduction "none").
__global__ void __launch_bounds__(1024) ce_rows_kernel(const long long* __restrict__ targets, int n, int vocab, long long ignore, CeRows r, float* zero_loss) {
  __shared__ int warps[32];
  __shared__ int base;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  if (t == 0) base = 0;
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += 1024) {
    const int i = i0 + t;
    const long long tgt = i < n ? targets[i] : ignore;
    const bool live = i < n && tgt != ignore;
    const unsigned m = __ballot_sync(0xffffffffu, live);
    if (lane == 0) warps[warp] = __popc(m);
    __syncthreads();
    int before = base, all = 0;
    for (int w = 0; w < 32; ++w) {
      const int c = warps[w];
      if (w < warp) before += c;
      all += c;
    }
    if (live) {
      const int at = before + __popc(m & ((1u << lane) - 1));
      r.index[at] = i;
      r.target[at] = tgt >= 0 && tgt < vocab ? (int)tgt : -1;
    } else if (i < n && zero_loss != nullptr) {
      zero_loss[i] = 0.0f;
    }
    __syncthreads();
    if (t == 0) base += all;
    __syncthreads();
  }
  if (t == 0) *r.count = base;
}

template <typename LA, typename LB>
__device__ __forceinline__ void ce_tile(LA a, LB b, int K, float (&acc)[4][4], float (*sa)[kCeTile + 4], float (*sb)[kCeTile + 4]) {
  const int t = threadIdx.x, tx = t & 15, ty = t >> 4;
  for (int k0 = 0; k0 < K; k0 += kCeK) {
    for (int i = t; i < kCeTile * kCeK; i += kCeThreads) {
      sa[i & 15][i >> 4] = k0 + (i & 15) < K ? a(i >> 4, k0 + (i & 15)) : 0.0f;
      sb[i & 15][i >> 4] = k0 + (i & 15) < K ? b(i >> 4, k0 + (i & 15)) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kCeK; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][4 * ty + i], sb[k][4 * tx + j], acc[i][j]);
    __syncthreads();
  }
}

template <typename T>
struct CeHead {
  const T* h;
  const T* w;
  long long ldh, ldw;
  int vocab, hidden;
};

// partial [slot][N] = (maximum, sum of exp below it, sum of z) of a row over 64 vocabulary rows; zt: z at the target
template <typename T>
__global__ void __launch_bounds__(kCeThreads) ce_lse_kernel(CeHead<T> p, CeRows r, float* part, float* zt, long long n_ld) {
  __shared__ float sa[kCeK][kCeTile + 4], sb[kCeK][kCeTile + 4];
  const int n = *r.count, r0 = blockIdx.y * kCeTile, v0 = blockIdx.x * kCeTile;
  if (r0 >= n) return;
  float acc[4][4] = {};
  ce_tile([&](int m, int k) { return r0 + m < n ? ce_f32(p.h[(long long)r.index[r0 + m] * p.ldh + k]) : 0.0f; },
          [&](int m, int k) { return v0 + m < p.vocab ? ce_f32(p.w[(long long)(v0 + m) * p.ldw + k]) : 0.0f; }, p.hidden, acc, sa, sb);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + 4 * ty + i;
    float m = -INFINITY, s = 0.0f, z = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (v0 + 4 * tx + j >= p.vocab) acc[i][j] = -INFINITY;
      else z += acc[i][j];
      m = fmaxf(m, acc[i][j]);
    }
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
    for (int j = 0; j < 4; ++j) s += __expf(acc[i][j] - m);
    for (int o = 8; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      z += __shfl_xor_sync(0xffffffffu, z, o);
    }
    if (row < n) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v0 + 4 * tx + j == r.target[row]) zt[row] = acc[i][j];
      if (tx == 0) {
        float* o = part + (long long)blockIdx.x * 3 * n_ld + row;
        o[0] = m;
        o[n_ld] = s;
        o[2 * n_ld] = z;
      }
    }
  }
}

__global__ void __launch_bounds__(256) ce_merge_kernel(CeRows r, const float* part, const float* zt, long long n_ld, int slots, int vocab, float smoothing, float* row_loss,
                                                       float* each) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= *r.count) return;
  float m = -INFINITY, s = 0.0f, z = 0.0f;
  for (int k = 0; k < slots; ++k) m = fmaxf(m, part[(long long)k * 3 * n_ld + i]);
  for (int k = 0; k < slots; ++k) {
    s += part[((long long)k * 3 + 1) * n_ld + i] * expf(part[(long long)k * 3 * n_ld + i] - m);
    z += part[((long long)k * 3 + 2) * n_ld + i];
  }
  const float lse = m + logf(s);
  r.lse[i] = lse;
  const float loss = r.target[i] < 0 ? NAN : lse - (1.0f - smoothing) * zt[i] - smoothing / vocab * z;
  row_loss[i] = loss;
  if (each != nullptr) each[r.index[i]] = loss;
}

__global__ void __launch_bounds__(256) ce_total_kernel(CeRows r, const float* row_loss, int reduce, float* loss) {
  __shared__ double s[256];
  double v = 0.0;
  for (int i = threadIdx.x; i < *r.count; i += 256) v += (double)row_loss[i];
  s[threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 256; ++i) v += s[i];
    *loss = (float)(reduce == CE_MEAN ? v / (double)*r.count : v);
  }
}

struct CeUp {           // u_i
  const float* up;
  int reduce;
};
__device__ __forceinline__ float ce_weight(const CeUp& u, const CeRows& r, int i) {
  const float g = u.reduce == CE_NONE ? u.up[r.index[i]] : u.reduce == CE_MEAN ? u.up[0] / (float)*r.count : u.up[0];
  return r.target[i] < 0 ? NAN : g;
}

template <typename T>
__global__ void __launch_bounds__(kCeThreads) ce_dz_kernel(CeHead<T> p, CeRows r, CeUp u, float smoothing, int c0, int width, float* dz) {
  __shared__ float sa[kCeK][kCeTile + 4], sb[kCeK][kCeTile + 4];
  const int n = *r.count, r0 = blockIdx.y * kCeTile, v0 = c0 + blockIdx.x * kCeTile, end = min(p.vocab, c0 + width);
  if (r0 >= n) return;
  float acc[4][4] = {};
  ce_tile([&](int m, int k) { return r0 + m < n ? ce_f32(p.h[(long long)r.index[r0 + m] * p.ldh + k]) : 0.0f; },
          [&](int m, int k) { return v0 + m < end ? ce_f32(p.w[(long long)(v0 + m) * p.ldw + k]) : 0.0f; }, p.hidden, acc, sa, sb);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + 4 * ty + i;
    if (row >= n) continue;
    const float g = ce_weight(u, r, row), lse = r.lse[row];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int v = v0 + 4 * tx + j;
      if (v < end) dz[(long long)row * width + v - c0] = g * (expf(acc[i][j] - lse) - (v == r.target[row] ? 1.0f - smoothing : 0.0f) - smoothing / p.vocab);
    }
  }
}

// dh [N][D] f32 += dz W of one piece (the list's order)
template <typename T>
__global__ void __launch_bounds__(kCeThreads) ce_dh_kernel(CeHead<T> p, CeRows r, const float* dz, int c0, int width, int first, float* dh) {
  __shared__ float sa[kCeK][kCeTile + 4], sb[kCeK][kCeTile + 4];
  const int n = *r.count, r0 = blockIdx.y * kCeTile, d0 = blockIdx.x * kCeTile, k = min(width, p.vocab - c0);
  if (r0 >= n) return;
  float acc[4][4] = {};
  ce_tile([&](int m, int v) { return r0 + m < n ? dz[(long long)(r0 + m) * width + v] : 0.0f; },
          [&](int m, int v) { return d0 + m < p.hidden ? ce_f32(p.w[(long long)(c0 + v) * p.ldw + d0 + m]) : 0.0f; }, k, acc, sa, sb);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (r0 + 4 * ty + i < n && d0 + 4 * tx + j < p.hidden) {
        float* o = dh + (long long)(r0 + 4 * ty + i) * p.hidden + d0 + 4 * tx + j;
        *o = first ? acc[i][j] : *o + acc[i][j];
      }
}

template <typename T>
__global__ void __launch_bounds__(kCeThreads) ce_dw_kernel(CeHead<T> p, CeRows r, const float* dz, int c0, int width, T* dw) {
  __shared__ float sa[kCeK][kCeTile + 4], sb[kCeK][kCeTile + 4];
  const int n = *r.count, m0 = blockIdx.y * kCeTile, d0 = blockIdx.x * kCeTile, rows = min(width, p.vocab - c0);
  float acc[4][4] = {};
  ce_tile([&](int m, int i) { return m0 + m < rows ? dz[(long long)i * width + m0 + m] : 0.0f; },
          [&](int m, int i) { return d0 + m < p.hidden ? ce_f32(p.h[(long long)r.index[i] * p.ldh + d0 + m]) : 0.0f; }, n, acc, sa, sb);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (m0 + 4 * ty + i < rows && d0 + 4 * tx + j < p.hidden) ce_put(dw + (long long)(c0 + m0 + 4 * ty + i) * p.hidden + d0 + 4 * tx + j, acc[i][j]);
}

// rows of dh to their places; the others are cleared before
template <typename T>
__global__ void __launch_bounds__(256) ce_scatter_kernel(CeRows r, const float* dh, int hidden, T* out) {
  const int i = blockIdx.x;
  if (i >= *r.count) return;
  for (int k = threadIdx.x; k < hidden; k += 256) ce_put(out + (long long)r.index[i] * hidden + k, dh[(long long)i * hidden + k]);
}

struct CeArgs {
  const void *hidden, *weight;
  const long long* targets;
  long long ldh, ldw, ignore;
  int rows, vocab, width, type, reduce;
  float smoothing;
  CeRows live;
  float* loss;
  const float* up;
  void *dhidden, *dweight;
  uint8_t* ws;
  long long ws_bytes;
};

static long long ce_piece(const CeArgs& a) {      // vocabulary rows of a piece of dz
  const long long most = (1ll << 28) / a.rows / kCeTile * kCeTile;
  return most < kCeTile ? kCeTile : most > a.vocab ? a.vocab : most;
}
static int ce_slots(const CeArgs& a) { return (a.vocab + kCeTile - 1) / kCeTile; }
static long long ce_forward_bytes(const CeArgs& a) { return 4ll * a.rows * (3ll * ce_slots(a) + 2); }
static long long ce_backward_bytes(const CeArgs& a) { return 4ll * a.rows * (ce_piece(a) + a.width); }

template <typename T>
static int ce_forward(const CeArgs& a, cudaStream_t st) {
  float *part = (float*)a.ws, *zt = part + 3ll * ce_slots(a) * a.rows, *row_loss = zt + a.rows;
  const CeHead<T> p = {(const T*)a.hidden, (const T*)a.weight, a.ldh, a.ldw, a.vocab, a.width};
  ce_rows_kernel<<<1, 1024, 0, st>>>(a.targets, a.rows, a.vocab, a.ignore, a.live, a.reduce == CE_NONE ? a.loss : nullptr);
  ce_lse_kernel<T><<<dim3(ce_slots(a), (a.rows + kCeTile - 1) / kCeTile), kCeThreads, 0, st>>>(p, a.live, part, zt, a.rows);
  ce_merge_kernel<<<(a.rows + 255) / 256, 256, 0, st>>>(a.live, part, zt, a.rows, ce_slots(a), a.vocab, a.smoothing, row_loss,
                                                       a.reduce == CE_NONE ? a.loss : nullptr);
  if (a.reduce != CE_NONE) ce_total_kernel<<<1, 256, 0, st>>>(a.live, row_loss, a.reduce, a.loss);
  return launch_status();
}

template <typename T>
static int ce_backward(const CeArgs& a, cudaStream_t st) {
  const int piece = (int)ce_piece(a), row_tiles = (a.rows + kCeTile - 1) / kCeTile, d_tiles = (a.width + kCeTile - 1) / kCeTile;
  float *dz = (float*)a.ws, *dh = dz + (long long)a.rows * piece;
  const CeHead<T> p = {(const T*)a.hidden, (const T*)a.weight, a.ldh, a.ldw, a.vocab, a.width};
  const CeUp u = {a.up, a.reduce};
  for (int c0 = 0; c0 < a.vocab; c0 += piece) {
    const int tiles = (piece + kCeTile - 1) / kCeTile;
    ce_dz_kernel<T><<<dim3(tiles, row_tiles), kCeThreads, 0, st>>>(p, a.live, u, a.smoothing, c0, piece, dz);
    if (a.dhidden != nullptr) ce_dh_kernel<T><<<dim3(d_tiles, row_tiles), kCeThreads, 0, st>>>(p, a.live, dz, c0, piece, c0 == 0, dh);
    if (a.dweight != nullptr) ce_dw_kernel<T><<<dim3(d_tiles, tiles), kCeThreads, 0, st>>>(p, a.live, dz, c0, piece, (T*)a.dweight);
  }
  if (a.dhidden != nullptr) {
    if (cudaMemsetAsync(a.dhidden, 0, (size_t)a.rows * a.width * sizeof(T), st) != cudaSuccess) return BONSAI_CUDA_LAUNCH_FAILED;
    ce_scatter_kernel<T><<<a.rows, 256, 0, st>>>(a.live, dh, a.width, (T*)a.dhidden);
  }
  return launch_status();
}

static bool ce_good(const CeArgs& a) {
  return a.rows >= 1 && a.vocab >= 1 && a.width >= 1 && a.type >= CE_F32 && a.type <= CE_BF16 && a.reduce >= CE_MEAN && a.reduce <= CE_NONE;
}

}  // namespace bonsai

extern "C" {

long long bonsai_ce_workspace(int rows, int vocab, int width, int type, int backward, int want_hidden, int want_weight) {
  using namespace bonsai;
  CeArgs a = {};
  a.rows = rows; a.vocab = vocab; a.width = width; a.type = type;
  (void)want_hidden; (void)want_weight;
  return ce_good(a) ? (backward ? ce_backward_bytes(a) : ce_forward_bytes(a)) : -1;
}

// hidden [rows][ldh], weight [vocab][ldw] of one type (0 f32, 1 f16, 2 bf16), targets [rows].  live: 4 + 2 rows int32, lse: rows f32; both are
// filled here and read by the backward call.  loss: one f32, or one for each row (reduce 2).
int bonsai_ce_forward(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* targets, int rows, int vocab, int width,
                      int type, long long ignore, int reduce, float smoothing, int* live, float* lse, float* loss, void* ws, long long ws_bytes,
                      cudaStream_t st) {
  using namespace bonsai;
  CeArgs a = {};
  a.hidden = hidden; a.weight = weight; a.targets = targets; a.ldh = ldh; a.ldw = ldw; a.ignore = ignore;
  a.rows = rows; a.vocab = vocab; a.width = width; a.type = type; a.reduce = reduce; a.smoothing = smoothing;
  a.live = CeRows{live, live + 4, live + 4 + rows, lse};
  a.loss = loss; a.ws = (uint8_t*)ws; a.ws_bytes = ws_bytes;
  if (!ce_good(a) || hidden == nullptr || weight == nullptr || targets == nullptr || live == nullptr || lse == nullptr || loss == nullptr ||
      ldh < width || ldw < width || ws == nullptr || ws_bytes < ce_forward_bytes(a))
    return BONSAI_CUDA_BAD_ARG;
  return type == CE_F32 ? ce_forward<float>(a, st) : type == CE_F16 ? ce_forward<__half>(a, st) : ce_forward<__nv_bfloat16>(a, st);
}

// up: d loss, one f32 or one for each row.  dhidden [rows][width], dweight [vocab][width] of the inputs' type; null: not wanted.
int bonsai_ce_backward(const void* hidden, long long ldh, const void* weight, long long ldw, int rows, int vocab, int width, int type, int reduce,
                       float smoothing, int* live, float* lse, const float* up, void* dhidden, void* dweight, void* ws, long long ws_bytes,
                       cudaStream_t st) {
  using namespace bonsai;
  CeArgs a = {};
  a.hidden = hidden; a.weight = weight; a.ldh = ldh; a.ldw = ldw;
  a.rows = rows; a.vocab = vocab; a.width = width; a.type = type; a.reduce = reduce; a.smoothing = smoothing;
  a.live = CeRows{live, live + 4, live + 4 + rows, lse};
  a.up = up; a.dhidden = dhidden; a.dweight = dweight; a.ws = (uint8_t*)ws; a.ws_bytes = ws_bytes;
  if (!ce_good(a) || hidden == nullptr || weight == nullptr || live == nullptr || lse == nullptr || up == nullptr || ldh < width || ldw < width ||
      ws == nullptr || ws_bytes < ce_backward_bytes(a))
    return BONSAI_CUDA_BAD_ARG;
  return type == CE_F32 ? ce_backward<float>(a, st) : type == CE_F16 ? ce_backward<__half>(a, st) : ce_backward<__nv_bfloat16>(a, st);
}

}  // extern "C"
