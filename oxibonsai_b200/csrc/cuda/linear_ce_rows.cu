// The loss of an f32 head and its gradients for up to 24 live rows, on the CUDA cores.
//
// Here the head's bytes are all there is to it, and the tensor-core path has to copy them into three bfloat16 parts first: 4 + 6 bytes moved for each value
// before the first product reads 6.  These kernels read the head as it lies, in any alignment, and multiply in f32; a value's multiplications, one
// for each row, take less time than its bytes.  One row of 4096 x 151 936: 429 us for the whole call (5.8 TB/s), 2200 by parts.  From 17 rows on the tokens
// come in two launches of 16, which read the head twice: 24 rows of 4096 x 151 936 1.42 ms (its bytes: 0.38), 2.25 by parts, 17 rows of 2048 x 50 000
// with both gradients 1.11 and 1.32; with 32 rows the two are even.  With 16-bit types the tensor cores need no copies and are faster from one row on.
//   ce_few_z_kernel   z = h W^T: a warp takes 64 / TN rows of the head against TN tokens, its lanes share the width; then the loss's running
//                     maxima and sums (in registers, over all rows a warp takes) or dz = u (exp(z - lse) - q), f32
//   ce_few_h_kernel   dh = dz W: a thread has four columns of dh in registers and walks down the head's rows; ce_few_join_kernel adds the parts
//   ce_few_w_kernel   dW = dz^T h: four columns of h in registers, down the rows of dW
// dh and dW in one walk would read nothing less (dW does not need the head) and took 200 registers a thread, half of the threads and twice the time.
#include "linear_ce.cuh"

namespace bonsai {

constexpr int kFewBlocks = 148;
constexpr int kGradThreads = 256, kGradRows = 64;

// Four values of a row: neighbours from column c (WIDE: aligned, and inside the row as a whole or not at all), or columns c, c + step, c + 2 step,
// c + 3 step.  STREAM: of the head, which nothing reads again soon enough to keep it in L1.
template <bool WIDE, bool STREAM>
__device__ __forceinline__ void few_load(const float* row, int c, int step, int width, float* v) {
  if constexpr (!WIDE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c + i * step < width ? row[c + i * step] : 0.0f;
  } else if (c >= width) {
    v[0] = v[1] = v[2] = v[3] = 0.0f;
  } else if (STREAM) {
    asm volatile("ld.global.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "l"(row + c));
  } else {
    const float4 q = *reinterpret_cast<const float4*>(row + c);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  }
}

template <bool WIDE>
__device__ __forceinline__ void few_store(float* row, int c, int step, int width, const float* v) {
  if constexpr (!WIDE) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i * step < width) row[c + i * step] = v[i];
  } else if (c < width) {
    *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
  }
}

// Registers against warps: with 16 tokens eight warps of 255 registers beat sixteen of 128 (2048 x 50 000: 180 us, 238), with 8 it is the other way
// (1344 x 71 426: 108 us, 91); with 4 there is room for two steps of loads in flight (4096 x 151 936: 418 us, 436 for one).
__host__ __device__ constexpr int few_threads(int tn) { return tn == 16 ? 256 : 512; }

template <bool WIDE, int TN, bool DZ>
__global__ void __launch_bounds__(few_threads(TN), 1) ce_few_z_kernel(const CeFewArgs p) {
  constexpr int R = TN < 8 ? 8 : 64 / TN, NV = R * TN, J = NV / 32;          // rows of the head, sums of a warp and of a lane
  constexpr int kFewWarps = few_threads(TN) / 32, kSteps = TN < 8 ? 2 : 1;
  __shared__ float block[3][DZ ? 1 : kFewWarps][TN];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = blockIdx.x * kFewWarps + (threadIdx.x >> 5), warps = gridDim.x * kFewWarps, all = *p.rows.count, n = all - p.first;
  if (n <= 0) return;
  // this lane's sums after the reduction: row (J lane + j) / TN, token (J lane + j) % TN
  const int t0 = (J * lane) % TN, r0 = J * lane / TN;
  int target[J];
  float lse2[J], f[J], top[J], sum[J], sum_z[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int t = t0 + j;
    const bool ok = t < n;
    target[j] = ok ? p.rows.target[t] : -1;
    top[j] = -INFINITY;
    sum[j] = sum_z[j] = 0.0f;
    lse2[j] = DZ && ok ? p.rows.lse2[t] : 0.0f;
    f[j] = DZ && ok ? ce_up_factor(p.up, p.rows, t) * ce_up_scale(p.up, all) : 0.0f;
  }
  const float even = p.smoothing / (float)p.vocab;
  const int begin = (int)((long long)p.vocab * warp / warps), end = (int)((long long)p.vocab * (warp + 1) / warps);
  for (int v0 = begin; v0 < end; v0 += R) {
    const float* w[R];
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = (const float*)p.weight + (long long)min(v0 + r, end - 1) * p.ldw;
    float acc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = 0.0f;
#pragma unroll kSteps
    for (int k0 = 0; k0 < p.width; k0 += 128) {
      const int k = k0 + (WIDE ? 4 * lane : lane);
      float a[R][4];
#pragma unroll
      for (int r = 0; r < R; ++r) few_load<WIDE, true>(w[r], k, 32, p.width, a[r]);
#pragma unroll
      for (int t = 0; t < TN; ++t) {
        float x[4];
        few_load<WIDE, false>((const float*)p.x + t * p.ldx, k, 32, p.width, x);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r * TN + t] = fmaf(a[r][i], x[i], acc[r * TN + t]);
      }
    }
    // NV sums over 32 lanes: each step sends half of the values and keeps the other half
#pragma unroll
    for (int step = 16; step >= 1; step >>= 1) {
      const bool up = lane & step;
#pragma unroll
      for (int i = 0; i < step * J; ++i) {
        const float give = up ? acc[i] : acc[i + step * J], keep = up ? acc[i + step * J] : acc[i];
        acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, step);
      }
    }
    const int v = v0 + r0;
    if (v < end) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float z = acc[j];
        const int t = t0 + j;
        if (DZ) {
          if (t < n) p.dz[t * p.ldz + v] = f[j] * (ce_exp2(fmaf(z, kCeLog2e, -lse2[j])) - even - (v == target[j] ? 1.0f - p.smoothing : 0.0f));
        } else {
          if (v == target[j]) p.at_target[t] = z;
          const float m = fmaxf(top[j], z * kCeLog2e), ref = m == -INFINITY ? 0.0f : m;
          sum[j] = sum[j] * ce_exp2(top[j] - ref) + ce_exp2(fmaf(z, kCeLog2e, -ref));
          top[j] = m;
          sum_z[j] += z;
        }
      }
    }
  }
  if (!DZ) {          // the lanes of a token, then the warps of the block
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float m = top[j], s = sum[j], z = sum_z[j];
#pragma unroll
      for (int o = 16; o >= TN / J; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o), both = fmaxf(m, m2);
        const float ref = both == -INFINITY ? 0.0f : both;
        s = s * ce_exp2(m - ref) + s2 * ce_exp2(m2 - ref);
        z += __shfl_xor_sync(0xffffffffu, z, o);
        m = both;
      }
      if (lane < TN / J) {
        const int w = threadIdx.x >> 5, t = t0 + j;
        block[0][w][t] = m;
        block[1][w][t] = s;
        block[2][w][t] = z;
      }
    }
    __syncthreads();
    const int t = threadIdx.x;
    if (t < TN && t < n) {
      float m = -INFINITY, s = 0.0f, z = 0.0f;
      for (int w = 0; w < kFewWarps; ++w) m = fmaxf(m, block[0][w][t]);
      const float ref = m == -INFINITY ? 0.0f : m;
      for (int w = 0; w < kFewWarps; ++w) {
        s += block[1][w][t] * ce_exp2(block[0][w][t] - ref);
        z += block[2][w][t];
      }
      const long long at = blockIdx.x * p.ldn + t;
      p.part_m[at] = m;
      p.part_s[at] = s;
      if (p.smoothing != 0.0f) p.part_z[at] = z;
    }
  }
}

// Threads of a block side by side along the width, four columns each; the others of its 256 take other rows of the head.
__host__ __device__ inline int few_across(int width) {
  int c = 32;
  while (c < kGradThreads && c * 4 < width) c *= 2;
  return c;
}

// What the two kernels below have in common: a block's columns and rows, and its tokens' dz of 64 rows at a time in shared memory.
template <int TN, typename Row>
__device__ __forceinline__ void few_rows(const CeFewArgs& p, int n, Row row) {
  __shared__ __align__(16) float dz[kGradRows][TN];
  const int begin = (int)((long long)p.vocab * blockIdx.y / gridDim.y), end = (int)((long long)p.vocab * (blockIdx.y + 1) / gridDim.y);
  for (int v0 = begin; v0 < end; v0 += kGradRows) {
    __syncthreads();
    for (int i = threadIdx.x; i < kGradRows * TN; i += kGradThreads) {
      const int t = i / kGradRows, v = i % kGradRows;
      dz[v][t] = t < n && v0 + v < end ? p.dz[t * p.ldz + v0 + v] : 0.0f;
    }
    __syncthreads();
    row(v0, min(kGradRows, end - v0), dz);
  }
}

template <bool WIDE, int TN>
__global__ void __launch_bounds__(kGradThreads, 2) ce_few_h_kernel(const CeFewArgs p) {
  constexpr int U = 4;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = *p.rows.count - p.first, across = few_across(p.width), down = kGradThreads / across, x = threadIdx.x % across, y = threadIdx.x / across;
  const int c = blockIdx.x * across * 4 + (WIDE ? 4 * x : x);
  if (n <= 0) return;
  float acc[TN][4];
#pragma unroll
  for (int t = 0; t < TN; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.0f;
  few_rows<TN>(p, n, [&](int v0, int rows, float (*dz)[TN]) {
    for (int v = y; v < rows; v += down * U) {
      float w[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) few_load<WIDE, true>((const float*)p.weight + (long long)(v0 + min(v + u * down, rows - 1)) * p.ldw, c, across, p.width, w[u]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v + u * down < rows) {
#pragma unroll
          for (int t = 0; t < TN; t += 4) {
            const float4 q = *reinterpret_cast<const float4*>(&dz[v + u * down][t]);
            const float e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[t + k][i] = fmaf(e[k], w[u][i], acc[t + k][i]);
          }
        }
      }
    }
  });
#pragma unroll
  for (int t = 0; t < TN; ++t)
    if (t < n) few_store<false>(p.part + ((long long)(blockIdx.y * down + y) * p.tokens + t) * p.width, c, WIDE ? 1 : across, p.width, acc[t]);
}

template <bool WIDE, int TN>
__global__ void __launch_bounds__(kGradThreads, 2) ce_few_w_kernel(const CeFewArgs p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = *p.rows.count - p.first, across = few_across(p.width), down = kGradThreads / across, x = threadIdx.x % across, y = threadIdx.x / across;
  const int c = blockIdx.x * across * 4 + (WIDE ? 4 * x : x);
  if (p.first > 0 && n <= 0) return;
  float h[TN][4];
#pragma unroll
  for (int t = 0; t < TN; ++t) {
    h[t][0] = h[t][1] = h[t][2] = h[t][3] = 0.0f;
    if (t < n) few_load<WIDE, false>((const float*)p.x + t * p.ldx, c, across, p.width, h[t]);
  }
  few_rows<TN>(p, n, [&](int v0, int rows, float (*dz)[TN]) {
#pragma unroll 2
    for (int v = y; v < rows; v += down) {
      float* o = (float*)p.dweight + (long long)(v0 + v) * p.width;
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (p.first > 0) few_load<WIDE, false>(o, c, across, p.width, s);          // the earlier tokens' sums
#pragma unroll
      for (int t = 0; t < TN; t += 4) {
        const float4 q = *reinterpret_cast<const float4*>(&dz[v][t]);
        const float e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[i] = fmaf(e[k], h[t + k][i], s[i]);
      }
      few_store<WIDE>(o, c, across, p.width, s);
    }
  });
}

// dh: 32 columns of a row, eight threads for the parts of each
__global__ void __launch_bounds__(256) ce_few_join_kernel(const CeFewArgs p, int slots) {
  __shared__ float s[8][33];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, row = blockIdx.y, at = p.rows.place[row];
  float v = 0.0f;
  if (at >= 0 && c < p.width) {
#pragma unroll 8
    for (int i = k; i < slots; i += 8) v += p.part[((long long)i * p.tokens + at) * p.width + c];
  }
  s[k][lane] = v;
  __syncthreads();
  if (k == 0 && c < p.width) {
    for (int i = 1; i < 8; ++i) v += s[i][lane];
    ((float*)p.dhidden)[(long long)row * p.width + c] = v;
  }
}

static bool few_wide(const CeFewArgs& a) { return a.width % 4 == 0 && a.ldw % 4 == 0 && (reinterpret_cast<uintptr_t>(a.weight) & 15) == 0; }

// Blocks down the head: four for each SM over the column groups, their threads' parts at most 512
static int few_blocks(int width) {
  const int across = few_across(width), groups = (width + across * 4 - 1) / (across * 4), most = 512 / (kGradThreads / across), blocks = kFewBlocks * 4 / groups;
  return blocks < 1 ? 1 : blocks < most ? blocks : most;
}

int ce_few_slots(int width) { return few_blocks(width) * (kGradThreads / few_across(width)); }
int ce_few_loss_slots() { return kFewBlocks; }

// The arguments for tokens `first` and on: every list and matrix of tokens moved up.
static CeFewArgs few_from(CeFewArgs a, int first) {
  a.first = first;
  a.tokens_left = a.tokens - first;
  a.rows.index += first; a.rows.target += first; a.rows.lse2 += first;
  a.x = (const float*)a.x + first * a.ldx;
  if (a.part_m != nullptr) { a.part_m += first; a.part_s += first; a.part_z += first; a.at_target += first; }
  if (a.dz != nullptr) { a.dz += first * a.ldz; a.part += (long long)first * a.width; }
  return a;
}

template <bool WIDE, bool DZ>
static cudaError_t few_z(const CeFewArgs& a, cudaStream_t st) {
  const dim3 grid(kFewBlocks);
  if (a.tokens_left <= 4) return launch_pdl(ce_few_z_kernel<WIDE, 4, DZ>, grid, dim3(few_threads(4)), 0, st, a);
  if (a.tokens_left <= 8) return launch_pdl(ce_few_z_kernel<WIDE, 8, DZ>, grid, dim3(few_threads(8)), 0, st, a);
  return launch_pdl(ce_few_z_kernel<WIDE, 16, DZ>, grid, dim3(few_threads(16)), 0, st, a);
}

template <bool WIDE, int TN>
static cudaError_t few_g(const CeFewArgs& a, cudaStream_t st) {
  const int across = few_across(a.width);
  const dim3 grid((a.width + across * 4 - 1) / (across * 4), few_blocks(a.width)), block(kGradThreads);
  cudaError_t e = cudaSuccess;
  if (a.dhidden != nullptr) e = launch_pdl(ce_few_h_kernel<WIDE, TN>, grid, block, 0, st, a);
  if (e == cudaSuccess && a.dweight != nullptr) e = launch_pdl(ce_few_w_kernel<WIDE, TN>, grid, block, 0, st, a);
  return e;
}

template <bool WIDE>
static cudaError_t few_gradients(const CeFewArgs& a, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  for (int first = 0; first < a.tokens && e == cudaSuccess; first += 16) {
    const CeFewArgs b = few_from(a, first);
    e = few_z<WIDE, true>(b, st);
    if (e == cudaSuccess) e = b.tokens_left <= 8 ? few_g<WIDE, 8>(b, st) : few_g<WIDE, 16>(b, st);
  }
  if (e == cudaSuccess && a.dhidden != nullptr) e = launch_pdl(ce_few_join_kernel, dim3((a.width + 31) / 32, a.row_count), dim3(256), 0, st, a, ce_few_slots(a.width));
  return e;
}

cudaError_t ce_few_loss(const CeFewArgs& a, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  for (int first = 0; first < a.tokens && e == cudaSuccess; first += 16)
    e = few_wide(a) ? few_z<true, false>(few_from(a, first), st) : few_z<false, false>(few_from(a, first), st);
  return e;
}

cudaError_t ce_few_gradients(const CeFewArgs& a, cudaStream_t st) { return few_wide(a) ? few_gradients<true>(a, st) : few_gradients<false>(a, st); }

}  // namespace bonsai
