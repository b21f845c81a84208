// Dropout over rows of d values, with a mask that is made from the counter of philox.cuh and never stored:
//
//   y = x * 65536 / steps where the value's 16 random bits are below steps, else 0 (whatever x holds there)
//
// The backward pass is the same kernel over the gradient.  A thread takes eight neighbouring values, one counter, and walks on by the
// grid; its place (row, group of eight) is advanced by a quotient and a remainder from the host, without a division.
//
// Some 90 instructions go into eight values (ten rounds of two wide multiplications), about as long as 16-bit values take from memory: 8192 x 4096 bf16 (134 MB)
// in 26.5 us, 5.1 TB/s.  Eight blocks an SM of which six fit are faster than six (30 us): the last ones fill in where others end.  The next kernel is not let
// in early: its blocks would take places of this one's (333 x 2049 f32, there and back: 21 us, 11 without).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "philox.cuh"

namespace bonsai {

constexpr int kDropThreads = 256;

template <typename T> struct Eight;            // eight neighbouring values in registers
template <> struct Eight<float> { float4 a, b; };
template <> struct Eight<__half> { uint4 a; };
template <> struct Eight<__nv_bfloat16> { uint4 a; };

__device__ __forceinline__ void unpack(const Eight<float>& v, float* f) {
  f[0] = v.a.x; f[1] = v.a.y; f[2] = v.a.z; f[3] = v.a.w; f[4] = v.b.x; f[5] = v.b.y; f[6] = v.b.z; f[7] = v.b.w;
}
__device__ __forceinline__ void unpack(const Eight<__half>& v, float* f) {
  const unsigned w[4] = {v.a.x, v.a.y, v.a.z, v.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void unpack(const Eight<__nv_bfloat16>& v, float* f) {
  const unsigned w[4] = {v.a.x, v.a.y, v.a.z, v.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void pack(Eight<float>& v, const float* f) { v.a = make_float4(f[0], f[1], f[2], f[3]); v.b = make_float4(f[4], f[5], f[6], f[7]); }
__device__ __forceinline__ void pack(Eight<__half>& v, const float* f) {
  __half2 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  v.a = *reinterpret_cast<const uint4*>(h);
}
__device__ __forceinline__ void pack(Eight<__nv_bfloat16>& v, const float* f) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  v.a = *reinterpret_cast<const uint4*>(h);
}

__device__ __forceinline__ void mask(Eight<float>& v, const uint4& words, unsigned limit) {
  v.a.x = dropout_keeps(words, 0, limit) ? v.a.x : 0.0f; v.a.y = dropout_keeps(words, 1, limit) ? v.a.y : 0.0f;
  v.a.z = dropout_keeps(words, 2, limit) ? v.a.z : 0.0f; v.a.w = dropout_keeps(words, 3, limit) ? v.a.w : 0.0f;
  v.b.x = dropout_keeps(words, 4, limit) ? v.b.x : 0.0f; v.b.y = dropout_keeps(words, 5, limit) ? v.b.y : 0.0f;
  v.b.z = dropout_keeps(words, 6, limit) ? v.b.z : 0.0f; v.b.w = dropout_keeps(words, 7, limit) ? v.b.w : 0.0f;
}
template <typename T>
__device__ __forceinline__ void mask(Eight<T>& v, const uint4& words, unsigned limit) {
  v.a.x = dropout_pair(v.a.x, words.x, limit); v.a.y = dropout_pair(v.a.y, words.y, limit);
  v.a.z = dropout_pair(v.a.z, words.z, limit); v.a.w = dropout_pair(v.a.w, words.w, limit);
}

template <typename T> __device__ __forceinline__ float one_of(T v);
template <> __device__ __forceinline__ float one_of(float v) { return v; }
template <> __device__ __forceinline__ float one_of(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float one_of(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

struct DropPlace {
  long long row;
  unsigned group;
};

// WHOLE: rows of whole eights that begin at multiples of 16 bytes.  A thread has U counters in flight.
template <typename T, bool WHOLE, int U>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const T* __restrict__ x, long long ldx, T* __restrict__ y, long long rows, unsigned d,
                                                               unsigned groups, long long step_rows, unsigned step_groups, DropoutRule rule) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint2 key = philox_key(rule);
  const long long first = (long long)blockIdx.x * kDropThreads + threadIdx.x;
  DropPlace at = {first / groups, (unsigned)(first % groups)};
  auto next = [&](DropPlace p) {
    p.group += step_groups;
    const bool over = p.group >= groups;
    p.group -= over ? groups : 0u;
    p.row += step_rows + (over ? 1 : 0);
    return p;
  };
  while (at.row < rows) {
    DropPlace p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) { p[u] = at; at = next(at); }
    if (WHOLE) {
      Eight<T> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p[u].row < rows) v[u] = *reinterpret_cast<const Eight<T>*>(x + p[u].row * ldx + 8ll * p[u].group);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint4 words = dropout_words(p[u].group, p[u].row, key);
        if (p[u].row < rows) {
          float f[8];
          unpack(v[u], f);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = f[j] * rule.share;
          pack(v[u], f);
          mask(v[u], words, rule.limit);
          *reinterpret_cast<Eight<T>*>(y + p[u].row * (long long)d + 8ll * p[u].group) = v[u];
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p[u].row >= rows) continue;
        const uint4 words = dropout_words(p[u].group, p[u].row, key);
        const unsigned c = 8u * p[u].group, n = d - c < 8u ? d - c : 8u;
        const T* from = x + p[u].row * ldx + c;
        T* to = y + p[u].row * (long long)d + c;
#pragma unroll
        for (unsigned j = 0; j < 8; ++j)
          if (j < n) put(to + j, dropout_keeps(words, j, rule.limit) ? one_of<T>(from[j]) * rule.share : 0.0f);
      }
    }
  }
}

template <typename T>
static cudaError_t dropout_launch(const T* x, long long ldx, T* y, long long rows, unsigned d, const DropoutRule& rule, cudaStream_t st) {
  constexpr int kMost = 148 * 8;
  const unsigned groups = (d + 7) / 8;
  const long long total = rows * groups, want = (total + kDropThreads - 1) / kDropThreads;
  const int blocks = (int)(want < kMost ? want : kMost);
  const long long step = (long long)blocks * kDropThreads;
  const bool whole = d % 8 == 0 && (ldx * sizeof(T)) % 16 == 0 && ((uintptr_t)x | (uintptr_t)y) % 16 == 0;
  const long long step_rows = step / groups;
  const unsigned step_groups = (unsigned)(step % groups);
  return whole ? launch_pdl(dropout_kernel<T, true, 2>, dim3(blocks), dim3(kDropThreads), 0, st, x, ldx, y, rows, d, groups, step_rows, step_groups, rule)
               : launch_pdl(dropout_kernel<T, false, 2>, dim3(blocks), dim3(kDropThreads), 0, st, x, ldx, y, rows, d, groups, step_rows, step_groups, rule);
}

}  // namespace bonsai

extern "C" {

// x: rows of d values (type 0 f32, 1 f16, 2 bf16) at distances of ldx; y: the same rows side by side.  steps: of 65536 values that many
// stay, less than all.  seed_dev, where given, holds the seed.
int bonsai_dropout(const void* x, long long ldx, void* y, long long rows, long long d, int type, unsigned long long seed, const long long* seed_dev,
                   int steps, cudaStream_t st) {
  using namespace bonsai;
  if (x == nullptr || y == nullptr || rows < 1 || d < 1 || d >= 1ll << 31 || rows >= 1ll << 40 || rows > (1ll << 62) / d || type < 0 || type > 2 ||
      steps < 0 || steps > 65535)
    return BONSAI_CUDA_BAD_ARG;
  const DropoutRule rule = dropout_rule(seed, seed_dev, steps);
  cudaError_t e;
  if (type == 0) e = dropout_launch((const float*)x, ldx, (float*)y, rows, (unsigned)d, rule, st);
  else if (type == 1) e = dropout_launch((const __half*)x, ldx, (__half*)y, rows, (unsigned)d, rule, st);
  else e = dropout_launch((const __nv_bfloat16*)x, ldx, (__nv_bfloat16*)y, rows, (unsigned)d, rule, st);
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

}  // extern "C"
