// Global norm, clipping and Adam steps over many tensors, a few launches whatever their number.
//
//   norm   s = sqrt(sum over all tensors of g^2)
//   clip   out = c g,  c = max / (s + 1e-6) where s > max > 0, else 1
//   Adam   g' = c g (+ wd p);  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2;
//          p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// The tensors of one launch lie one behind another on a line of values that is cut into equal pieces, one for each block, so that 300
// adapters of 32 K values and one matrix of 100 M cost the same per byte.  Addresses and places come as kernel parameters: nothing is
// copied to the device, and a captured launch carries its own table.  Squares are added in f32 over eight neighbours and in f64 from
// there on; the partial sums of the blocks are added in one order by every block that needs the norm, so that there is no atomic, no
// counter to reset, and the same values give the same bits.  All three are bound by memory: a clipped AdamW step of 705 M bf16 parameters with f32
// moments moves 16.9 GB in 2.73 to 2.79 ms (6.1 TB/s), clipping 705 M bf16 gradients into f32 ones 5.6 GB in 0.94 ms (6.0 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace bonsai {

constexpr int kMtTensors = 512;        // tensors of one launch; larger sets take several
// Blocks of a launch: sets that take some tens of microseconds go in one wave (three blocks an SM, two of the Adam step), larger ones in pieces that
// even the SMs out (13 M f32, clipped: 29.7 us in one wave, 31.2 in 888 pieces; 705 M bf16 into f32: 948 and 932).
constexpr int kMtBlocksMax = 148 * 6, kMtWave = 148 * 3, kMtWaveAdam = 148 * 2;
constexpr long long kMtSmall = 1ll << 24;
constexpr int kMtThreads = 512;
enum MtType : unsigned char { MT_F32 = 0, MT_F16 = 1, MT_BF16 = 2 };

template <int NP>
struct MtTable {
  void* ptr[NP][kMtTensors];
  long long start[kMtTensors + 1];      // place on the line
  unsigned short first[kMtBlocksMax];   // tensor in which a block's piece begins
  unsigned char type[2][kMtTensors];
  int tensors;
  long long per_block;
};

template <typename T> __device__ __forceinline__ float mt_load(const void* p, long long i);
template <> __device__ __forceinline__ float mt_load<float>(const void* p, long long i) { return ((const float*)p)[i]; }
template <> __device__ __forceinline__ float mt_load<__half>(const void* p, long long i) { return __half2float(((const __half*)p)[i]); }
template <> __device__ __forceinline__ float mt_load<__nv_bfloat16>(const void* p, long long i) { return __bfloat162float(((const __nv_bfloat16*)p)[i]); }
template <typename T> __device__ __forceinline__ void mt_store(void* p, long long i, float v);
template <> __device__ __forceinline__ void mt_store<float>(void* p, long long i, float v) { ((float*)p)[i] = v; }
template <> __device__ __forceinline__ void mt_store<__half>(void* p, long long i, float v) { ((__half*)p)[i] = __float2half_rn(v); }
template <> __device__ __forceinline__ void mt_store<__nv_bfloat16>(void* p, long long i, float v) { ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v); }

// eight neighbouring values as one access of 16 (16-bit types) or 32 bytes
__device__ __forceinline__ void mt_load8(const float* p, float* v) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void mt_load8(const __half* p, float* v) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void mt_load8(const __nv_bfloat16* p, float* v) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void mt_store8(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]),
               "f"(v[7])
               : "memory");
}
__device__ __forceinline__ void mt_store8(__half* p, const float* v) {
  __half2 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}
__device__ __forceinline__ void mt_store8(__nv_bfloat16* p, const float* v) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}

template <typename T>
__device__ __forceinline__ bool mt_aligned(const T* p) { return (reinterpret_cast<uintptr_t>(p) & (8 * sizeof(T) - 1)) == 0; }

// Runs one(i) for the values before the first place where every pointer is aligned for eight and behind the last whole eight, and
// eights<n>(i, stride) for n eights at a time between; pointers that never line up go value by value.
template <int U, typename Lined, typename One, typename Eights>
__device__ __forceinline__ void mt_walk(long long lo, long long hi, Lined lined, One one, Eights eights) {
  const int t = threadIdx.x;
  int head = 0;
  while (head < 8 && !lined(lo + head)) ++head;
  const long long n8 = head < 8 && hi - lo > head ? (hi - lo - head) >> 3 : 0;
  if (n8 > 0) {
    if (t < head) one(lo + t);
    long long i = t;
    for (; i + (U - 1) * kMtThreads < n8; i += U * kMtThreads) eights(std::integral_constant<int, U>(), lo + head + 8 * i);
    for (; i < n8; i += kMtThreads) eights(std::integral_constant<int, 1>(), lo + head + 8 * i);
    for (long long k = lo + head + 8 * n8 + t; k < hi; k += kMtThreads) one(k);
  } else {
    for (long long i = lo + t; i < hi; i += kMtThreads) one(i);
  }
}

// Calls body(tensor, lo, hi) for the parts of tensors that this block's piece of the line covers.
template <int NP, typename Body>
__device__ __forceinline__ void mt_pieces(const MtTable<NP>& tb, Body body) {
  const long long end = tb.start[tb.tensors];
  const long long a = (long long)blockIdx.x * tb.per_block, b = a + tb.per_block < end ? a + tb.per_block : end;
  for (int i = tb.first[blockIdx.x]; i < tb.tensors && tb.start[i] < b; ++i) {
    const long long s = tb.start[i], e = tb.start[i + 1];
    const long long lo = (a > s ? a : s) - s, hi = (b < e ? b : e) - s;
    if (lo < hi) body(i, lo, hi);
  }
}

__device__ __forceinline__ double mt_block_sum(double v, double* s) {      // in every thread, added in one order
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < kMtThreads / 32; ++i) t += s[i];
  __syncthreads();
  return t;
}

template <typename T>
__device__ __forceinline__ double mt_squares(const void* g, long long lo, long long hi) {
  double acc = 0.0;
  const T* p = (const T*)g;
  mt_walk<4>(
      lo, hi, [&](long long i) { return mt_aligned(p + i); },
      [&](long long i) { const double x = (double)mt_load<T>(p, i); acc += x * x; },
      [&](auto count, long long i) {
        constexpr int N = decltype(count)::value;
        float x[N][8];
#pragma unroll
        for (int u = 0; u < N; ++u) mt_load8(p + i + u * 8ll * kMtThreads, x[u]);
#pragma unroll
        for (int u = 0; u < N; ++u) {
          float s = 0.0f;
#pragma unroll
          for (int k = 0; k < 8; ++k) s = fmaf(x[u][k], x[u][k], s);
          if (s > 1e-30f && s < 1e37f) {
            acc += (double)s;
          } else {                    // squares that leave the range of f32, zeros and NaN
#pragma unroll
            for (int k = 0; k < 8; ++k) acc += (double)x[u][k] * (double)x[u][k];
          }
        }
      });
  return acc;
}

// `step`, where given, counts this optimizer step before the kernel that reads it.
__global__ void __launch_bounds__(kMtThreads, 3) mt_norm_kernel(const __grid_constant__ MtTable<1> tb, double* partial, long long* step) {
  __shared__ double s[kMtThreads / 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (step != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *step += 1;
  double acc = 0.0;
  mt_pieces(tb, [&](int i, long long lo, long long hi) {
    const void* g = tb.ptr[0][i];
    switch (tb.type[0][i]) {
      case MT_F32: acc += mt_squares<float>(g, lo, hi); break;
      case MT_F16: acc += mt_squares<__half>(g, lo, hi); break;
      default: acc += mt_squares<__nv_bfloat16>(g, lo, hi); break;
    }
  });
  acc = mt_block_sum(acc, s);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

__global__ void mt_count_kernel(long long* step) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  *step += 1;
}

struct MtClip {
  const double* partial;      // of the norm; null: no clipping
  int partials;
  float* norm;                // block 0 writes it
  double max_norm;
};

__device__ __forceinline__ float mt_share(const MtClip& c, double* s) {
  if (c.partial == nullptr) return 1.0f;
  double v = 0.0;
  for (int i = threadIdx.x; i < c.partials; i += kMtThreads) v += c.partial[i];
  const double n = sqrt(mt_block_sum(v, s));
  if (c.norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *c.norm = (float)n;
  return n > c.max_norm && c.max_norm > 0.0 ? (float)(c.max_norm / (n + 1e-6)) : 1.0f;
}

__global__ void __launch_bounds__(kMtThreads) mt_finish_kernel(MtClip c) {
  __shared__ double s[kMtThreads / 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  mt_share(c, s);
}

template <typename T, typename O>
__device__ __forceinline__ void mt_scale(const void* g, void* out, long long lo, long long hi, float share) {
  const T* p = (const T*)g;
  O* o = (O*)out;
  mt_walk<2>(
      lo, hi, [&](long long i) { return mt_aligned(p + i) && mt_aligned(o + i); },
      [&](long long i) { mt_store<O>(o, i, mt_load<T>(p, i) * share); },
      [&](auto count, long long i) {
        constexpr int N = decltype(count)::value;
        float x[N][8];
#pragma unroll
        for (int u = 0; u < N; ++u) mt_load8(p + i + u * 8ll * kMtThreads, x[u]);
#pragma unroll
        for (int u = 0; u < N; ++u) {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[u][k] *= share;
          mt_store8(o + i + u * 8ll * kMtThreads, x[u]);
        }
      });
}

template <typename T>
__device__ __forceinline__ void mt_scale_to(int type, const void* g, void* out, long long lo, long long hi, float share) {
  switch (type) {
    case MT_F32: mt_scale<T, float>(g, out, lo, hi, share); break;
    case MT_F16: mt_scale<T, __half>(g, out, lo, hi, share); break;
    default: mt_scale<T, __nv_bfloat16>(g, out, lo, hi, share); break;
  }
}

__global__ void __launch_bounds__(kMtThreads, 3) mt_scale_kernel(const __grid_constant__ MtTable<2> tb, MtClip c) {
  __shared__ double s[kMtThreads / 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float share = mt_share(c, s);
  mt_pieces(tb, [&](int i, long long lo, long long hi) {
    const void* g = tb.ptr[0][i];
    void* o = tb.ptr[1][i];
    if (share == 1.0f && g == o) return;
    switch (tb.type[0][i]) {
      case MT_F32: mt_scale_to<float>(tb.type[1][i], g, o, lo, hi, share); break;
      case MT_F16: mt_scale_to<__half>(tb.type[1][i], g, o, lo, hi, share); break;
      default: mt_scale_to<__nv_bfloat16>(tb.type[1][i], g, o, lo, hi, share); break;
    }
  });
}

struct MtAdam {
  const float* lr_dev;          // where given, in place of lr
  const long long* step;
  double lr, beta1, beta2, eps, decay;
  int decoupled;
};

struct MtAdamNow {              // the constants of this step
  float share, beta1, keep1, beta2, keep2, step_size, root, eps, shrink, decay;
};

__device__ __forceinline__ void mt_adam_one(const MtAdamNow& a, float& p, float g, float& m, float& v) {
  g *= a.share;
  if (a.decay != 0.0f) g = fmaf(a.decay, p, g);
  m = fmaf(a.beta1, m, a.keep1 * g);
  v = fmaf(a.beta2, v, a.keep2 * g * g);
  p = p * a.shrink - a.step_size * m / (sqrtf(v) * a.root + a.eps);
}

template <typename P, typename G>
__device__ __forceinline__ void mt_adam(const MtAdamNow& a, void* pp, const void* gg, float* m, float* v, long long lo, long long hi) {
  P* p = (P*)pp;
  const G* g = (const G*)gg;
  mt_walk<1>(
      lo, hi, [&](long long i) { return mt_aligned(p + i) && mt_aligned(g + i) && mt_aligned(m + i) && mt_aligned(v + i); },
      [&](long long i) {
        float x = mt_load<P>(p, i), mi = m[i], vi = v[i];
        mt_adam_one(a, x, mt_load<G>(g, i), mi, vi);
        mt_store<P>(p, i, x);
        m[i] = mi;
        v[i] = vi;
      },
      [&](auto, long long i) {
        float x[8], y[8], mi[8], vi[8];
        mt_load8(p + i, x);
        mt_load8(g + i, y);
        mt_load8(m + i, mi);
        mt_load8(v + i, vi);
#pragma unroll
        for (int k = 0; k < 8; ++k) mt_adam_one(a, x[k], y[k], mi[k], vi[k]);
        mt_store8(p + i, x);
        mt_store8(m + i, mi);
        mt_store8(v + i, vi);
      });
}

template <typename P>
__device__ __forceinline__ void mt_adam_by(int type, const MtAdamNow& a, void* p, const void* g, float* m, float* v, long long lo, long long hi) {
  switch (type) {
    case MT_F32: mt_adam<P, float>(a, p, g, m, v, lo, hi); break;
    case MT_F16: mt_adam<P, __half>(a, p, g, m, v, lo, hi); break;
    default: mt_adam<P, __nv_bfloat16>(a, p, g, m, v, lo, hi); break;
  }
}

__global__ void __launch_bounds__(kMtThreads, 2) mt_adam_kernel(const __grid_constant__ MtTable<4> tb, MtClip c, MtAdam h) {
  __shared__ double s[kMtThreads / 32];
  __shared__ MtAdamNow now;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float share = mt_share(c, s);
  if (threadIdx.x == 0) {
    const double t = (double)*h.step, lr = h.lr_dev != nullptr ? (double)*h.lr_dev : h.lr;
    now.share = share;
    now.beta1 = (float)h.beta1;
    now.keep1 = (float)(1.0 - h.beta1);
    now.beta2 = (float)h.beta2;
    now.keep2 = (float)(1.0 - h.beta2);
    now.step_size = (float)(lr / (1.0 - pow(h.beta1, t)));
    now.root = (float)(1.0 / sqrt(1.0 - pow(h.beta2, t)));
    now.eps = (float)h.eps;
    now.shrink = h.decoupled ? (float)(1.0 - lr * h.decay) : 1.0f;
    now.decay = h.decoupled ? 0.0f : (float)h.decay;
  }
  __syncthreads();
  const MtAdamNow a = now;
  mt_pieces(tb, [&](int i, long long lo, long long hi) {
    void* p = tb.ptr[0][i];
    const void* g = tb.ptr[1][i];
    float *m = (float*)tb.ptr[2][i], *v = (float*)tb.ptr[3][i];
    switch (tb.type[0][i]) {
      case MT_F32: mt_adam_by<float>(tb.type[1][i], a, p, g, m, v, lo, hi); break;
      case MT_F16: mt_adam_by<__half>(tb.type[1][i], a, p, g, m, v, lo, hi); break;
      default: mt_adam_by<__nv_bfloat16>(tb.type[1][i], a, p, g, m, v, lo, hi); break;
    }
  });
}

// Tensors [at, at + n) of the set as one launch's table; returns its blocks.
template <int NP>
static int mt_table(MtTable<NP>* tb, int wave, void* const* const* ptrs, const long long* numel, const unsigned char* const* types, int at, int n) {
  tb->tensors = n;
  tb->start[0] = 0;
  for (int i = 0; i < n; ++i) {
    for (int k = 0; k < NP; ++k) tb->ptr[k][i] = ptrs[k][at + i];
    for (int k = 0; k < (NP < 2 ? 1 : 2); ++k) tb->type[k][i] = types[k][at + i];
    tb->start[i + 1] = tb->start[i] + numel[at + i];
  }
  const long long total = tb->start[n], least = 8 * kMtThreads;      // eight values for every thread
  const int most = total < kMtSmall ? wave : kMtBlocksMax;
  long long per = (total + most - 1) / most;
  per = (per + 1023) / 1024 * 1024;
  tb->per_block = per < least ? least : per;
  const int blocks = (int)((total + tb->per_block - 1) / tb->per_block);
  for (int b = 0, i = 0; b < blocks; ++b) {
    while (i + 1 < n && tb->start[i + 1] <= (long long)b * tb->per_block) ++i;
    tb->first[b] = (unsigned short)i;
  }
  return blocks;
}

static bool mt_good(int n, const long long* numel, const unsigned char* type) {
  if (n < 1 || numel == nullptr || type == nullptr) return false;
  for (int i = 0; i < n; ++i)
    if (numel[i] < 1 || type[i] > MT_BF16) return false;
  return true;
}

static cudaError_t mt_norm(int n, void* const* g, const long long* numel, const unsigned char* type, double* partial, int* partials, long long* step,
                           cudaStream_t st) {
  MtTable<1> tb;
  cudaError_t e = cudaSuccess;
  *partials = 0;
  for (int at = 0; at < n && e == cudaSuccess; at += kMtTensors) {
    const int blocks = mt_table<1>(&tb, kMtWave, &g, numel, &type, at, n - at < kMtTensors ? n - at : kMtTensors);
    e = launch_pdl(mt_norm_kernel, dim3(blocks), dim3(kMtThreads), 0, st, tb, partial + *partials, at == 0 ? step : (long long*)nullptr);
    *partials += blocks;
  }
  return e;
}

}  // namespace bonsai

extern "C" {

// Doubles of workspace that the norm of n tensors needs.
long long bonsai_mt_partials(int n) { return n < 1 ? 0 : (long long)((n + bonsai::kMtTensors - 1) / bonsai::kMtTensors) * bonsai::kMtBlocksMax; }

// g: addresses of n dense tensors, numel (at least 1), type (0 f32, 1 f16, 2 bf16).  norm: one f32.  partial: bonsai_mt_partials(n) doubles.
int bonsai_mt_norm(int n, void* const* g, const long long* numel, const unsigned char* type, double* partial, float* norm, cudaStream_t st) {
  using namespace bonsai;
  if (!mt_good(n, numel, type) || g == nullptr || partial == nullptr || norm == nullptr) return BONSAI_CUDA_BAD_ARG;
  int partials = 0;
  cudaError_t e = mt_norm(n, g, numel, type, partial, &partials, nullptr, st);
  if (e == cudaSuccess) e = launch_pdl(mt_finish_kernel, dim3(1), dim3(kMtThreads), 0, st, MtClip{partial, partials, norm, 0.0});
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

// out: where the clipped values go (the addresses of g for clipping in place), of types otype.
int bonsai_mt_clip(int n, void* const* g, void* const* out, const long long* numel, const unsigned char* type, const unsigned char* otype,
                   double max_norm, double* partial, float* norm, cudaStream_t st) {
  using namespace bonsai;
  if (!mt_good(n, numel, type) || !mt_good(n, numel, otype) || g == nullptr || out == nullptr || partial == nullptr || norm == nullptr)
    return BONSAI_CUDA_BAD_ARG;
  int partials = 0;
  cudaError_t e = mt_norm(n, g, numel, type, partial, &partials, nullptr, st);
  MtTable<2> tb;
  void* const* ptrs[2] = {g, out};
  const unsigned char* types[2] = {type, otype};
  for (int at = 0; at < n && e == cudaSuccess; at += kMtTensors) {
    const int blocks = mt_table<2>(&tb, kMtWave, ptrs, numel, types, at, n - at < kMtTensors ? n - at : kMtTensors);
    e = launch_pdl(mt_scale_kernel, dim3(blocks), dim3(kMtThreads), 0, st, tb, MtClip{partial, partials, norm, max_norm});
  }
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

// One step over n parameters p (ptype) with gradients g (gtype) and f32 moments m, v.  step: device counter, raised by one here.  partial, norm:
// given where the gradients are clipped to max_norm first (they are left as they are).
int bonsai_mt_adam(int n, void* const* p, void* const* g, void* const* m, void* const* v, const long long* numel, const unsigned char* ptype,
                   const unsigned char* gtype, double lr, const float* lr_dev, double beta1, double beta2, double eps, double decay, int decoupled,
                   long long* step, double max_norm, double* partial, float* norm, cudaStream_t st) {
  using namespace bonsai;
  if (!mt_good(n, numel, ptype) || !mt_good(n, numel, gtype) || p == nullptr || g == nullptr || m == nullptr || v == nullptr || step == nullptr ||
      (partial == nullptr) != (norm == nullptr))
    return BONSAI_CUDA_BAD_ARG;
  int partials = 0;
  cudaError_t e = partial != nullptr ? mt_norm(n, g, numel, gtype, partial, &partials, step, st)
                                     : launch_pdl(mt_count_kernel, dim3(1), dim3(1), 0, st, step);
  MtTable<4> tb;
  void* const* ptrs[4] = {p, g, m, v};
  const unsigned char* types[2] = {ptype, gtype};
  const MtAdam h = {lr_dev, step, lr, beta1, beta2, eps, decay, decoupled};
  for (int at = 0; at < n && e == cudaSuccess; at += kMtTensors) {
    const int blocks = mt_table<4>(&tb, kMtWaveAdam, ptrs, numel, types, at, n - at < kMtTensors ? n - at : kMtTensors);
    e = launch_pdl(mt_adam_kernel, dim3(blocks), dim3(kMtThreads), 0, st, tb, MtClip{partial, partials, norm, max_norm}, h);
  }
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

}  // extern "C"
