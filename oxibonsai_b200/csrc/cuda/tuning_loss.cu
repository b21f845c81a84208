// Losses over log-probabilities of tokens, rows of `length` tokens of which a mask says which count:
//
//   preference  s_r = sum over the row's tokens of (l - ref) [over their number];  z = s_chosen - s_rejected, rows p and pairs + p;  m = beta z
//               sigmoid  (1 - e) log(1 + exp(-m)) + e log(1 + exp(m))        hinge  max(0, 1 - m)        ipo  (z - 1 / (2 beta))^2
//   policy      q = exp(l - old);  each = -min(q g, clip(q, 1 - lo, 1 + hi) g) + w (exp(ref - l) - (ref - l) - 1),  summed or averaged
//
// Both are bound by memory when they are large and by launches when they are small.  A block takes a chunk of one row and leaves its sums in
// f64, one block adds them in one order: no atomics, the same values give the same bits.  The forward pass of the policy loss leaves each token's
// slope in f32, which the backward pass scales (4 bytes written and read for a token instead of the 13 to 17 that it is made from); the
// preference loss has one slope for a row.  Whether a ratio is clipped goes by l - old as f64 has it, exactly, so that a token next to a border falls on the
// same side whatever exp rounds; only steps that f32 cannot tell from the border are made again in f64.  Masked places reach nothing, whatever they hold.
//
// Measured on one B200, forward and backward in a graph: 1024 x 8192 f32 tokens with gains, mask and penalty (176 MB and 67 MB) 64 us; 512 rows of 4096 tokens of
// preference pairs 12 us; 16 rows of 300 to 511 tokens 7 us, three launches.  The policy pass is bound by its 128 instructions a token, not by memory (47 of the 64 us, 70 % of the
// issue slots).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <math.h>

#include "common.cuh"

namespace bonsai {

constexpr int kTuneThreads = 256, kTuneQuads = 2, kTuneFinish = 512;

template <typename T> __device__ __forceinline__ float tune_float(T v);
template <> __device__ __forceinline__ float tune_float(float v) { return v; }
template <> __device__ __forceinline__ float tune_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float tune_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Four neighbouring tokens from `p` on; WIDE: aligned, so that they are one access.  `n`: how many there are; the others are 0.
template <bool WIDE>
__device__ __forceinline__ void tune_load4(const float* p, int n, float* v) {
  if (WIDE && n >= 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.0f;
  }
}
template <bool WIDE, typename T>
__device__ __forceinline__ void tune_load4(const T* p, int n, float* v) {
  if (WIDE && n >= 4) {
    __align__(8) T t[4];
    *reinterpret_cast<uint2*>(t) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = tune_float<T>(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? tune_float<T>(p[i]) : 0.0f;
  }
}
// bit i: token i counts
template <bool WIDE>
__device__ __forceinline__ unsigned tune_mask4(const unsigned char* p, int n) {
  if (p == nullptr) return n >= 4 ? 15u : (1u << n) - 1u;
  unsigned m = 0;
  if (WIDE && n >= 4) {
    const uchar4 u = *reinterpret_cast<const uchar4*>(p);
    m = (u.x != 0) | (u.y != 0) << 1 | (u.z != 0) << 2 | (u.w != 0) << 3;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) m |= (i < n && p[i] != 0 ? 1u : 0u) << i;
  }
  return m;
}
__device__ __forceinline__ void tune_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void tune_put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void tune_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
template <bool WIDE>
__device__ __forceinline__ void tune_store4(float* p, int n, const float* v) {
  if (WIDE && n >= 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = v[i];
  }
}
template <bool WIDE, typename T>
__device__ __forceinline__ void tune_store4(T* p, int n, const float* v) {
  if (WIDE && n >= 4) {
    __align__(8) T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) tune_put(&t[i], v[i]);
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(t);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) tune_put(p + i, v[i]);
  }
}

// Sums over a block of `blockDim.x` threads (whole warps), in thread 0, in one order; room for N of each warp.
template <int N>
__device__ __forceinline__ void tune_block_sums(double* v, double (*room)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) room[threadIdx.x >> 5][i] = v[i];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = room[0][i];
      for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v[i] += room[w][i];
    }
  }
}

struct TuneRows {            // rows of tokens: an address and the distance of rows
  const void* p;
  long long ld;
};
struct TunePart {            // of one chunk
  double loss, kl;           // preference: loss is the sum of l - ref
  int live, clipped;
};
struct TuneShape {
  long long rows;
  int length, chunks;        // tokens of a row, blocks of a row
};

// The tokens of this block's chunk of its row, four at a time: body(place, number of tokens there).
template <typename Body>
__device__ __forceinline__ void tune_quads(const TuneShape& sh, int chunk, Body body) {
  const int first = chunk * (int)blockDim.x * 4 * kTuneQuads + (int)threadIdx.x * 4;
#pragma unroll
  for (int q = 0; q < kTuneQuads; ++q) {
    const int at = first + q * (int)blockDim.x * 4;
    if (at < sh.length) body(at, sh.length - at);
  }
}

// exp(x) - x - 1, and exp(x) - 1.  Up to 1/2 by the series x^2 / 2! + x^3 / 3! + ..., whose ninth term is below 2^-24 of the first; from there on
// no more than two bits cancel.
__device__ __forceinline__ float tune_excess(float x, float* grown) {
  float p = 1.0f / 362880.0f;
  p = fmaf(p, x, 1.0f / 40320.0f);
  p = fmaf(p, x, 1.0f / 5040.0f);
  p = fmaf(p, x, 1.0f / 720.0f);
  p = fmaf(p, x, 1.0f / 120.0f);
  p = fmaf(p, x, 1.0f / 24.0f);
  p = fmaf(p, x, 1.0f / 6.0f);
  p = fmaf(p, x, 0.5f);
  const float small = p * x * x, large = expf(x) - 1.0f;
  const bool near = fabsf(x) <= 0.5f;
  *grown = near ? small + x : large;
  return near ? small : large - x;
}

struct PolicyArgs {
  TuneShape shape;
  TuneRows logps, old, ref, mask;       // old, ref and mask may be absent
  const float* gain;
  long long gain_ld;
  int gain_per_token;
  double log_low, log_high;             // of the borders 1 - lo and 1 + hi
  float low_below, low_above, high_below, high_above;      // f32 next to them, or they themselves
  float low, high, kl_weight;
  float* slope;                         // [rows][length], absent where no gradient is wanted
  float* each;                          // [rows][length], absent where the loss is added up
  TunePart* part;                       // [rows][chunks]
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kTuneThreads) policy_kernel(PolicyArgs a) {
  __shared__ double room[kTuneThreads / 32][4];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long row = blockIdx.x / a.shape.chunks;
  const int chunk = (int)(blockIdx.x % a.shape.chunks);
  const T* logps = (const T*)a.logps.p + row * a.logps.ld;
  const T* old = a.old.p != nullptr ? (const T*)a.old.p + row * a.old.ld : nullptr;
  const T* ref = a.ref.p != nullptr ? (const T*)a.ref.p + row * a.ref.ld : nullptr;
  const unsigned char* mask = a.mask.p != nullptr ? (const unsigned char*)a.mask.p + row * a.mask.ld : nullptr;
  const float* gain = a.gain + row * a.gain_ld;
  const float row_gain = a.gain_per_token ? 0.0f : *gain;
  double v[4] = {0.0, 0.0, 0.0, 0.0};          // loss, divergence, live tokens, clipped ones
  tune_quads(a.shape, chunk, [&](int at, int n) {
    float l[4], o[4], r[4], g[4] = {row_gain, row_gain, row_gain, row_gain}, e[4], s[4];
    const unsigned m = tune_mask4<WIDE>(mask == nullptr ? nullptr : mask + at, n);
    tune_load4<WIDE>(logps + at, n, l);
    if (old != nullptr) tune_load4<WIDE>(old + at, n, o);
    if (ref != nullptr) tune_load4<WIDE>(ref + at, n, r);
    if (a.gain_per_token) tune_load4<WIDE>(gain + at, n, g);
    // Rounding keeps order: a step above the f32 behind a border is above the border, and only one between its neighbours needs l - old itself
    float step[4];
    unsigned over = 0, under = 0, near = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      step[i] = old != nullptr ? l[i] - o[i] : l[i] - l[i];
      over |= (step[i] > a.high_above ? 1u : 0u) << i;
      under |= (step[i] < a.low_below ? 1u : 0u) << i;
      near |= (step[i] >= a.high_below && step[i] <= a.high_above) || (step[i] >= a.low_below && step[i] <= a.low_above) ? 1u : 0u;
    }
    if (near && old != nullptr) {
      over = under = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double exact = (double)l[i] - (double)o[i];
        over |= (exact > a.log_high ? 1u : 0u) << i;
        under |= (exact < a.log_low ? 1u : 0u) << i;
      }
    }
    unsigned cut = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // a gain of 0 leaves 0, also where the ratio is infinite
      const float gained = g[i] == 0.0f ? 0.0f : expf(step[i]) * g[i];
      const unsigned clipped = (g[i] > 0.0f ? over : g[i] < 0.0f ? under : 0u) >> i & 1u;
      cut |= clipped << i;
      e[i] = clipped ? (g[i] > 0.0f ? -a.high : -a.low) * g[i] : -gained;
      s[i] = clipped ? 0.0f : -gained;
    }
    float loss = 0.0f, kls = 0.0f;             // of four tokens: no more rounding than each of them has, and a quarter of the conversions
    if (ref != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float grown;
        const float kl = tune_excess(r[i] - l[i], &grown);
        if (a.kl_weight != 0.0f) {
          e[i] = fmaf(a.kl_weight, kl, e[i]);
          s[i] = fmaf(-a.kl_weight, grown, s[i]);
        }
        kls += m >> i & 1u ? kl : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = m >> i & 1u ? e[i] : 0.0f;
      s[i] = m >> i & 1u ? s[i] : 0.0f;
      loss += e[i];
    }
    v[0] += (double)loss;
    v[1] += (double)kls;
    v[2] += (double)__popc(m);
    v[3] += (double)__popc(cut & m);
    if (a.slope != nullptr) tune_store4<WIDE>(a.slope + row * a.shape.length + at, n, s);
    if (a.each != nullptr) tune_store4<WIDE>(a.each + row * a.shape.length + at, n, e);
  });
  tune_block_sums<4>(v, room);
  if (threadIdx.x == 0) a.part[blockIdx.x] = {v[0], v[1], (int)v[2], (int)v[3]};
}

enum TuneReduction { TUNE_TOKENS = 0, TUNE_SEQUENCES = 1, TUNE_SUM = 2, TUNE_NONE = 3 };

// Adds the chunks up; weight[row] is what a token's loss counts in the whole.  One block.
__global__ void __launch_bounds__(kTuneFinish) policy_finish_kernel(TuneShape sh, const TunePart* part, int reduction, float* loss, float* stats, float* weight) {
  __shared__ double room[kTuneFinish / 32][6];
  __shared__ double counts[2];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double v[6] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0};        // loss, divergence, live, clipped, rows with live tokens, means of rows
  for (long long row = threadIdx.x; row < sh.rows; row += kTuneFinish) {
    double s = 0.0, n = 0.0;
#pragma unroll 4
    for (int c = 0; c < sh.chunks; ++c) {
      const TunePart p = part[row * sh.chunks + c];
      s += p.loss;
      v[1] += p.kl;
      n += (double)p.live;
      v[3] += (double)p.clipped;
    }
    v[0] += s;
    v[2] += n;
    v[4] += n > 0.0 ? 1.0 : 0.0;
    if (reduction == TUNE_SEQUENCES) v[5] += n > 0.0 ? s / n : 0.0;
  }
  tune_block_sums<6>(v, room);
  if (threadIdx.x == 0) {
    const double one = 1.0 / v[2];              // 0 / 0 is NaN: the mean of no tokens
    if (loss != nullptr) *loss = (float)(reduction == TUNE_TOKENS ? v[0] * one : reduction == TUNE_SEQUENCES ? v[5] / v[4] : v[0]);
    stats[0] = (float)(v[1] * one);
    stats[1] = (float)(v[3] * one);
    counts[0] = v[2];
    counts[1] = v[4];
  }
  if (weight == nullptr) return;
  __syncthreads();
  for (long long row = threadIdx.x; row < sh.rows; row += kTuneFinish) {
    double n = 1.0;
    if (reduction == TUNE_TOKENS) {
      n = counts[0];
    } else if (reduction == TUNE_SEQUENCES) {
      n = 0.0;
      for (int c = 0; c < sh.chunks; ++c) n += (double)part[row * sh.chunks + c].live;
      n *= counts[1];
    }
    weight[row] = n > 0.0 ? (float)(1.0 / n) : 0.0f;
  }
}

struct ScaleArgs {
  TuneShape shape;
  const float* slope;        // [rows][length], or one for a row
  int slope_per_token;
  const float* weight;       // for a row, absent: 1
  const float* up;           // one, one for every `up_rows`-th row, or [rows][length]
  int up_kind;               // 0, 1, 2
  long long up_rows;
  TuneRows mask;
};

// The gradient of the log-probabilities: slope * weight * the loss's gradient where the mask is set, else 0.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kTuneThreads) tune_scale_kernel(ScaleArgs a, T* __restrict__ out) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long row = blockIdx.x / a.shape.chunks, base = row * a.shape.length;
  const int chunk = (int)(blockIdx.x % a.shape.chunks);
  const unsigned char* mask = a.mask.p != nullptr ? (const unsigned char*)a.mask.p + row * a.mask.ld : nullptr;
  float by = a.weight != nullptr ? a.weight[row] : 1.0f;
  if (a.up_kind < 2) by *= a.up[a.up_kind == 0 ? 0 : row % a.up_rows];
  if (!a.slope_per_token) by *= a.slope[row];
  tune_quads(a.shape, chunk, [&](int at, int n) {
    float s[4] = {1.0f, 1.0f, 1.0f, 1.0f}, u[4] = {1.0f, 1.0f, 1.0f, 1.0f}, g[4];
    const unsigned m = tune_mask4<WIDE>(mask == nullptr ? nullptr : mask + at, n);
    if (a.slope_per_token) tune_load4<WIDE>(a.slope + base + at, n, s);
    if (a.up_kind == 2) tune_load4<WIDE>(a.up + base + at, n, u);
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = (m >> i & 1u) && s[i] != 0.0f ? s[i] * by * u[i] : 0.0f;        // masked tokens have slopes of 0
    tune_store4<WIDE>(out + base + at, n, g);
  });
}

struct PreferenceArgs {
  TuneShape shape;           // 2 * pairs rows: the chosen ones, then the rejected ones
  TuneRows logps, ref, mask;
  TunePart* part;
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kTuneThreads) preference_kernel(PreferenceArgs a) {
  __shared__ double room[kTuneThreads / 32][2];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long row = blockIdx.x / a.shape.chunks;
  const int chunk = (int)(blockIdx.x % a.shape.chunks);
  const T* logps = (const T*)a.logps.p + row * a.logps.ld;
  const T* ref = a.ref.p != nullptr ? (const T*)a.ref.p + row * a.ref.ld : nullptr;
  const unsigned char* mask = a.mask.p != nullptr ? (const unsigned char*)a.mask.p + row * a.mask.ld : nullptr;
  double v[2] = {0.0, 0.0};             // differences, live tokens
  tune_quads(a.shape, chunk, [&](int at, int n) {
    float l[4], r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const unsigned m = tune_mask4<WIDE>(mask == nullptr ? nullptr : mask + at, n);
    tune_load4<WIDE>(logps + at, n, l);
    if (ref != nullptr) tune_load4<WIDE>(ref + at, n, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[0] += m >> i & 1u ? (double)l[i] - (double)r[i] : 0.0;
    v[1] += (double)__popc(m);
  });
  tune_block_sums<2>(v, room);
  if (threadIdx.x == 0) a.part[blockIdx.x] = {v[0], 0.0, (int)v[1], 0};
}

enum PreferenceKind { PREF_SIGMOID = 0, PREF_HINGE = 1, PREF_IPO = 2 };
struct PreferenceRule {
  int kind, average, reduction;      // reduction: 0 mean, 1 sum, 2 none
  double beta, smoothing;
};

// Of one row: the sum over its chunks, and what a token counts in it (1, or one over their number).
__device__ __forceinline__ double preference_row(const TunePart* part, int chunks, int average, double* token) {
  double s = 0.0;
  long long n = 0;
  for (int c = 0; c < chunks; ++c) { s += part[c].loss; n += part[c].live; }
  *token = average ? (n > 0 ? 1.0 / (double)n : 0.0) : 1.0;
  return n > 0 ? s * *token : 0.0;
}

__global__ void __launch_bounds__(kTuneFinish) preference_finish_kernel(long long pairs, int chunks, const TunePart* part, PreferenceRule rule, float* loss,
                                                                        float* chosen, float* rejected, float* slope) {
  __shared__ double room[kTuneFinish / 32][1];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double sum[1] = {0.0};
  for (long long p = threadIdx.x; p < pairs; p += kTuneFinish) {
    double tc, tr;
    const double sc = preference_row(part + p * chunks, chunks, rule.average, &tc), sr = preference_row(part + (pairs + p) * chunks, chunks, rule.average, &tr);
    const double z = sc - sr, m = rule.beta * z;
    double v, d;                                  // the pair's loss and its derivative by z
    if (rule.kind == PREF_SIGMOID) {
      const double fall = exp(-fabs(m)), soft = log1p(fall), on = (m < 0.0 ? fall : 1.0) / (1.0 + fall);        // on = 1 / (1 + exp(-m))
      const double off = (m < 0.0 ? 1.0 : fall) / (1.0 + fall);
      const double minus = soft + fmax(-m, 0.0), plus = soft + fmax(m, 0.0);     // log(1 + exp(-m)), log(1 + exp(m))
      v = m != m ? m : rule.smoothing == 0.0 ? minus : (1.0 - rule.smoothing) * minus + rule.smoothing * plus;
      d = rule.beta * (rule.smoothing * on - (1.0 - rule.smoothing) * off);
    } else if (rule.kind == PREF_HINGE) {
      v = m < 1.0 ? 1.0 - m : m != m ? m : 0.0;
      d = m < 1.0 ? -rule.beta : m != m ? m : 0.0;
    } else {
      const double t = z - 0.5 / rule.beta;
      v = t * t;
      d = 2.0 * t;
    }
    if (rule.reduction == 2) loss[p] = (float)v;
    sum[0] += v;
    chosen[p] = (float)(rule.beta * sc);
    rejected[p] = (float)(rule.beta * sr);
    if (slope != nullptr) {
      if (rule.reduction == 0) d /= (double)pairs;
      slope[p] = (float)(d * tc);
      slope[pairs + p] = (float)(-d * tr);
    }
  }
  tune_block_sums<1>(sum, room);
  if (threadIdx.x == 0 && rule.reduction != 2) *loss = (float)(rule.reduction == 0 ? sum[0] / (double)pairs : sum[0]);
}

// Threads of a block: rows that fit a few warps take no more.
static int tune_threads(long long length) { return length <= 128 ? 32 : length <= 256 ? 64 : length <= 512 ? 128 : kTuneThreads; }
static int tune_chunks(long long length) {
  const int tokens = tune_threads(length) * 4 * kTuneQuads;
  return (int)((length + tokens - 1) / tokens);
}
static bool tune_good(long long rows, long long length) {
  return rows >= 1 && length >= 1 && length < 1ll << 30 && rows < 1ll << 31 && rows * tune_chunks(length) < 1ll << 31;
}
static TuneShape tune_shape(long long rows, long long length) { return {rows, (int)length, tune_chunks(length)}; }

// What a forward pass keeps: the chunks' sums, then where a gradient is wanted the weights of rows and the slopes (1: of rows, without weights; 2: of tokens).
struct TuneKept {
  long long weight, slope, bytes;
};
static TuneKept tune_kept(long long rows, long long length, int slopes) {
  TuneKept k;
  k.weight = (rows * tune_chunks(length) * (long long)sizeof(TunePart) + 15) / 16 * 16;
  k.slope = k.weight + (slopes == 2 ? (rows * 4 + 15) / 16 * 16 : 0);
  k.bytes = k.slope + (slopes == 2 ? rows * length * 4 : slopes == 1 ? rows * 4 : 0);
  return k;
}

// The largest f32 at most v, and the smallest at least v.
static float tune_below(double v) {
  const float f = (float)v;
  return (double)f <= v ? f : nextafterf(f, -INFINITY);
}
static float tune_above(double v) {
  const float f = (float)v;
  return (double)f >= v ? f : nextafterf(f, INFINITY);
}

// Whether four neighbouring tokens of every row are one aligned access; an absent array does not matter.
static bool tune_wide(const void* p, long long ld, int size) { return p == nullptr || (((uintptr_t)p | (uintptr_t)(ld * size)) % (4 * size) == 0); }


}  // namespace bonsai

extern "C" {

// Bytes that a forward pass over rows of `length` tokens keeps; slopes: 0 where no gradient is wanted, 1 preference, 2 policy.  Negative for sizes that are
// refused.
long long bonsai_tune_bytes(long long rows, long long length, int slopes) {
  using namespace bonsai;
  return tune_good(rows, length) ? tune_kept(rows, length, slopes).bytes : BONSAI_CUDA_BAD_ARG;
}

// logps, old, ref: rows of tokens at distances of their ld (type 0 f32, 1 f16, 2 bf16), mask: bytes; old, ref and mask may be null.  gain: f32, for a
// row or for a token.  reduction: TuneReduction.  Out: loss (f32, or [rows][length]), stats (f32: the mean divergence, the share of clipped tokens), kept:
// bonsai_tune_bytes(rows, length, 2 where a gradient is wanted, else 0).
int bonsai_policy_loss(const void* logps, long long ld_logps, const void* old, long long ld_old, const void* ref, long long ld_ref, const void* mask,
                       long long ld_mask, const float* gain, long long ld_gain, int gain_per_token, long long rows, long long length, int type, double low,
                       double high, double kl_weight, int reduction, float* loss, float* stats, void* kept, long long kept_bytes, int gradient, cudaStream_t st) {
  using namespace bonsai;
  if (logps == nullptr || gain == nullptr || loss == nullptr || stats == nullptr || kept == nullptr || !tune_good(rows, length) || type < 0 || type > 2 ||
      reduction < 0 || reduction > 3 || kept_bytes < tune_kept(rows, length, gradient ? 2 : 0).bytes || !(low >= 0.0) || !(low <= 1.0) || !(high >= 0.0))
    return BONSAI_CUDA_BAD_ARG;
  const TuneKept at = tune_kept(rows, length, gradient ? 2 : 0);
  float* slope = gradient ? (float*)((char*)kept + at.slope) : nullptr;
  float* weight = gradient ? (float*)((char*)kept + at.weight) : nullptr;
  const TuneShape sh = tune_shape(rows, length);
  const int size = type == 0 ? 4 : 2, threads = tune_threads(length);
  const double log_low = log1p(-low), log_high = log1p(high);
  PolicyArgs a = {sh, {logps, ld_logps}, {old, ld_old}, {ref, ld_ref}, {mask, ld_mask}, gain, ld_gain, gain_per_token, log_low, log_high, tune_below(log_low), tune_above(log_low), tune_below(log_high),
                  tune_above(log_high), (float)(1.0 - low), (float)(1.0 + high), (float)kl_weight, slope, reduction == TUNE_NONE ? loss : nullptr, (TunePart*)kept};
  const bool wide = length % 4 == 0 && tune_wide(logps, ld_logps, size) && tune_wide(old, ld_old, size) && tune_wide(ref, ld_ref, size) &&
                    tune_wide(mask, ld_mask, 1) && (!gain_per_token || tune_wide(gain, ld_gain, 4)) && tune_wide(slope, length, 4) &&
                    tune_wide(a.each, length, 4);
  const dim3 grid((unsigned)(rows * sh.chunks)), block(threads);
  cudaError_t e;
  if (type == 0) e = wide ? launch_pdl(policy_kernel<float, true>, grid, block, 0, st, a) : launch_pdl(policy_kernel<float, false>, grid, block, 0, st, a);
  else if (type == 1) e = wide ? launch_pdl(policy_kernel<__half, true>, grid, block, 0, st, a) : launch_pdl(policy_kernel<__half, false>, grid, block, 0, st, a);
  else e = wide ? launch_pdl(policy_kernel<__nv_bfloat16, true>, grid, block, 0, st, a) : launch_pdl(policy_kernel<__nv_bfloat16, false>, grid, block, 0, st, a);
  if (e == cudaSuccess)
    e = launch_pdl(policy_finish_kernel, dim3(1), dim3(kTuneFinish), 0, st, sh, (const TunePart*)kept, reduction, reduction == TUNE_NONE ? (float*)nullptr : loss, stats,
                   weight);
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

// Rows 0 .. pairs - 1 are the chosen answers, the next `pairs` the rejected ones; ref and mask may be null.  kind: PreferenceKind; reduction 0 mean, 1 sum,
// 2 none.  Out: loss (f32, or [pairs]), rewards [2 * pairs], kept: bonsai_tune_bytes(2 * pairs, length, 1 where a gradient is wanted, else 0).
int bonsai_preference_loss(const void* logps, long long ld_logps, const void* ref, long long ld_ref, const void* mask, long long ld_mask, long long pairs,
                           long long length, int type, int kind, int average, int reduction, double beta, double smoothing, float* loss, float* rewards,
                           void* kept, long long kept_bytes, int gradient, cudaStream_t st) {
  using namespace bonsai;
  if (logps == nullptr || loss == nullptr || rewards == nullptr || kept == nullptr || pairs < 1 || !tune_good(2 * pairs, length) || type < 0 || type > 2 ||
      kind < 0 || kind > 2 || reduction < 0 || reduction > 2 || kept_bytes < tune_kept(2 * pairs, length, gradient ? 1 : 0).bytes || !(beta > 0.0))
    return BONSAI_CUDA_BAD_ARG;
  float* slope = gradient ? (float*)((char*)kept + tune_kept(2 * pairs, length, 1).slope) : nullptr;
  const TuneShape sh = tune_shape(2 * pairs, length);
  const int size = type == 0 ? 4 : 2, threads = tune_threads(length);
  const PreferenceArgs a = {sh, {logps, ld_logps}, {ref, ld_ref}, {mask, ld_mask}, (TunePart*)kept};
  const bool wide = length % 4 == 0 && tune_wide(logps, ld_logps, size) && tune_wide(ref, ld_ref, size) && tune_wide(mask, ld_mask, 1);
  const dim3 grid((unsigned)(sh.rows * sh.chunks)), block(threads);
  cudaError_t e;
  if (type == 0) e = wide ? launch_pdl(preference_kernel<float, true>, grid, block, 0, st, a) : launch_pdl(preference_kernel<float, false>, grid, block, 0, st, a);
  else if (type == 1) e = wide ? launch_pdl(preference_kernel<__half, true>, grid, block, 0, st, a) : launch_pdl(preference_kernel<__half, false>, grid, block, 0, st, a);
  else
    e = wide ? launch_pdl(preference_kernel<__nv_bfloat16, true>, grid, block, 0, st, a) : launch_pdl(preference_kernel<__nv_bfloat16, false>, grid, block, 0, st, a);
  if (e == cudaSuccess)
    e = launch_pdl(preference_finish_kernel, dim3(1), dim3(kTuneFinish), 0, st, pairs, sh.chunks, (const TunePart*)kept,
                   PreferenceRule{kind, average, reduction, beta, smoothing}, loss, rewards, rewards + pairs, slope);
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

// Gradient out [rows][length] of a forward pass from what it kept (slopes: 1 preference, 2 policy): slope * weight * up, 0 where the mask (may be null) is
// not set.  up: one value (up_kind 0), that of row % up_rows (1), or one for a token (2).
int bonsai_tune_scale(const void* kept, long long kept_bytes, int slopes, const float* up, int up_kind, long long up_rows, const void* mask, long long ld_mask,
                      long long rows, long long length, int type, void* out, cudaStream_t st) {
  using namespace bonsai;
  if (kept == nullptr || up == nullptr || out == nullptr || !tune_good(rows, length) || type < 0 || type > 2 || up_kind < 0 || up_kind > 2 || up_rows < 1 ||
      slopes < 1 || slopes > 2 || kept_bytes < tune_kept(rows, length, slopes).bytes)
    return BONSAI_CUDA_BAD_ARG;
  const TuneKept at = tune_kept(rows, length, slopes);
  const int slope_per_token = slopes == 2;
  const float *slope = (const float*)((const char*)kept + at.slope), *weight = slope_per_token ? (const float*)((const char*)kept + at.weight) : nullptr;
  const TuneShape sh = tune_shape(rows, length);
  const int size = type == 0 ? 4 : 2;
  const ScaleArgs a = {sh, slope, slope_per_token, weight, up, up_kind, up_rows, {mask, ld_mask}};
  const bool wide = length % 4 == 0 && (!slope_per_token || tune_wide(slope, length, 4)) && (up_kind < 2 || tune_wide(up, length, 4)) &&
                    tune_wide(mask, ld_mask, 1) && tune_wide(out, length, size);
  const dim3 grid((unsigned)(rows * sh.chunks)), block(tune_threads(length));
  cudaError_t e;
  if (type == 0) e = wide ? launch_pdl(tune_scale_kernel<float, true>, grid, block, 0, st, a, (float*)out) : launch_pdl(tune_scale_kernel<float, false>, grid, block, 0, st, a, (float*)out);
  else if (type == 1) e = wide ? launch_pdl(tune_scale_kernel<__half, true>, grid, block, 0, st, a, (__half*)out) : launch_pdl(tune_scale_kernel<__half, false>, grid, block, 0, st, a, (__half*)out);
  else e = wide ? launch_pdl(tune_scale_kernel<__nv_bfloat16, true>, grid, block, 0, st, a, (__nv_bfloat16*)out) : launch_pdl(tune_scale_kernel<__nv_bfloat16, false>, grid, block, 0, st, a, (__nv_bfloat16*)out);
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

}  // extern "C"
