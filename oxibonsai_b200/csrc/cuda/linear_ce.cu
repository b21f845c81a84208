// Softmax cross entropy of a linear head, in pieces of the vocabulary, without the logits, and its gradients.
//
//   z_iv = h_i . w_v,   lse_i = log sum_v exp z_iv,   q_iv = (1 - a) [v = t_i] + a / V
//   loss_i = lse_i - sum_v q_iv z_iv
//   dz_iv = u_i (exp(z_iv - lse_i) - q_iv),   dh = dz W,   dW = dz^T h
//
// Four products of 2 n V D operations: the logits for the loss, the logits again piece by piece for dz, and the two gradients.  One
// kernel makes them all (ce_gemm_kernel), on pairs of SMs with tcgen05.mma cta_group::2 over tiles of 256 x up to 256, and differs
// by where its operands lie and what happens to a finished tile:
//   CE_LSE  h [n][D] x W [V][D]: a row's maximum and sum of exponentials over its half of the tile's columns; no logit leaves the SM
//   CE_FEW  the same for up to 128 tokens, W [V][D] x h: the head's rows fill the tile and its columns are the tokens.  The head's bytes bound it, if
//           the tensor cores leave them the power: one token in a tile of 256 rows had the card at 1 GHz under its cap, 294 us for the
//           8B head where its bytes take 190
//   CE_DZ   the product again; exp(z - lse) - q in 16 bits into the piece's buffer [n][piece]
//   CE_DH   dz [n][piece] x W [piece][D], summed over the piece: W is read across its rows (MN-major operand), nothing is transposed
//   CE_DW   dz^T [piece][n] x h [n][D]: both operands across their rows
// The tensor cores bound all four where there are many tokens; with few, the head's bytes do.
//
// Rows whose target is the ignored one are left out before anything is multiplied: the live rows are copied side by side, and their number
// stays on the device.  A target outside the vocabulary makes its row's loss and gradients NaN, and so does a wait that expires.
//
// dz is rounded to the inputs' 16-bit type before it is multiplied, as the operand of a tensor-core product has to be.  It is stored over the largest
// finite upstream gradient (that factor enters with the products' sums), in f16 times 2^15: in a row that has it probabilities down to 2^-29 stay normal. Where
// rows bring gradients of their own (reduction "none"), dz of a row 2^k below the largest is held in steps of 2^(k-39) of its own.
//
// float32 inputs become three bfloat16 parts each (8 bits a part, exact down to 2^-24) and six products of parts: the parts that are left out
// are below 2^-24 of the product.
//
// The tensor cores' sums truncate: over a few hundred steps a logit of 10 loses some 1e-5, always downwards, which an f32 loss shows.  Where the result is f32
// (the loss of any type, all products of f32) a tile is therefore added to registers, with rounding, every few blocks of k.  Gradients in 16 bits
// round a hundred times coarser and take the tensor cores' sum as it is.
#include <cuda.h>

#include "linear_ce.cuh"
#include "linear_ce_issue.h"
#include "tcgen05.cuh"

namespace bonsai {

enum CeMode { CE_LSE, CE_FEW, CE_DZ, CE_DH, CE_DW };

constexpr int kCeStages = 6;
constexpr int kCeBlock = 64;                            // k per stage
constexpr int kCeOperand = 128 * kCeBlock * 2;          // 16 KB: a CTA's half of one operand
constexpr int kCeEpiWarps = 8;
constexpr int kCeThreads = (kCeEpiWarps + 2) * 32;
constexpr int kCeCols = 512;                            // TMEM columns, for two accumulators of 256 or, with few tokens, four of 128
constexpr int kCeFew = 128;                             // tokens up to which the head's rows fill the tile
constexpr int kCeGroup = 16;                            // row tiles that share the head's tiles while those are in L2
constexpr int kCeStage = 32 * 128;                      // shared memory of an epilogue warp: 32 rows of 128 bytes on their way out
constexpr int kCeSegment32 = 2, kCeSegment16 = 16, kCeSegmentFew = 4;          // blocks of k between two additions to registers: f32; the loss; of few tokens
constexpr int kCeTerms = 6;
__device__ const unsigned char kCeTermA[kCeTerms] = {2, 0, 1, 1, 0, 0}, kCeTermB[kCeTerms] = {0, 2, 1, 0, 1, 0};      // the small ones first

struct CeGemm {
  CeRows rows;
  int columns;          // LSE, DZ: vocabulary rows of the piece; DH, DW: width
  int depth;            // k: width (LSE, DZ), vocabulary rows of the piece (DH); DW: the live rows
  int m;                // DW: vocabulary rows of the piece
  int tile_n;           // columns of a tile, a multiple of 16
  int a_rows;           // K-major A: rows of a copy; FEW: rows of the head in a CTA's half of a tile
  int c0;               // first vocabulary row of the piece; where the head's rows start in its tensor map: w_row
  int w_row;
  int vocab;
  float smoothing;
  // LSE
  float *part_m, *part_s, *part_z, *at_target;
  long long ldn;
  int slot;             // first slot of this piece
  // DZ
  CeUp up;
  uint16_t* dz;
  long long ldz, plane; // elements of a row, of a plane
  // DH, DW
  int piece_blocks, clusters, acc_rows, first, last;
  float* acc;           // DH: [splits][live rows up to 256][columns] sums of several pieces or parts
  void* out;            // [..][columns] of the inputs' type
};

// ---- rows ---------------------------------------------------------------------------------------------------------------------------
// One block walks the targets and lists the live rows in order.  `each`: the loss of ignored rows (reduction "none").
__global__ void __launch_bounds__(1024) ce_rows_kernel(const long long* targets, int n, int vocab, long long ignore, CeRows r, float* each) {
  __shared__ int warps[32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += 1024) {
    const int i = i0 + t;
    const long long tgt = i < n ? targets[i] : ignore;
    const bool live = i < n && tgt != ignore;
    const unsigned m = __ballot_sync(0xffffffffu, live);
    if (lane == 0) warps[warp] = __popc(m);
    __syncthreads();
    const int c = warps[lane];
    int before = lane < warp ? c : 0, all = c;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    if (i < n && !live) r.place[i] = -1;
    if (live) {
      const int at = base + before + __popc(m & ((1u << lane) - 1));
      r.index[at] = i;
      r.place[i] = at;
      r.target[at] = tgt >= 0 && tgt < vocab ? (int)tgt : -1;
    } else if (i < n && each != nullptr) {
      each[i] = 0.0f;
    }
    base += all;
    __syncthreads();
  }
  if (t == 0) {
    r.count[0] = base;
    r.count[1] = 0;
  }
}

__device__ __forceinline__ float ce_f32(float x) { return x; }
__device__ __forceinline__ uint16_t ce_bits(__half x) { return __half_as_ushort(x); }
__device__ __forceinline__ uint16_t ce_bits(__nv_bfloat16 x) { return __bfloat16_as_ushort(x); }

// x as the sum of three bfloat16; what is not finite stays in the first
__device__ __forceinline__ void ce_split(float x, uint16_t* p) {
  const __nv_bfloat16 a = __float2bfloat16_rn(x);
  const float fa = __bfloat162float(a), r = isfinite(fa) ? x - fa : 0.0f;
  const __nv_bfloat16 b = __float2bfloat16_rn(r);
  p[0] = ce_bits(a);
  p[1] = ce_bits(b);
  p[2] = ce_bits(__float2bfloat16_rn(r - __bfloat162float(b)));
}

// Rows of a matrix side by side with a row stride of whole 16-byte words: the live rows (count given; zeros up to the next 256) or all of
// them; f32 as three planes, or as it is for the few-rows kernels.  A thread takes eight values.  Bound by memory.
template <typename T, bool kPlain = false>
__global__ void __launch_bounds__(256) ce_pack_kernel(const T* src, long long ld, long long row0, int rows, const int* count, const int* index,
                                                      int width, uint16_t* dst, int ldd, long long plane) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = count != nullptr ? *count : rows, n_out = count != nullptr ? (n + 255) / 256 * 256 : rows, words = ldd >> 3;
  const bool wide = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t)(ld * sizeof(T))) & 15) == 0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)n_out * words; i += (long long)gridDim.x * 256) {
    const int r = (int)(i / words), k0 = (int)(i % words) * 8;
    __align__(16) T v[8];
    const T* s = src + (index != nullptr && r < n ? (long long)index[r] : row0 + r) * ld + k0;
    if (r < n && wide && k0 + 8 <= width) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; ++j) reinterpret_cast<uint4*>(v)[j] = reinterpret_cast<const uint4*>(s)[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = r < n && k0 + j < width ? s[j] : T(0.0f);
    }
    uint16_t* o = dst + (long long)r * ldd + k0;
    if constexpr (kPlain) {
      uint4* w = reinterpret_cast<uint4*>(reinterpret_cast<T*>(dst) + (long long)r * ldd + k0);
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; ++j) w[j] = reinterpret_cast<const uint4*>(v)[j];
    } else if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(v);
    } else {
      __align__(16) uint16_t p[3][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint16_t q[3];
        ce_split(ce_f32(v[j]), q);
        p[0][j] = q[0]; p[1][j] = q[1]; p[2][j] = q[2];
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(o + k * plane) = *reinterpret_cast<const uint4*>(p[k]);
    }
  }
}

// ---- the product ----------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t ce_map(uint32_t addr, uint32_t rank) {      // the same shared-memory place in CTA `rank` of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void ce_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void ce_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrives on the barrier at this place in both CTAs once the MMAs issued so far are done
__device__ __forceinline__ void ce_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(tc::smem_u32(bar)),
               "h"((uint16_t)3)
               : "memory");
}
// Says that this warp has read an accumulator (its tcgen05.ld have come back, and the tensor-memory fence is behind them).  Nothing in memory is handed over,
// so the arrive releases nothing at cluster scope: that cost some 1.4 us each time, the stores before it included, and one token of the 8B head
// took 250 us with sums in registers every 4 blocks instead of 217.
__device__ __forceinline__ void ce_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void ce_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// An operand across its rows (MN-major): a tile of 64 columns x 64 k is 64 rows of 128 bytes, swizzled like the K-major tiles; the next 64 columns
// begin 8 KB further (leading offset), the next eight k 1 KB (stride), sixteen k 2 KB.
__device__ __forceinline__ uint64_t ce_desc_mn(uint32_t smem_addr) {
  return (tc::smem_desc_sw128(smem_addr) & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(8192 >> 4) << 16);
}

// DH: parts into which the sum over a piece is cut, from the number of live rows, which only the device knows: as many as even out the rounds of
// tiles over the clusters.  Costs are in times of one block of k (0.27 us): a part costs its blocks and an epilogue of some eight, and its sums are
// written and read again at some 200 000 values in that time.  1640 live rows x 4096 over 50 688 vocabulary rows: one part, two rounds
// for one and a half, 658 us; three parts 560.
__device__ __forceinline__ int ce_splits(int n, int width, int piece_blocks, int terms, int clusters, int acc_rows) {
  const int rows = (n + 255) & ~255, tiles = (rows >> 8) * ((width + 255) >> 8);
  int best = 1;
  float best_cost = 0.0f;
  for (int s = 1; s <= 16 && (s == 1 || ((long long)s * rows <= acc_rows && piece_blocks / s >= 8)); ++s) {
    const int rounds = (tiles * s + clusters - 1) / clusters;
    const float cost = (float)rounds * ((float)piece_blocks * terms / s + 8.0f) + (s > 1 ? (float)s * n * width * 5e-6f : 0.0f);
    if (s == 1 || cost < best_cost) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

template <int MODE>
struct CeTiles {       // tiles of a launch, and which one has which number
  int rt, ct, all, splits;
  __device__ __forceinline__ CeTiles(const CeGemm& p, int n, int terms) {
    rt = MODE == CE_FEW ? (n > 0 ? (p.columns + 2 * p.a_rows - 1) / (2 * p.a_rows) : 0) : ((MODE == CE_DW ? p.m : n) + 255) >> 8;
    ct = MODE == CE_FEW ? 1 : (p.columns + p.tile_n - 1) / p.tile_n;
    splits = MODE == CE_DH ? ce_splits(n, p.columns, p.piece_blocks, terms, p.clusters, p.acc_rows) : 1;
    all = rt * ct * splits;
  }
  __device__ __forceinline__ void at(int i, int* r, int* c, int* split) const {
    *split = 0;
    if (MODE == CE_LSE || MODE == CE_DZ) {      // groups of row tiles; in a group the row tiles of one column tile after another
      const int g = i / (kCeGroup * ct), in = i - g * kCeGroup * ct, high = min(kCeGroup, rt - g * kCeGroup);
      *c = in / high;
      *r = g * kCeGroup + in % high;
    } else {                                    // the column tiles of a row tile one after another
      *c = i % ct;
      *r = i / ct % rt;
      *split = i / ct / rt;
    }
  }
};

template <typename T> __device__ __forceinline__ uint32_t ce_pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t ce_pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t ce_pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp's 32 rows on their way out: every thread has a row's values, 32 columns at a time, and writes them to shared memory (128 bytes a row, 16-byte
// chunks swizzled); then eight threads store a row's chunks side by side, four rows per instruction.  From the rows' own threads each
// store met 32 different lines, and rows of odd widths went value by value: 777 x 32003 x 1001 took 300 us for dW, 64 MB.
template <typename T>
__device__ __forceinline__ void ce_stage(uint8_t* stage, int lane, int chunk0, const float* v) {
  uint8_t* row = stage + lane * 128;
#pragma unroll
  for (int j = 0; j < (int)sizeof(T) * 2; ++j) {
    uint4 w;
    if constexpr (sizeof(T) == 4) {
      w = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
    } else {
      w = make_uint4(ce_pack2<T>(v[8 * j], v[8 * j + 1]), ce_pack2<T>(v[8 * j + 2], v[8 * j + 3]), ce_pack2<T>(v[8 * j + 4], v[8 * j + 5]),
                     ce_pack2<T>(v[8 * j + 6], v[8 * j + 7]));
    }
    *reinterpret_cast<uint4*>(row + (((chunk0 + j) ^ (lane & 7)) << 4)) = w;
  }
}

// A row's 32 columns from its own thread (f32's parts of dz, 64 bytes each on aligned rows: staged they took twice as long)
__device__ __forceinline__ void ce_store32(__nv_bfloat16* dst, const float* v, int valid) {
  if (valid >= 32) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      reinterpret_cast<uint4*>(dst)[j] = make_uint4(ce_pack2<__nv_bfloat16>(v[8 * j], v[8 * j + 1]), ce_pack2<__nv_bfloat16>(v[8 * j + 2], v[8 * j + 3]),
                                                    ce_pack2<__nv_bfloat16>(v[8 * j + 4], v[8 * j + 5]), ce_pack2<__nv_bfloat16>(v[8 * j + 6], v[8 * j + 7]));
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < valid) dst[j] = __float2bfloat16_rn(v[j]);
  }
}

// dst: this thread's row, at the block's first column; `valid` of the staged columns are inside, `add`: f32 sums that are there already
template <typename T>
__device__ __forceinline__ void ce_flush(const uint8_t* stage, int lane, T* dst, bool ok, int valid, bool add = false) {
  constexpr int kPer = 16 / sizeof(T);
  __syncwarp();
  const unsigned rows = __ballot_sync(0xffffffffu, ok), odd = __ballot_sync(0xffffffffu, ok && (reinterpret_cast<uintptr_t>(dst) & 15) != 0);
  const unsigned long long mine = reinterpret_cast<unsigned long long>(dst);
  if (odd == 0) {
    const int c = lane & 7, n = valid - c * kPer;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 3);
      T* o = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, mine, r)) + c * kPer;
      if (((rows >> r) & 1) == 0 || n <= 0) continue;
      const uint4* from = reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
      if (n >= kPer) {
        uint4 w = *from;
        if constexpr (sizeof(T) == 4) {
          if (add) {
            const float4 a = *reinterpret_cast<const float4*>(o);
            w = make_uint4(__float_as_uint(__uint_as_float(w.x) + a.x), __float_as_uint(__uint_as_float(w.y) + a.y),
                           __float_as_uint(__uint_as_float(w.z) + a.z), __float_as_uint(__uint_as_float(w.w) + a.w));
          }
        }
        *reinterpret_cast<uint4*>(o) = w;
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (j < n) {
            T x = reinterpret_cast<const T*>(from)[j];
            if constexpr (sizeof(T) == 4) {
              if (add) x += o[j];
            }
            o[j] = x;
          }
      }
    }
  } else {
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      T* o = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, mine, r));
      const int n = (rows >> r) & 1 ? valid : 0;
#pragma unroll
      for (int j = lane; j < 128 / (int)sizeof(T); j += 32)
        if (j < n) {
          T x = *reinterpret_cast<const T*>(stage + r * 128 + (((j / kPer) ^ (r & 7)) << 4) + (j % kPer) * sizeof(T));
          if constexpr (sizeof(T) == 4) {
            if (add) x += o[j];
          }
          o[j] = x;
        }
    }
  }
  __syncwarp();
}

// `valid` of 32 neighbouring logits of a row into its running maximum (of z log2 e) and sums; at: the target's place among them
__device__ __forceinline__ void ce_lse_add(float* v, int valid, bool with_z, int at, float* at_target, float& top, float& sum, float& sum_z) {
  if (valid < 32) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j >= valid) v[j] = -INFINITY;
  }
  float m = v[0];
#pragma unroll
  for (int j = 1; j < 32; ++j) m = fmaxf(m, v[j]);
  if (with_z) {
#pragma unroll
    for (int j = 0; j < 32; ++j) sum_z += j < valid ? v[j] : 0.0f;
  }
  if ((unsigned)at < 32u && at < valid) {          // behind the end it is another half's or tile's
    float z = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) z = j == at ? v[j] : z;
    *at_target = z;
  }
  m = fmaxf(top, m * kCeLog2e);
  float s0 = 0.0f, s1 = 0.0f;
  const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    s0 += ce_exp2(fmaf(v[j], kCeLog2e, -ref));
    s1 += ce_exp2(fmaf(v[j + 1], kCeLog2e, -ref));
  }
  sum = sum * ce_exp2(top - ref) + (s0 + s1);
  top = m;
}

// T: the inputs' type.  The operands in shared memory are T, or bfloat16 parts of f32.
template <typename T, int MODE>
__global__ void __launch_bounds__(kCeThreads, 1) __cluster_dims__(2, 1, 1) ce_gemm_kernel(const __grid_constant__ CUtensorMap amap,
                                                                                         const __grid_constant__ CUtensorMap bmap, const CeGemm p) {
  constexpr bool kF32 = sizeof(T) == 4, kAcross = MODE == CE_DH || MODE == CE_DW;      // B is MN-major
  constexpr int kTerms = kF32 ? kCeTerms : 1, kSegment = kF32 ? kCeSegment32 : MODE == CE_FEW ? kCeSegmentFew : kCeSegment16;
  constexpr bool kSums = kF32 || MODE == CE_LSE || MODE == CE_FEW;           // sums in registers
  // few tokens: the second operand is half as long, which makes room for eight stages of the head's bytes
  constexpr int kStages = MODE == CE_FEW ? 8 : kCeStages, kOperandB = MODE == CE_FEW ? kCeOperand / 2 : kCeOperand;
  constexpr int kBufs = MODE == CE_FEW ? 4 : 2, kCols = kCeCols / kBufs;
  constexpr int kChunks = MODE == CE_FEW ? 2 : 4;          // of 32 columns, in a half of a tile
  extern __shared__ uint8_t ce_smem[];
  uint8_t* base = (uint8_t*)(((uintptr_t)ce_smem + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = base;
  uint8_t* sB = base + kStages * kCeOperand;
  __shared__ uint64_t full[kStages], empty[kStages], accf[kBufs], acce[kBufs];
  __shared__ uint32_t tmem_slot;
  const int t = threadIdx.x, warp = __shfl_sync(0xffffffffu, t >> 5, 0), lane = t & 31;
  const uint32_t rank = blockIdx.x & 1;
  const int cid = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (MODE != CE_DW && p.a_rows < 128) {          // rows that no copy fills: zeros draw less power than what an earlier kernel has left there
    for (int i = t; i < kStages * kCeOperand / 16; i += kCeThreads) reinterpret_cast<uint4*>(sA)[i] = make_uint4(0, 0, 0, 0);
    tc::fence_proxy_async();
  }
  if (warp == kCeEpiWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_slot)), "r"(kCeCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (t == 0) {
    for (int i = 0; i < kStages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kBufs; ++i) {
      tc::mbar_init(&accf[i], 1);
      tc::mbar_init(&acce[i], 2 * kCeEpiWarps);
    }
    tc::mbar_fence_init();
  }
  tc::tc_fence_before();
  __syncthreads();
  ce_cluster_sync();                 // both CTAs' barriers exist and both have their TMEM
  tc::tc_fence_after();
  const uint32_t taddr = tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = *p.rows.count;
  const CeTiles<MODE> tiles(p, n, kTerms);
  const int blocks_all = ((MODE == CE_DW ? n : p.depth) + kCeBlock - 1) / kCeBlock;
  // blocks of k that a part of a split tile takes
  auto part = [&](int split, int* b0, int* b1) {
    *b0 = 0;
    *b1 = blocks_all;
    if (MODE == CE_DH) {
      *b0 = (int)((long long)blocks_all * split / tiles.splits);
      *b1 = (int)((long long)blocks_all * (split + 1) / tiles.splits);
    }
  };

  if (warp == kCeEpiWarps) {
    if (tc::elect_one()) {
      bool failed = false;
      int s = 0, issued = 0;
      uint32_t phase = 1;
      for (int tile = cid; tile < tiles.all && !failed; tile += nclusters) {
        int rt, ct, split, b0, b1;
        tiles.at(tile, &rt, &ct, &split);
        part(split, &b0, &b1);
        const int row0 = rt * 256 + (int)rank * 128, col0 = ct * p.tile_n + (int)rank * (p.tile_n >> 1);
        // rows behind the last live one are not copied: what lies in their place meets no other row
        const bool has = MODE == CE_DW || MODE == CE_FEW || row0 < n, other = MODE == CE_DW || MODE == CE_FEW || rt * 256 + 128 < n;
        const uint32_t abytes = MODE == CE_DW ? kCeOperand : (uint32_t)p.a_rows * kCeBlock * 2;
        const uint32_t bytes = abytes * (1 + (other ? 1 : 0)) + 2 * (kAcross ? (uint32_t)kCeOperand : (uint32_t)p.tile_n * kCeBlock);
        for (int kb = b0; kb < b1 && !failed; ++kb) {
          const int k = kb * kCeBlock;
          for (int term = 0; term < kTerms; ++term, ++issued) {
            const int pa = kF32 ? kCeTermA[term] : 0, pb = kF32 ? kCeTermB[term] : 0;
            if (!tc::mbar_wait(&empty[s], phase)) { failed = true; break; }
            const uint32_t bar = ce_map(tc::smem_u32(&full[s]), 0), a = tc::smem_u32(sA + s * kCeOperand), b = tc::smem_u32(sB + s * kOperandB);
            if (rank == 0) tc::mbar_arrive_expect_tx(&full[s], bytes);
            if (MODE == CE_DW) {
              ce_load(a, &amap, row0, k, pa, bar);
              ce_load(a + 8192, &amap, row0 + 64, k, pa, bar);
            } else if (MODE == CE_FEW) {
              ce_load(a, &amap, k, p.w_row + (rt * 2 + (int)rank) * p.a_rows, pa, bar);
            } else if (has) {
              ce_load(a, &amap, k, row0, pa, bar);
            }
            if (kAcross) {
              const int kw = MODE == CE_DH ? p.w_row + k : k;
              ce_load(b, &bmap, col0, kw, pb, bar);
              ce_load(b + 8192, &bmap, col0 + 64, kw, pb, bar);
            } else {
              ce_load(b, &bmap, k, MODE == CE_FEW ? col0 : p.w_row + col0, pb, bar);
            }
            if (++s == kStages) { s = 0; phase ^= 1; }
          }
        }
      }
      if (rank == 0) tc::mbar_drain(full, issued, kStages);      // both CTAs' copies; the other one waits at the barrier below
    }
  } else if (warp == kCeEpiWarps + 1) {
    if (rank == 0 && tc::elect_one()) {
      constexpr uint32_t fmt = sizeof(T) == 2 && __is_same(T, __half) ? tc::FMT_F16 : tc::FMT_BF16;
      const uint32_t idesc = tc::idesc_f32acc(fmt, fmt, 256, (uint32_t)p.tile_n) | (MODE == CE_DW ? 1u << 15 : 0u) | (kAcross ? 1u << 16 : 0u);
      struct Issue {
        uint8_t *sA, *sB;
        uint64_t *full, *empty, *accf, *acce;
        uint32_t taddr, idesc, phase;
        int s;
        __device__ __forceinline__ bool wait_acc(int ab, uint32_t parity) {
          const bool ok = tc::mbar_wait(&acce[ab], parity);
          tc::tc_fence_after();
          return ok;
        }
        __device__ __forceinline__ bool wait_full() {
          const bool ok = tc::mbar_wait(&full[s], phase);
          tc::tc_fence_after();
          return ok;
        }
        __device__ __forceinline__ void product(int ab, bool first) {
          const uint32_t a = tc::smem_u32(sA + s * kCeOperand), b = tc::smem_u32(sB + s * kOperandB);
          const uint64_t da = MODE == CE_DW ? ce_desc_mn(a) : tc::smem_desc_sw128(a), db = kAcross ? ce_desc_mn(b) : tc::smem_desc_sw128(b);
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k)
            ce_mma(taddr + ab * kCols, da + (MODE == CE_DW ? 128 : 2) * k, db + (kAcross ? 128 : 2) * k, idesc, !first || k > 0);
          ce_commit(&empty[s]);
          if (++s == kStages) { s = 0; phase ^= 1; }
        }
        __device__ __forceinline__ void commit_acc(int ab) { ce_commit(&accf[ab]); }
      } issue = {sA, sB, full, empty, accf, acce, taddr, idesc, 0, 0};
      bool ok = true;
      int seg = 0;
      for (int tile = cid; tile < tiles.all && ok; tile += nclusters) {
        int rt, ct, split, b0, b1;
        tiles.at(tile, &rt, &ct, &split);
        part(split, &b0, &b1);
        ok = ce_issue<kBufs, kSums ? kSegment : 0>(issue, b0, b1, kTerms, &seg);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = warp >> 2, middle = ((p.tile_n >> 1) + 31) & ~31;      // a half's columns: 0 .. middle, middle .. tile_n
    uint8_t* stage = base + kStages * (kCeOperand + kOperandB) + warp * kCeStage;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t drained = ce_map(tc::smem_u32(&acce[0]), 0);
    bool failed = false;
    int seg = 0;
    float few_top[2], few_sum[2], few_z[2];          // FEW: a thread's tokens, over all tiles
    int few_target[2];
    if (MODE == CE_FEW) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int token = (half ? middle : 0) + 32 * i + lane;
        few_top[i] = -INFINITY;
        few_sum[i] = few_z[i] = 0.0f;
        few_target[i] = token < n ? p.rows.target[token] : -1;
      }
    }
    for (int tile = cid; tile < tiles.all; tile += nclusters) {
      int rt, ct, split, b0, b1;
      tiles.at(tile, &rt, &ct, &split);
      part(split, &b0, &b1);
      const int row = rt * 256 + (int)rank * 128 + quarter * 32 + lane, col0 = ct * p.tile_n, cols = MODE == CE_FEW ? p.tile_n : min(p.tile_n, p.columns - col0);
      const bool live = row < (MODE == CE_DW ? p.m : n);
      // what a row brings
      float lse2 = 0.0f, f = 0.0f, scale = 0.0f;
      int target = -1;
      if (MODE == CE_LSE || MODE == CE_DZ) {
        if (live) target = p.rows.target[row] - p.c0 - col0;
        if (MODE == CE_DZ && live) {
          lse2 = p.rows.lse2[row];
          f = ce_up_factor(p.up, p.rows, row);
        }
      } else if (MODE != CE_FEW) {
        scale = ce_up_scale(p.up, n);
      }
      float top = -INFINITY, sum = 0.0f, sum_z = 0.0f;

      // 16-bit rows go out 64 columns at a time, the last 32 of a half alone
      const int begin = half ? middle : 0, end = min(cols, half ? p.tile_n : middle);
      auto put16 = [&](const float* v, int c0, T* o, bool ok) {
        if constexpr (!kF32) {
          const int odd = ((c0 - begin) >> 5) & 1, first = c0 - 32 * odd;
          ce_stage<T>(stage, lane, 4 * odd, v);
          if (odd || c0 + 32 >= end) ce_flush<T>(stage, lane, o + first, ok, min(32 + 32 * odd, end - first));
        }
      };
      auto finish = [&](float* v, int c0) {      // columns c0 .. c0 + 31 of the tile
        const int valid = end - c0;
        if (failed) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = NAN;
        }
        if constexpr (MODE == CE_LSE) {
          ce_lse_add(v, valid, p.smoothing != 0.0f, target - c0, p.at_target + row, top, sum, sum_z);
        } else if constexpr (MODE == CE_FEW) {
          // the tile's rows are the head's: transposed through shared memory, a thread has a token's logits of 32 rows
          ce_stage<float>(stage, lane, 0, v);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = *reinterpret_cast<const float*>(stage + j * 128 + (((lane >> 2) ^ (j & 7)) << 4) + (lane & 3) * 4);
          __syncwarp();
          const int i = (c0 - begin) >> 5, v0 = (rt * 2 + (int)rank) * p.a_rows + quarter * 32, inside = min(p.a_rows - quarter * 32, p.columns - v0);
          if (inside > 0) ce_lse_add(v, inside, p.smoothing != 0.0f, few_target[i] - p.c0 - v0, p.at_target + begin + 32 * i + lane, few_top[i], few_sum[i], few_z[i]);
        } else if constexpr (MODE == CE_DZ) {
          const float even = p.smoothing / (float)p.vocab, up = f * p.up.dz_scale;
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = up * (ce_exp2(fmaf(v[j], kCeLog2e, -lse2)) - even);
          if ((unsigned)(target - c0) < 32u) {
            const float q = up * (1.0f - p.smoothing);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] -= j == target - c0 ? q : 0.0f;
          }
          if (!live) {          // up to the end of the tile: rows are a product's k
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.0f;
          }
          uint16_t* o = p.dz + (long long)row * p.ldz + col0;
          if constexpr (!kF32) {
            put16(v, c0, reinterpret_cast<T*>(o), true);
          } else {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              ce_store32(reinterpret_cast<__nv_bfloat16*>(o + c0 + k * p.plane), v, valid);
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float a = __bfloat162float(__float2bfloat16_rn(v[j]));
                v[j] = isfinite(a) ? v[j] - a : 0.0f;
              }
            }
          }
        } else if constexpr (MODE == CE_DH) {
          float* acc = p.acc + ((long long)split * ((n + 255) & ~255) + row) * p.columns + col0 + c0;
          if (tiles.splits == 1 && p.last) {
            if (!p.first && live) {
              if (valid >= 32 && (reinterpret_cast<uintptr_t>(acc) & 15) == 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const float4 a = reinterpret_cast<const float4*>(acc)[j];
                  v[4 * j] += a.x; v[4 * j + 1] += a.y; v[4 * j + 2] += a.z; v[4 * j + 3] += a.w;
                }
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (j < valid) v[j] += acc[j];
              }
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= scale;
            T* o = (T*)p.out + (long long)(live ? p.rows.index[row] : 0) * p.columns + col0;
            if constexpr (!kF32) {
              put16(v, c0, o, live);
            } else {
              ce_stage<float>(stage, lane, 0, v);
              ce_flush<float>(stage, lane, o + c0, live, min(32, valid));
            }
          } else {
            ce_stage<float>(stage, lane, 0, v);
            ce_flush<float>(stage, lane, acc, live, min(32, valid), !p.first);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= scale;
          T* o = (T*)p.out + (long long)(p.c0 + row) * p.columns + col0;
          if constexpr (!kF32) {
            put16(v, c0, o, live);
          } else {
            ce_stage<float>(stage, lane, 0, v);
            ce_flush<float>(stage, lane, o + c0, live, min(32, valid));
          }
        }
      };

      if constexpr (kSums) {
        float acc[kChunks][32];
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[i][j] = 0.0f;
#pragma unroll 1
        for (int k0 = b0; k0 < b1; k0 += kSegment, ++seg) {
          const int ab = seg % kBufs;
          if (!failed && !tc::mbar_wait_warp<64>(&accf[ab], (seg / kBufs) & 1, lane)) failed = true;
          tc::tc_fence_after();
#pragma unroll
          for (int i = 0; i < kChunks; ++i) {
            if (begin + 32 * i < end) {
              uint32_t r[32];
              tc::tmem_ld32(taddr + lane_base + ab * kCols + begin + 32 * i, r);
              tc::tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) acc[i][j] += __uint_as_float(r[j]);
            }
          }
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) ce_arrive_at(drained + ab * 8);
        }
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
          if (begin + 32 * i < end) finish(acc[i], begin + 32 * i);
      } else {
        const bool none = b0 == b1;            // an empty sum: no live row
        const int ab = seg % kBufs;
        if (!none && !failed && !tc::mbar_wait_warp<64>(&accf[ab], (seg / kBufs) & 1, lane)) failed = true;
        tc::tc_fence_after();
#pragma unroll 1
        for (int c0 = begin; c0 < end; c0 += 32) {
          uint32_t r[32];
          float v[32];
          tc::tmem_ld32(taddr + lane_base + ab * kCols + c0, r);
          tc::tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = none ? 0.0f : __uint_as_float(r[j]);
          finish(v, c0);
        }
        if (!none) {
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) ce_arrive_at(drained + ab * 8);
          ++seg;
        }
      }
      if (MODE == CE_LSE && live) {
        const long long at = (long long)(p.slot + 2 * ct + half) * p.ldn + row;
        p.part_m[at] = top;
        p.part_s[at] = sum;
        if (p.smoothing != 0.0f) p.part_z[at] = sum_z;
      }
    }
    if (MODE == CE_FEW) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int token = (half ? middle : 0) + 32 * i + lane;
        const long long at = (long long)(p.slot + (cid * 2 + (int)rank) * 4 + quarter) * p.ldn + token;
        if (token < n && token < (half ? p.tile_n : middle)) {
          p.part_m[at] = few_top[i];
          p.part_s[at] = few_sum[i];
          if (p.smoothing != 0.0f) p.part_z[at] = few_z[i];
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncwarp();
  ce_cluster_sync();                 // nobody leaves while the other CTA may still read its shared memory or TMEM, or signal it
  tc::tc_fence_after();
  if (warp == kCeEpiWarps + 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(kCeCols) : "memory");
}

// ---- joining ----------------------------------------------------------------------------------------------------------------------------
// Sixteen rows a block (64 bytes of every slot's line), 32 threads for a row's slots; then the row's loss.  The last block to finish
// adds up the rows, in their order.
constexpr int kCeMergeRows = 16, kCeMergeLanes = 32;
__global__ void __launch_bounds__(kCeMergeRows * kCeMergeLanes) ce_merge_kernel(CeRows r, const float* part_m, const float* part_s,
                                                                               const float* part_z, const float* at_target, long long ldn, int slots,
                                                                               int vocab, float smoothing, int reduce, float* row_loss, float* loss) {
  __shared__ float sm[kCeMergeLanes][kCeMergeRows];
  __shared__ double ss[kCeMergeLanes][kCeMergeRows], sz[kCeMergeLanes][kCeMergeRows];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int i = threadIdx.x % kCeMergeRows, l = threadIdx.x / kCeMergeRows, row = blockIdx.x * kCeMergeRows + i, n = *r.count;
  const int blocks = n > 0 ? (n + kCeMergeRows - 1) / kCeMergeRows : 1;
  if (blockIdx.x >= blocks) return;
  float top = -INFINITY;
  double s = 0.0, z = 0.0;
  if (row < n) {
    constexpr int U = 8;
    for (int k = l; k < slots; k += U * kCeMergeLanes) {
      float m[U], e[U], m8 = top, s8 = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int q = k + u * kCeMergeLanes;
        m[u] = q < slots ? part_m[q * ldn + row] : -INFINITY;
        e[u] = q < slots ? part_s[q * ldn + row] : 0.0f;
        if (smoothing != 0.0f && q < slots) z += (double)part_z[q * ldn + row];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) m8 = fmaxf(m8, m[u]);
      const float ref = m8 == -INFINITY ? 0.0f : m8;
#pragma unroll
      for (int u = 0; u < U; ++u) s8 += e[u] * ce_exp2(m[u] - ref);
      s = s * (double)ce_exp2(top - ref) + (double)s8;
      top = m8;
    }
  }
  sm[l][i] = top;
  ss[l][i] = s;
  sz[l][i] = z;
  for (int o = kCeMergeLanes / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (l < o) {
      const float a = sm[l][i], b = sm[l + o][i], m = fmaxf(a, b), ref = m == -INFINITY ? 0.0f : m;
      ss[l][i] = ss[l][i] * (double)ce_exp2(a - ref) + ss[l + o][i] * (double)ce_exp2(b - ref);
      sz[l][i] += sz[l + o][i];
      sm[l][i] = m;
    }
  }
  if (l == 0 && row < n) {
    const double lse2 = (double)sm[0][i] + log2(ss[0][i]);
    r.lse2[row] = (float)lse2;
    double x = lse2 * 0.69314718055994530942 - (double)(1.0f - smoothing) * (double)at_target[row];
    if (smoothing != 0.0f) x -= (double)smoothing * sz[0][i] / vocab;
    if (r.target[row] < 0) x = NAN;
    if (reduce == CE_NONE)
      loss[r.index[row]] = (float)x;
    else
      row_loss[row] = (float)x;
  }
  if (reduce == CE_NONE) return;
  __shared__ int last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(r.count + 1, 1) == blocks - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double v = 0.0;
  for (int k = threadIdx.x; k < n; k += kCeMergeRows * kCeMergeLanes) v += (double)__ldcg(row_loss + k);
  double* sums = &ss[0][0];
  sums[threadIdx.x] = v;
  for (int o = kCeMergeRows * kCeMergeLanes / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (threadIdx.x < o) sums[threadIdx.x] += sums[threadIdx.x + o];
  }
  if (threadIdx.x == 0) *loss = (float)(reduce == CE_MEAN ? sums[0] / (double)n : sums[0]);
}

// max |u| over the live rows whose u is finite: an infinite one, as a NaN, is for its own row alone
__global__ void __launch_bounds__(1024) ce_top_kernel(CeRows r, const float* up, float* out) {
  __shared__ float s[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = *r.count;
  float top = 0.0f;
  for (int i = threadIdx.x; i < n; i += 1024) {
    const float u = fabsf(up[r.index[i]]);
    if (u < INFINITY) top = fmaxf(top, u);
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = top;
  __syncthreads();
  top = warp_max(s[threadIdx.x & 31]);
  if (threadIdx.x == 0) *out = top;
}

// dh: zeros for ignored rows, and the parts' sums where there are several
template <typename T>
__global__ void __launch_bounds__(256) ce_join_kernel(CeRows r, CeUp u, const float* acc, int rows, int piece_blocks, int terms, int clusters, int acc_rows,
                                                      int width, T* out) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = *r.count, splits = ce_splits(n, width, piece_blocks, terms, clusters, acc_rows);
  if (splits == 1 && n == rows) return;          // the product has stored its tiles itself
  const float f = ce_up_scale(u, n);
  const int fours = (width + 3) >> 2;
  const bool wide = (width & 3) == 0;
  const long long ldn = (n + 255) & ~255, all = (long long)rows * fours;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
    const int row = (int)(i / fours), d = (int)(i % fours) * 4, at = r.place[row];
    if (at >= 0 && splits == 1) continue;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (at >= 0) {
#pragma unroll 4
      for (int k = 0; k < splits; ++k) {
        const float* a = acc + (k * ldn + at) * width + d;
        if (wide) {
          const float4 q = *reinterpret_cast<const float4*>(a);
          v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (d + j < width) v[j] += a[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= f;
    }
    T* o = out + (long long)row * width + d;
    if (wide && sizeof(T) == 2) {
      __align__(8) T w[4] = {T(v[0]), T(v[1]), T(v[2]), T(v[3])};
      *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(w);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d + j < width) o[j] = T(v[j]);
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------
struct CeArgs {
  const void *hidden, *weight;
  const long long* targets;
  long long ldh, ldw, ignore;
  int rows, vocab, width, type, reduce;
  float smoothing;
  CeRows live;
  uint16_t* x;          // the live rows side by side, kept between the calls
  float* loss;
  const float* up;
  void *dhidden, *dweight;
  uint8_t* ws;
};

struct CePlan {
  int planes, ldd, padded, tile_v, clusters;
  bool few;                    // the loss by CE_FEW
  bool rows32;                 // f32 by the few-rows kernels
  bool packed;                 // the head is copied piece by piece: f32, or rows that TMA cannot take
  int piece, pieces, acc_rows;
  long long lists, kept;       // bytes of one of the live rows' lists, and of all that the forward call keeps for the backward one
  long long w, parts, part, rows, dz, acc, bytes;      // places in the workspace, and its size
};

static long long ce_up_to(long long v, long long unit) { return (v + unit - 1) / unit * unit; }

static int ce_sms() {
  int dev = 0, sms = 148;
  // the driver encodes tensor maps in the calling thread's context, and a thread that has launched nothing yet (autograd's) has none
  if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Vocabulary rows of a tile: the fewest rounds of tiles times the cycles of a block of k, 2 per column on the tensor core or the copies at
// some 70 bytes a cycle, whichever is longer.
static int ce_tile_columns(int rows, int vocab, int clusters) {
  const long long row_tiles = (rows + 255) / 256;
  const long long a_bytes = (rows < 128 ? rows : 128) * 128;
  int best = 256;
  long long best_cost = -1;
  for (int tn = 256; tn >= 128; tn -= 16) {
    const long long tiles = row_tiles * ((vocab + tn - 1) / tn), rounds = (tiles + clusters - 1) / clusters;
    const long long tensor = 2 * tn, copies = (a_bytes + 64 * tn) / 70, cost = rounds * ((tensor > copies ? tensor : copies) + 16);
    if (best_cost < 0 || cost < best_cost) {
      best_cost = cost;
      best = tn;
    }
  }
  return best;
}

static CePlan ce_plan(const CeArgs& a, bool backward) {
  CePlan p = {};
  p.planes = a.type == CE_F32 ? 3 : 1;
  p.ldd = (int)ce_up_to(a.width, 8);
  p.padded = (int)ce_up_to(a.rows, 256);
  p.clusters = ce_sms() / 2 < 1 ? 1 : ce_sms() / 2;
  p.rows32 = a.type == CE_F32 && a.rows <= kCeFew32;
  p.packed = (p.planes == 3 && !p.rows32) || a.ldw % 8 != 0 || (reinterpret_cast<uintptr_t>(a.weight) & 15) != 0;
  // pieces of the vocabulary: half a gigabyte of dz and of the copied head, at least 4096 rows
  long long most = ce_up_to(a.vocab, 256);
  const long long room = 1ll << 29;
  if (backward && room / (2ll * p.planes * p.padded) < most) most = room / (2ll * p.planes * p.padded);
  if (p.packed && room / (2ll * p.planes * p.ldd) < most) most = room / (2ll * p.planes * p.ldd);
  if (most < 4096) most = 4096;
  p.pieces = (int)((a.vocab + most - 1) / most);
  p.piece = (int)ce_up_to((a.vocab + p.pieces - 1) / p.pieces, 256);
  p.pieces = (a.vocab + p.piece - 1) / p.piece;
  p.tile_v = ce_tile_columns(a.rows, p.piece < a.vocab ? p.piece : a.vocab, p.clusters);
  p.acc_rows = p.padded + 4096;
  const long long planes = p.rows32 ? 2 : p.planes;      // 16-bit words of a kept value
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long place = at;
    at = ce_up_to(at + bytes, 1024);
    return place;
  };
  p.lists = ce_up_to(4ll * a.rows, 256);
  p.kept = 256 + 4 * p.lists + 2 * planes * p.padded * p.ldd;
  if (p.rows32) {
    p.rows = take(8ll * p.padded);
    if (!backward) {
      p.parts = ce_few_loss_slots();
      p.part = take(12ll * p.parts * p.padded);
    } else {
      p.dz = take(4ll * a.rows * ce_up_to(a.vocab, 4));
      if (a.dhidden != nullptr) p.acc = take(4ll * ce_few_slots(a.width) * a.rows * a.width);
    }
    p.bytes = at;
    return p;
  }
  p.w = p.packed ? take(2ll * p.planes * p.piece * p.ldd) : 0;
  p.rows = take(8ll * p.padded);                       // forward: z at the target, the rows' losses; backward: max |u|
  if (!backward) {
    p.few = a.rows <= kCeFew;
    p.parts = p.few ? 8ll * p.clusters * p.pieces : 2ll * p.pieces * ((p.piece + p.tile_v - 1) / p.tile_v);
    p.part = take((a.smoothing != 0.0f ? 12ll : 8ll) * p.parts * p.padded);
  } else {
    p.dz = take(2ll * p.planes * p.padded * p.piece);
    if (a.dhidden != nullptr) p.acc = take(4ll * p.acc_rows * a.width);
  }
  p.bytes = at;
  return p;
}

static bool ce_tensor_map(CUtensorMap* map, const void* base, int type, long long inner, long long rows, long long ld, int planes, long long plane, int box_x, int box_y) {
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(planes > 1 ? plane * 2 : ld * 2)};
  cuuint32_t box[3] = {(cuuint32_t)box_x, (cuuint32_t)box_y, 1}, estr[3] = {1, 1, 1};
  return cuTensorMapEncodeTiled(map, type == CE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims,
                                strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int MODE>
static cudaError_t ce_launch(const CUtensorMap& am, const CUtensorMap& bm, const CeGemm& g, long long tiles, int clusters, cudaStream_t st) {
  const size_t smem = 1024 + (size_t)kCeStages * 2 * kCeOperand + kCeEpiWarps * kCeStage;
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(ce_gemm_kernel<T, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return launch_pdl(ce_gemm_kernel<T, MODE>, dim3(2 * (unsigned)(tiles < clusters ? tiles : clusters)), dim3(kCeThreads), smem, st, am, bm, g);
}

template <typename T, bool kPlain = false>
static cudaError_t ce_pack(const void* src, long long ld, long long row0, int rows, const int* count, const int* index, int width, void* dst, int ldd,
                           long long plane, cudaStream_t st) {
  const long long words = ce_up_to(rows, count != nullptr ? 256 : 1) * (ldd >> 3), blocks = (words + 255) / 256;
  return launch_pdl(ce_pack_kernel<T, kPlain>, dim3((unsigned)(blocks < 148 * 16 ? blocks : 148 * 16)), dim3(256), 0, st, (const T*)src, ld, row0, rows, count, index,
                    width, (uint16_t*)dst, ldd, plane);
}

// What the logits' product takes: maps of the live rows and of a piece's rows of the head.
struct CeLogits {
  CUtensorMap x, w;
  int w_row;             // the piece's first row in its map
};

template <typename T>
static bool ce_head_piece(const CeArgs& a, const CePlan& p, int c0, int rows, int box_x, int box_y, CUtensorMap* map, int* w_row) {
  if (p.packed) {
    *w_row = 0;
    return ce_tensor_map(map, a.ws + p.w, a.type, a.width, rows, p.ldd, p.planes, (long long)p.piece * p.ldd, box_x, box_y);
  }
  *w_row = c0;
  return ce_tensor_map(map, a.weight, a.type, a.width, c0 + rows, a.ldw, 1, 0, box_x, box_y);
}

static cudaError_t ce_merge(const CeArgs& a, const CePlan& p, const float* part_m, const float* part_s, const float* part_z, int slots, const float* at_target,
                            float* row_loss, cudaStream_t st) {
  return launch_pdl(ce_merge_kernel, dim3((a.rows + kCeMergeRows - 1) / kCeMergeRows), dim3(kCeMergeRows * kCeMergeLanes), 0, st, a.live, part_m, part_s, part_z,
                    at_target, (long long)p.padded, slots, a.vocab, a.smoothing, a.reduce, row_loss, a.loss);
}

static CeFewArgs ce_few_args(const CeArgs& a, const CePlan& p) {
  CeFewArgs f = {};
  f.rows = a.live; f.weight = a.weight; f.x = a.x; f.ldw = a.ldw; f.ldx = p.ldd;
  f.vocab = a.vocab; f.width = a.width; f.tokens = a.rows; f.smoothing = a.smoothing; f.row_count = a.rows;
  return f;
}

template <typename T>
static int ce_forward(const CeArgs& a, const CePlan& p, cudaStream_t st) {
  float *at_target = (float*)(a.ws + p.rows), *row_loss = at_target + p.padded;
  float* part = (float*)(a.ws + p.part);
  float* each = a.reduce == CE_NONE ? a.loss : nullptr;
  cudaError_t e = launch_pdl(ce_rows_kernel, dim3(1), dim3(1024), 0, st, a.targets, a.rows, a.vocab, a.ignore, a.live, each);
  if (p.rows32) {
    if (e == cudaSuccess) e = ce_pack<T, true>(a.hidden, a.ldh, 0, a.rows, a.live.count, a.live.index, a.width, a.x, p.ldd, 0, st);
    CeFewArgs f = ce_few_args(a, p);
    f.part_m = part; f.part_s = part + p.parts * p.padded; f.part_z = part + 2 * p.parts * p.padded; f.at_target = at_target; f.ldn = p.padded;
    if (e == cudaSuccess) e = ce_few_loss(f, st);
    if (e == cudaSuccess) e = ce_merge(a, p, f.part_m, f.part_s, f.part_z, (int)p.parts, at_target, row_loss, st);
    return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
  }
  if (e == cudaSuccess)
    e = ce_pack<T>(a.hidden, a.ldh, 0, a.rows, a.live.count, a.live.index, a.width, a.x, p.ldd, (long long)p.padded * p.ldd, st);
  CeGemm g = {};
  g.rows = a.live; g.depth = a.width; g.tile_n = p.tile_v; g.a_rows = a.rows < 128 ? (int)ce_up_to(a.rows, 8) : 128;
  g.vocab = a.vocab; g.smoothing = a.smoothing; g.ldn = p.padded;
  g.part_m = part; g.part_s = part + p.parts * p.padded; g.part_z = part + 2 * p.parts * p.padded; g.at_target = at_target;
  CUtensorMap xm, wm;
  if (p.few) g.tile_n = (int)ce_up_to(a.rows, 16);
  if (!ce_tensor_map(&xm, a.x, a.type, a.width, p.padded, p.ldd, p.planes, (long long)p.padded * p.ldd, kCeBlock, p.few ? g.tile_n / 2 : g.a_rows))
    return BONSAI_CUDA_BAD_ARG;
  for (int c0 = 0; c0 < a.vocab && e == cudaSuccess; c0 += p.piece) {
    const int rows = a.vocab - c0 < p.piece ? a.vocab - c0 : p.piece;
    if (p.packed) e = ce_pack<T>(a.weight, a.ldw, c0, rows, nullptr, nullptr, a.width, a.ws + p.w, p.ldd, (long long)p.piece * p.ldd, st);
    if (e != cudaSuccess) break;
    g.c0 = c0; g.columns = rows;
    if (p.few) {          // rows of the head in a tile: the clusters have whole rounds of them
      const int rounds = (rows + 256 * p.clusters - 1) / (256 * p.clusters), tiles = rounds * p.clusters;
      g.a_rows = (int)ce_up_to((rows + 2 * tiles - 1) / (2 * tiles), 8);
      if (!ce_head_piece<T>(a, p, c0, rows, kCeBlock, g.a_rows, &wm, &g.w_row)) return BONSAI_CUDA_BAD_ARG;
      const int launched = (rows + 2 * g.a_rows - 1) / (2 * g.a_rows) < p.clusters ? (rows + 2 * g.a_rows - 1) / (2 * g.a_rows) : p.clusters;
      e = ce_launch<T, CE_FEW>(wm, xm, g, launched, p.clusters, st);
      g.slot += 8 * launched;
      continue;
    }
    if (!ce_head_piece<T>(a, p, c0, rows, kCeBlock, p.tile_v / 2, &wm, &g.w_row)) return BONSAI_CUDA_BAD_ARG;
    const int ct = (rows + p.tile_v - 1) / p.tile_v;
    e = ce_launch<T, CE_LSE>(xm, wm, g, (long long)(p.padded / 256) * ct, p.clusters, st);
    g.slot += 2 * ct;
  }
  if (e == cudaSuccess) e = ce_merge(a, p, g.part_m, g.part_s, g.part_z, g.slot, at_target, row_loss, st);
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

template <typename T>
static int ce_backward(const CeArgs& a, const CePlan& p, cudaStream_t st) {
  float* top = (float*)(a.ws + p.rows);
  const CeUp up = {a.up, top, a.reduce, a.type == CE_F16 ? 32768.0f : 1.0f};
  cudaError_t e = cudaSuccess;
  if (a.reduce == CE_NONE) e = launch_pdl(ce_top_kernel, dim3(1), dim3(1024), 0, st, a.live, a.up, top);
  if (p.rows32) {
    CeFewArgs f = ce_few_args(a, p);
    f.up = CeUp{a.up, top, a.reduce, 1.0f};
    f.dz = (float*)(a.ws + p.dz); f.ldz = ce_up_to(a.vocab, 4); f.part = (float*)(a.ws + p.acc); f.dhidden = a.dhidden; f.dweight = a.dweight;
    if (e == cudaSuccess) e = ce_few_gradients(f, st);
    return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
  }
  const long long x_plane = (long long)p.padded * p.ldd, z_plane = (long long)p.padded * p.piece;
  CeGemm g = {};
  g.rows = a.live; g.vocab = a.vocab; g.smoothing = a.smoothing; g.ldn = p.padded; g.up = up;
  g.a_rows = a.rows < 128 ? (int)ce_up_to(a.rows, 8) : 128;
  g.dz = (uint16_t*)(a.ws + p.dz); g.ldz = p.piece; g.plane = z_plane; g.piece_blocks = p.piece / kCeBlock; g.clusters = p.clusters;
  g.acc_rows = p.acc_rows; g.acc = (float*)(a.ws + p.acc);
  CUtensorMap xm, wm, zm;
  for (int c0 = 0; c0 < a.vocab && e == cudaSuccess; c0 += p.piece) {
    const int rows = a.vocab - c0 < p.piece ? a.vocab - c0 : p.piece;
    if (p.packed) e = ce_pack<T>(a.weight, a.ldw, c0, rows, nullptr, nullptr, a.width, a.ws + p.w, p.ldd, (long long)p.piece * p.ldd, st);
    if (e != cudaSuccess) break;
    g.c0 = c0;
    if (!ce_tensor_map(&xm, a.x, a.type, a.width, p.padded, p.ldd, p.planes, x_plane, kCeBlock, g.a_rows) ||
        !ce_head_piece<T>(a, p, c0, rows, kCeBlock, p.tile_v / 2, &wm, &g.w_row))
      return BONSAI_CUDA_BAD_ARG;
    g.columns = rows; g.depth = a.width; g.tile_n = p.tile_v;
    e = ce_launch<T, CE_DZ>(xm, wm, g, (long long)(p.padded / 256) * ((rows + p.tile_v - 1) / p.tile_v), p.clusters, st);
    g.columns = a.width; g.tile_n = 256;
    const long long ct = (a.width + 255) / 256;
    if (e == cudaSuccess && a.dhidden != nullptr) {
      if (!ce_tensor_map(&zm, a.ws + p.dz, a.type, rows, p.padded, p.piece, p.planes, z_plane, kCeBlock, g.a_rows) ||
          !ce_head_piece<T>(a, p, c0, rows, 64, kCeBlock, &wm, &g.w_row))
        return BONSAI_CUDA_BAD_ARG;
      g.depth = rows; g.first = c0 == 0; g.last = c0 + rows == a.vocab; g.out = a.dhidden;
      e = ce_launch<T, CE_DH>(zm, wm, g, p.clusters, p.clusters, st);
    }
    if (e == cudaSuccess && a.dweight != nullptr) {
      if (!ce_tensor_map(&zm, a.ws + p.dz, a.type, rows, p.padded, p.piece, p.planes, z_plane, 64, kCeBlock) ||
          !ce_tensor_map(&xm, a.x, a.type, a.width, p.padded, p.ldd, p.planes, x_plane, 64, kCeBlock))
        return BONSAI_CUDA_BAD_ARG;
      g.m = rows; g.out = a.dweight;
      e = ce_launch<T, CE_DW>(zm, xm, g, (rows + 255) / 256 * ct, p.clusters, st);
    }
  }
  if (e == cudaSuccess && a.dhidden != nullptr) {
    const long long blocks = ((long long)a.rows * ((a.width + 3) / 4) + 255) / 256;
    e = launch_pdl(ce_join_kernel<T>, dim3((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8)), dim3(256), 0, st, a.live, up, (const float*)g.acc, a.rows, g.piece_blocks,
                   p.planes == 3 ? kCeTerms : 1, p.clusters, p.acc_rows, a.width, (T*)a.dhidden);
  }
  return e == cudaSuccess ? BONSAI_CUDA_OK : BONSAI_CUDA_LAUNCH_FAILED;
}

// Below 2^30 the sum of a row's number and a piece's or a tile's rows fits an int.
static bool ce_good(const CeArgs& a) {
  constexpr int most = 1 << 30;
  return a.weight != nullptr && a.rows >= 1 && a.vocab >= 1 && a.width >= 1 && a.ldw >= a.width && a.rows < most && a.vocab < most && a.width < most &&
         a.type >= CE_F32 && a.type <= CE_BF16 && a.reduce >= CE_MEAN && a.reduce <= CE_NONE;
}

static CeArgs ce_args(const void* weight, long long ldw, int rows, int vocab, int width, int type, int reduce, float smoothing, void* kept, void* ws) {
  CeArgs a = {};
  a.weight = weight; a.ldw = ldw;
  a.rows = rows; a.vocab = vocab; a.width = width; a.type = type; a.reduce = reduce; a.smoothing = smoothing;
  a.ws = (uint8_t*)ws;
  if (kept != nullptr && rows > 0) {
    uint8_t* at = (uint8_t*)kept + 256;
    const long long lists = ce_up_to(4ll * rows, 256);
    a.live = CeRows{(int*)kept, (int*)at, (int*)(at + lists), (int*)(at + 2 * lists), (float*)(at + 3 * lists)};
    a.x = (uint16_t*)(at + 4 * lists);
  }
  return a;
}

}  // namespace bonsai

extern "C" {

// Bytes for the calls below with these arguments: of what the forward call keeps for the backward one (what 0), of the forward call's workspace (1),
// of the backward call's without and with dhidden (2, 3); -1 for arguments that are refused.
long long bonsai_ce_bytes(const void* weight, long long ldw, int rows, int vocab, int width, int type, float smoothing, int what) {
  using namespace bonsai;
  CeArgs a = ce_args(weight, ldw, rows, vocab, width, type, CE_MEAN, smoothing, nullptr, nullptr);
  a.dhidden = what == 3 ? const_cast<void*>(weight) : nullptr;
  if (!ce_good(a) || what < 0 || what > 3) return -1;
  const CePlan p = ce_plan(a, what >= 2);
  return what == 0 ? p.kept : p.bytes;
}

// hidden [rows][ldh], weight [vocab][ldw] of one type (0 f32, 1 f16, 2 bf16), targets [rows].  loss: one f32, or one for each row (reduce 2).
// kept, ws: 256-byte aligned.
int bonsai_ce_forward(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* targets, int rows, int vocab, int width,
                      int type, long long ignore, int reduce, float smoothing, void* kept, long long kept_bytes, float* loss, void* ws, long long ws_bytes,
                      cudaStream_t st) {
  using namespace bonsai;
  CeArgs a = ce_args(weight, ldw, rows, vocab, width, type, reduce, smoothing, kept, ws);
  a.hidden = hidden; a.ldh = ldh; a.targets = targets; a.ignore = ignore; a.loss = loss;
  if (!ce_good(a) || hidden == nullptr || ldh < width || targets == nullptr || loss == nullptr || kept == nullptr || ws == nullptr ||
      ((reinterpret_cast<uintptr_t>(ws) | reinterpret_cast<uintptr_t>(kept)) & 255) != 0)
    return BONSAI_CUDA_BAD_ARG;
  const CePlan p = ce_plan(a, false);
  if (kept_bytes < p.kept || ws_bytes < p.bytes) return BONSAI_CUDA_BAD_ARG;
  return type == CE_F32 ? ce_forward<float>(a, p, st) : type == CE_F16 ? ce_forward<__half>(a, p, st) : ce_forward<__nv_bfloat16>(a, p, st);
}

// kept: from the forward call.  up: d loss, one f32 or one for each row.  dhidden [rows][width], dweight [vocab][width] of the inputs' type; null: not
// wanted.
int bonsai_ce_backward(const void* weight, long long ldw, int rows, int vocab, int width, int type, int reduce, float smoothing, void* kept,
                       long long kept_bytes, const float* up, void* dhidden, void* dweight, void* ws, long long ws_bytes, cudaStream_t st) {
  using namespace bonsai;
  CeArgs a = ce_args(weight, ldw, rows, vocab, width, type, reduce, smoothing, kept, ws);
  a.up = up; a.dhidden = dhidden; a.dweight = dweight;
  if (!ce_good(a) || kept == nullptr || up == nullptr || ws == nullptr || ((reinterpret_cast<uintptr_t>(ws) | reinterpret_cast<uintptr_t>(kept)) & 255) != 0)
    return BONSAI_CUDA_BAD_ARG;
  const CePlan p = ce_plan(a, true);
  if (kept_bytes < p.kept || ws_bytes < p.bytes) return BONSAI_CUDA_BAD_ARG;
  return type == CE_F32 ? ce_backward<float>(a, p, st) : type == CE_F16 ? ce_backward<__half>(a, p, st) : ce_backward<__nv_bfloat16>(a, p, st);
}

}  // extern "C"
