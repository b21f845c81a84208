// What the kernels of a head's loss share: linear_ce.cu (tensor cores) and linear_ce_rows.cu (few rows, on the CUDA cores).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace bonsai {

enum CeType { CE_F32 = 0, CE_F16 = 1, CE_BF16 = 2 };
enum CeReduce { CE_MEAN = 0, CE_SUM = 1, CE_NONE = 2 };

struct CeRows {         // the live rows, in order: filled by ce_rows_kernel
  int* count;           // [2]: how many; blocks of ce_merge_kernel that are done
  int* index;           // [N] row of the hidden states
  int* target;          // [N] its target, -1 outside the vocabulary
  int* place;           // [N] the other way: place of a row in this list, -1 for ignored ones
  float* lse2;          // [N] log2 of the sum of exponentials
};

struct CeUp {           // the upstream gradient u: one value, or one for each row ("none")
  const float* up;
  const float* top;     // "none": max |u| of the finite ones
  int reduce;
  float dz_scale;       // what dz is stored with
};
__device__ __forceinline__ float ce_up_top(const CeUp& u) { return u.reduce == CE_NONE ? *u.top : fabsf(*u.up); }
// u_i over the largest finite |u|; where none is above 0, u_i itself: 0 or not finite
__device__ __forceinline__ float ce_up_factor(const CeUp& u, const CeRows& r, int row) {
  const float top = ce_up_top(u), x = u.up[u.reduce == CE_NONE ? r.index[row] : 0];
  return r.target[row] < 0 ? NAN : top > 0.0f ? x / top : x;
}
// what the products' sums are multiplied by
__device__ __forceinline__ float ce_up_scale(const CeUp& u, int n) { return n > 0 ? ce_up_top(u) / u.dz_scale / (u.reduce == CE_MEAN ? (float)n : 1.0f) : 0.0f; }

__device__ __forceinline__ float ce_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr float kCeLog2e = 1.4426950408889634f;

// The f32 head and the live rows of the few-rows kernels.
struct CeFewArgs {
  CeRows rows;
  const void* weight;
  const void* x;             // [tokens of a launch][ldx] f32, zeros behind the last live row
  long long ldw, ldx;
  int vocab, width, tokens;  // tokens: the most there can be
  int first, tokens_left;    // a launch's first token, and how many there can be from it on (set here)
  float smoothing;
  CeUp up;
  // the loss
  float *part_m, *part_s, *part_z, *at_target;
  long long ldn;
  // the gradients
  float* dz;                 // [tokens][ldz] f32
  long long ldz;
  float* part;               // [slots][tokens][width]
  void *dhidden, *dweight;
  int row_count;             // rows of dhidden
};

constexpr int kCeFew32 = 24;          // rows up to which these kernels run
int ce_few_slots(int width);          // parts of dh
int ce_few_loss_slots();              // parts of the loss
cudaError_t ce_few_loss(const CeFewArgs& a, cudaStream_t st);
cudaError_t ce_few_gradients(const CeFewArgs& a, cudaStream_t st);

}  // namespace bonsai
