#include "low_rank_launch.cuh"

namespace bonsai {
template <> cudaError_t lr_rows<__nv_bfloat16>(const LrRowsArgs& a, bool back, cudaStream_t st) { return lr_rows_of<__nv_bfloat16>(a, back, st); }
template <> cudaError_t lr_outer<__nv_bfloat16>(const LrOuterArgs& a, cudaStream_t st) { return lr_outer_of<__nv_bfloat16>(a, st); }
}  // namespace bonsai
