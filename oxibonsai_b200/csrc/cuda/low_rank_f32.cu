#include "low_rank_launch.cuh"

namespace bonsai {
template <> cudaError_t lr_rows<float>(const LrRowsArgs& a, bool back, cudaStream_t st) { return lr_rows_of<float>(a, back, st); }
template <> cudaError_t lr_outer<float>(const LrOuterArgs& a, cudaStream_t st) { return lr_outer_of<float>(a, st); }
}  // namespace bonsai
