#include "low_rank_launch.cuh"

namespace bonsai {
template <> cudaError_t lr_rows<__half>(const LrRowsArgs& a, bool back, cudaStream_t st) { return lr_rows_of<__half>(a, back, st); }
template <> cudaError_t lr_outer<__half>(const LrOuterArgs& a, cudaStream_t st) { return lr_outer_of<__half>(a, st); }
}  // namespace bonsai
