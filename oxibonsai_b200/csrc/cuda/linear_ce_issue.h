// The order of waits, products and commits of the thread that issues a tile's products in linear_ce.cu, apart from the instructions themselves, so
// that the host can run it too.
#pragma once

#ifdef __CUDACC__
#define CE_ISSUE_FN __host__ __device__ __forceinline__
#else
#define CE_ISSUE_FN inline
#endif

namespace bonsai {

// Blocks b0 .. b1 - 1 of k, kSegment of them to an accumulator (all of them where it is 0), `terms` products for each; `segment` counts the
// accumulators handed out so far.  Ops: bool wait_acc(buffer, phase), bool wait_full(), void product(buffer, first), void commit_acc(buffer).
// False behind a wait that has expired: the accumulator at hand lacks blocks of k, or holds an older tile, and is not committed, so that the
// epilogues' waits for it expire as well and store NaN.
template <int kBufs, int kSegment, typename Ops>
CE_ISSUE_FN bool ce_issue(Ops& ops, int b0, int b1, int terms, int* segment) {
  for (int k0 = b0; k0 < b1; ++*segment) {
    const int ab = *segment % kBufs, k1 = kSegment != 0 && k0 + kSegment < b1 ? k0 + kSegment : b1;
    if (!ops.wait_acc(ab, ((*segment / kBufs) & 1) ^ 1)) return false;
    for (int i = 0; i < (k1 - k0) * terms; ++i) {
      if (!ops.wait_full()) return false;
      ops.product(ab, i == 0);
    }
    ops.commit_acc(ab);
    k0 = k1;
  }
  return true;
}

}  // namespace bonsai
