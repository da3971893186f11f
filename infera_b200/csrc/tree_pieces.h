// The pieces of a cut item of the tree attention: `count` of them, one of each
// of the runs first, first + 1, ...
#pragma once

#ifdef __CUDACC__
#define IB200_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define IB200_HOST_DEVICE inline
#endif

namespace ib200 {

// Whether all of them are pieces of `runs` runs. A CTA whose bounded wait gave
// up leaves the entries of its later items as the workspace was, and what that
// names is not read.
IB200_HOST_DEVICE bool pieces_exist(int first, int count, int runs) {
  return first >= 0 && count >= 0 && first <= runs && count <= runs - first;
}
// The piece k of an item in the partial results, two places a run: the piece
// that an item begins with in the odd one, another in the even one.
IB200_HOST_DEVICE long long piece_at(int first, int k) { return 2 * (static_cast<long long>(first) + k) + (k == 0); }

}  // namespace ib200
