// A tree of drafted tokens around the model's step: each node's mask before it,
// the accepted path after it. A sequence's nodes are rows start .. start + n of
// flat arrays, a parent before its children (-1: none). A few bytes a node: the
// time is the launch and the chain of dependent looks, one per generation, so
// the nodes are staged in shared memory once (3 to 4 us each, captured, for 8 to
// 2000 nodes).
#include "sm100.cuh"

namespace ib200 {
namespace tree {

constexpr int MAX_NODES = 256;
constexpr int THREADS = 256;

struct Rows {
  int start, n;  // rows of the sequence that exist
};
// Nodes of sequence s, at most `most` and as far as there are rows; the first
// thread reports what does not fit.
__device__ __forceinline__ Rows rows_of(const int* q_start, const int* q_len, int s, int T, int most, int* status) {
  const int start = q_start[s], n = max(q_len[s], 0);
  const int fit = start < 0 || start > T ? 0 : min(min(n, most), T - start);
  if (fit < n && threadIdx.x == 0) record_status_detail(status, kStatusBadIndex, 9, s, start < 0 || start > T ? start : n);
  return {start, fit};
}

// mask[row, w]: bit j of word w is node 32 w + j of the row's sequence, set for
// the row itself and its ancestors.
__global__ void __launch_bounds__(THREADS)
    mask_kernel(const int* parents, const int* q_start, const int* q_len, int T, int words, int* mask, int* status) {
  pdl_trigger();
  pdl_wait();
  __shared__ int up[MAX_NODES];
  const Rows r = rows_of(q_start, q_len, blockIdx.x, T, 32 * words, status);
  for (int i = threadIdx.x; i < r.n; i += THREADS) {
    int u = parents[r.start + i];
    if (u < -1 || u >= i) {  // not a node before this one
      record_status_detail(status, kStatusBadIndex, 10, r.start + i, u);
      u = -1;
    }
    up[i] = u;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < r.n * words; i += THREADS) {
    const int node = i / words, w = i - node * words;
    uint32_t bits = 0;
    for (int a = node; a >= 32 * w; a = up[a])  // ancestors have lower numbers
      if (a < 32 * w + 32) bits |= 1u << (a & 31);
    mask[(r.start + static_cast<size_t>(node)) * words + w] = static_cast<int>(bits);
  }
}

// The walk from node 0: on to the first child whose token is what the model
// chose at its parent. One warp per sequence.
__global__ void __launch_bounds__(32)
    accept_kernel(const int* tokens, const int* target, const int* parents, const int* q_start, const int* q_len,
                  int T, int most, int* path, int* count, int* after, int* status) {
  pdl_trigger();
  pdl_wait();
  __shared__ int up[MAX_NODES], tok[MAX_NODES], chosen[MAX_NODES];
  const int s = blockIdx.x, lane = threadIdx.x;
  const Rows r = rows_of(q_start, q_len, s, T, MAX_NODES, status);
  for (int i = lane; i < r.n; i += 32) {
    up[i] = parents[r.start + i];
    tok[i] = tokens[r.start + i];
    chosen[i] = target[r.start + i];
  }
  __syncwarp();
  int n = 0, node = r.n > 0 ? 0 : -1, last = -1;
  int* out = path + static_cast<size_t>(s) * most;
  while (node >= 0 && n < most) {
    if (lane == 0) out[n] = node;
    ++n;
    last = node;
    node = -1;
    const int want = chosen[last];
    for (int i0 = last + 1; i0 < r.n && node < 0; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t on = __ballot_sync(0xffffffffu, i < r.n && up[i] == last && tok[i] == want);
      if (on != 0) node = i0 + __ffs(on) - 1;
    }
  }
  for (int i = n + lane; i < most; i += 32) out[i] = -1;
  if (lane == 0) {
    count[s] = n;
    after[s] = last >= 0 ? chosen[last] : -1;
  }
}

}  // namespace tree
}  // namespace ib200

using namespace ib200;

// parents [T]; q_start / q_len [n]; mask int32 [T, words], words 1 to 8.
extern "C" int ib_tree_mask(const int* parents, const int* q_start, const int* q_len, int n, int T, int words, int* mask,
                            int* status, cudaStream_t stream) {
  if (n <= 0 || T <= 0) return 0;
  if (words < 1 || words > tree::MAX_NODES / 32) return -1;
  return static_cast<int>(launch_pdl(tree::mask_kernel, dim3(n), tree::THREADS, 0, stream, parents, q_start, q_len, T,
                                     words, mask, status));
}

// tokens / target / parents [T]; path [n, most], count / after [n].
extern "C" int ib_tree_accept(const int* tokens, const int* target, const int* parents, const int* q_start,
                              const int* q_len, int n, int T, int most, int* path, int* count, int* after, int* status,
                              cudaStream_t stream) {
  if (n <= 0) return 0;
  if (most < 1 || T < 0) return -1;
  return static_cast<int>(launch_pdl(tree::accept_kernel, dim3(n), dim3(32), 0, stream, tokens, target, parents, q_start,
                                     q_len, T, most, path, count, after, status));
}
