// The bits and depths of a tree of drafted tokens from its parents (tree.h; kvq_draft_tree).
//
// A thread per node walks to the root through the parents in LDS, twice: once for the depth and whether an absent
// node lies on the way, once to write the node's row of bits, whose set bits the walk meets from the highest
// down. Bound by its launch: a step costs an LDS round trip, and drafted trees are a few nodes deep. One
// launch serves every layer of a step.

#include "launch.h"
#include "tree.h"

namespace kvq {

__global__ __launch_bounds__(256) void draft_tree_kernel(const int32_t* parents, int64_t parents_sb, int L, uint32_t* bits,
                                                         int32_t* depths, const int32_t* starts, int64_t start,
                                                         int32_t* positions) {
  __shared__ int16_t par[KVQ_TREE_MAX_NODES];  // -1 a root, -2 an absent node
  const int b = blockIdx.y;
  const int32_t* pr = parents + (int64_t)b * parents_sb;
  for (int i = threadIdx.x; i < L; i += blockDim.x) {
    const int x = pr[i];
    par[i] = (int16_t)(x >= -1 && x < i ? x : -2);  // a parent comes before its children
  }
  __syncthreads();
  const int l = blockIdx.x * blockDim.x + threadIdx.x;
  if (l >= L) return;
  const int words = (L + 31) / 32;
  uint32_t* row = bits + ((int64_t)b * L + l) * words;
  int depth = -1, j = l;
  bool here;
  if (L <= 64) {  // one walk: the row fits a register
    uint64_t seen = 0;
    while (j >= 0) {
      ++depth;
      seen |= 1ull << j;
      j = par[j];
    }
    here = j == -1;
    if (!here) seen = 0;
    row[0] = (uint32_t)seen;
    if (words == 2) row[1] = (uint32_t)(seen >> 32);
  } else {
    while (j >= 0) {
      ++depth;
      j = par[j];
    }
    here = j == -1;
    j = here ? l : -1;
    for (int w = words - 1; w >= 0; --w) {
      uint32_t x = 0;
      while (j >= 32 * w) {
        x |= 1u << (j & 31);
        j = par[j];
      }
      row[w] = x;
    }
  }
  depths[(int64_t)b * L + l] = here ? depth : -1;
  if (positions) positions[(int64_t)b * L + l] = (int32_t)((starts ? starts[b] : start) + (here ? depth : 0));
}

hipError_t launch_draft_tree(const int32_t* parents, int64_t parents_sb, int B, int L, uint32_t* bits, int32_t* depths,
                             const int32_t* starts, int64_t start, int32_t* positions, hipStream_t stream) {
  hipLaunchKernelGGL(draft_tree_kernel, dim3((L + 255) / 256, B), dim3(256), 0, stream, parents, parents_sb, L, bits, depths,
                     starts, start, positions);
  return hipGetLastError();
}

}  // namespace kvq
