// A tree of drafted tokens, as the attention kernels read it.
//
// The tree's L nodes are the last L rows of a sequence, and the call's query rows. Node l sees every key
// before the tree and, of the tree, itself and its ancestors: bit j % 32 of word j / 32 of its row of
// `bits` says whether node j is one of them. A node sits at position (keys before the tree) + depth; an
// absent node (padding in a batch of unequal trees) has depth -1 and no bit set, and no node has its bit.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.h"

namespace kvq {

struct TreeParams {
  const uint32_t* bits;   // [B][L][words]
  const int32_t* depths;  // [B][L]
  int64_t bits_sb, depths_sb;
  int words;  // ceil(L / 32)
};

inline TreeParams tree_params(const kvq_tree* t, int L) {
  return {t->bits, t->depths, t->bits_stride_b, t->depths_stride_b, (L + 31) / 32};
}

// One node's row of the tree, held in vector registers (the prefill kernel's tile loop has no scalar ones
// to spare). `first` is the row of the cache that holds node 0.
struct TreeRow {
  const uint32_t* bits;
  int words, first, depth;
  __device__ __forceinline__ void load(const TreeParams& t, int b, int l, int first_row) {
    bits = t.bits + (int64_t)b * t.bits_sb + (int64_t)l * t.words;
    depth = t.depths[(int64_t)b * t.depths_sb + l];
    words = t.words;
    first = first_row;
    asm volatile("" : "+v"(words), "+v"(first));
  }
  // Which of the keys [k, k + 32) the node sees: all before the tree, none past its last node.
  __device__ __forceinline__ uint32_t keys(int k) const {
    const int j0 = k - first;
    if (j0 <= -32) return ~0u;
    if (j0 < 0) return (bits[0] << -j0) | ((1u << -j0) - 1u);
    const int w = j0 >> 5, sh = j0 & 31;
    const uint32_t lo = w < words ? bits[w] : 0u, hi = w + 1 < words ? bits[w + 1] : 0u;
    return (uint32_t)((((uint64_t)hi << 32) | lo) >> sh);
  }
};

}  // namespace kvq
