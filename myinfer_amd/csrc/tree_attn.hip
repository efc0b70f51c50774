// Host side of tree_attn_kernel (tree_kernel.h): plan, workspace, launch.

#include <algorithm>

#include "tree_kernel.h"

namespace kvq {

struct TreePlan {
  int rowblocks, nunits, nsplit, fused;
};

// Splits for about two workgroups a CU (one where the ring of an unquantized head_dim-128 cache fills a CU's LDS), each of
// at least two tiles a wave.
static TreePlan tree_plan(int B, int Hq, int Hkv, int L, int D, int S, int window, int bits) {
  TreePlan pl;
  const int nrows = (Hq / Hkv) * L;
  pl.rowblocks = (nrows + 31) / 32;
  pl.nunits = B * Hkv * pl.rowblocks;
  const int span = window > 0 ? std::min(S, window + L - 1 + kTile - 1) : S;
  const int tiles = (span + kTile - 1) / kTile;
  const int target = bits == 16 && D == 128 ? 256 : 512;
  const int most = std::max(1, tiles / (2 * kTW));
  pl.nsplit = std::max(1, std::min({target / pl.nunits, most, kMaxSplit}));
  pl.fused = pl.nsplit <= kFewSplits && pl.nunits <= kMaxCountedUnits;
  return pl;
}

// Workspace: [the split counters every launch reserves][(m, l) per row and split][o per row and split]
struct TreeLayout {
  size_t ml, o, total;
};
static TreeLayout tree_layout(const TreePlan& pl, int D) {
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t rows = pl.nsplit > 1 ? (size_t)pl.nunits * pl.nsplit * 32 : 0;
  TreeLayout l;
  l.ml = kCounterBytes;
  l.o = l.ml + up(rows * sizeof(float2));
  l.total = l.o + up(rows * D * sizeof(float));
  return l;
}

size_t tree_rows_bytes(int B, int Hq, int Hkv, int L, int D, int S, int window) {
  size_t n = 0;
  for (int bits : {8, 16}) n = std::max(n, tree_layout(tree_plan(B, Hq, Hkv, L, D, S, window, bits), D).total);
  return n;
}

template <typename T, int D, int BITS, int G, bool PAGED>
static hipError_t launch_t(const DecParams& p, int B, hipStream_t stream) {
  hipLaunchKernelGGL((tree_attn_kernel<T, D, BITS, G, PAGED>), dim3(p.nunits * p.nsplit), dim3(kTW * 64), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.nsplit == 1 || p.fused) return e;
  return launch_combine<T, D>(merge_params(p, 32), B, stream);
}

hipError_t launch_tree_rows(DecParams p, int B, int dtype, int D, int bits, int G, bool paged, void* workspace, hipStream_t stream) {
  const TreePlan pl = tree_plan(B, p.Hq, p.Hkv, p.L, D, p.S, p.window, bits);
  const TreeLayout lay = tree_layout(pl, D);
  p.counters = (unsigned*)workspace;
  p.part_ml = (float*)((char*)workspace + lay.ml);
  p.part_o = (float*)((char*)workspace + lay.o);
  p.rowblocks = pl.rowblocks;
  p.nunits = pl.nunits;
  p.nsplit = pl.nsplit;
  p.fused = pl.fused;
  p.xcd_remap = ((int64_t)pl.nunits * pl.nsplit) % kXcds == 0;
  p.d_nsplit = make_div31((uint32_t)pl.nsplit);
  p.d_rowblocks = make_div31((uint32_t)pl.rowblocks);
  auto go = [&](auto t) -> hipError_t {
    using T = decltype(t);
    if (bits == 16) {
      if (paged) return hipErrorInvalidValue;
      return D == 128 ? launch_t<T, 128, 16, 64, false>(p, B, stream) : launch_t<T, 64, 16, 64, false>(p, B, stream);
    }
    auto by_p = [&](auto d, auto b, auto g) -> hipError_t {
      constexpr int DD = decltype(d)::value, BB = decltype(b)::value, GG = decltype(g)::value;
      return paged ? launch_t<T, DD, BB, GG, true>(p, B, stream) : launch_t<T, DD, BB, GG, false>(p, B, stream);
    };
    auto by_b = [&](auto d, auto g) -> hipError_t { return bits == 8 ? by_p(d, IC<8>{}, g) : by_p(d, IC<4>{}, g); };
    if (D == 64) return G == 32 ? by_b(IC<64>{}, IC<32>{}) : by_b(IC<64>{}, IC<64>{});
    return G == 32 ? by_b(IC<128>{}, IC<32>{}) : G == 64 ? by_b(IC<128>{}, IC<64>{}) : by_b(IC<128>{}, IC<128>{});
  };
  return dtype == KVQ_DTYPE_BF16 ? go(BF16{}) : go(F16{});
}

}  // namespace kvq
