// Host side of tree_attn_kernel (tree_kernel.h): plan, workspace, launch.

#include <algorithm>

#include "tree_kernel.h"

namespace kvq {

struct TreePlan {
  int rowblocks, nunits, nsplit, fused;
  float us;  // its time by the model
};

// The number of splits of least time by a rough model of a launch, in us: a wave's 32-key tile takes 2.1 with two workgroups
// on its CU and 1.3 with one (half of it at 64 dims; the ring of an unquantized head_dim-128 cache leaves room for one), a
// workgroup's start and its waves' merge 5, the splits' merge 1.5 by the last to finish, else a launch, its bytes and
// the splits past the 32 that it loads at once. A wave gets at least two tiles.
static TreePlan tree_plan(int B, int Hq, int Hkv, int L, int D, int S, int window, int bits) {
  TreePlan pl;
  const int nrows = (Hq / Hkv) * L;
  pl.rowblocks = (nrows + 31) / 32;
  pl.nunits = B * Hkv * pl.rowblocks;
  const int span = window > 0 ? std::min(S, window + L - 1 + kTile - 1) : S;
  const int tiles = (span + kTile - 1) / kTile;
  const int per_cu = bits == 16 && D == 128 ? 1 : 2;
  const int most = std::max(1, std::min(tiles / (2 * kTW), kMaxSplit));
  pl.nsplit = 0;
  for (int ns = 1; ns <= most; ns += ns < 16 ? 1 : ns / 8) {
    const int64_t wgs = (int64_t)pl.nunits * ns, rounds = wgs / (256 * per_cu), rest = wgs % (256 * per_cu);
    const float per = ((tiles + ns - 1) / ns + kTW - 1) / kTW * (D == 64 ? 0.5f : 1.0f);
    const float one = per * 1.3f + 5.0f, two = per * (per_cu == 2 ? 2.1f : 1.3f) + 5.0f;
    const bool fused = ns <= kFewSplits && pl.nunits <= kMaxCountedUnits;
    const float merge = ns == 1 ? 0.0f : fused ? 1.5f : 3.5f + (float)wgs * (32 * D * 4) / 3e6f + (ns > 32 ? 0.06f * (ns - 32) : 0.0f);
    const float t = rounds * two + (rest > 256 ? two : rest > 0 ? one : 0.0f) + merge;
    if (pl.nsplit == 0 || t < pl.us) pl.nsplit = ns, pl.us = t;
  }
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

// (the model's time against 260 measured calls: 5.3 + 0.82 of it, within 16%)
float tree_rows_time(int B, int Hq, int Hkv, int L, int D, int S, int window, int bits) {
  return 5.3f + 0.82f * tree_plan(B, Hq, Hkv, L, D, S, window, bits).us;
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
  return launch_combine<T, D, 32>(merge_params(p, 32), B, stream);
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
