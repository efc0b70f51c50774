// The prefill kernel over the nodes of a tree of drafted tokens (tree.h): a row block is 256 rows of L nodes
// times the query heads of a KV head, every one of which sees the whole prefix.

#include "prefill_kernel.h"

namespace kvq {

template <typename T, int BITS, bool PAGED, int G, int D>
static hipError_t launch_tree_t(const PreParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((prefill_attn_kernel<T, BITS, PAGED, G, D, 0, true>), dim3(prefill_grid(p)), dim3(kPW * 64), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.nsplit == 1 || p.fused) return e;
  constexpr bool f32 = kF32Partials<BITS, D, 0>;
  hipLaunchKernelGGL((prefill_combine_kernel<T, D, f32, false, true>), dim3(p.nunits * kPW * (D / (f32 ? 8 : 16))),
                     dim3(kPW * 64), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_prefill_tree(const PreParams& p, int dtype, int D, int bits, int G, bool paged, hipStream_t stream) {
  auto go = [&](auto t) -> hipError_t {
    using TT = decltype(t);
    if (bits == 16) {
      if (paged) return hipErrorInvalidValue;
      return D == 64 ? launch_tree_t<TT, 16, false, 64, 64>(p, stream) : launch_tree_t<TT, 16, false, 64, 128>(p, stream);
    }
    auto by_p = [&](auto b, auto g, auto d) -> hipError_t {
      constexpr int BB = decltype(b)::value, GG = decltype(g)::value, DD = decltype(d)::value;
      return paged ? launch_tree_t<TT, BB, true, GG, DD>(p, stream) : launch_tree_t<TT, BB, false, GG, DD>(p, stream);
    };
    auto by_g = [&](auto b) -> hipError_t {
      using I32 = std::integral_constant<int, 32>;
      using I64 = std::integral_constant<int, 64>;
      using I128 = std::integral_constant<int, 128>;
      if (D == 96) return by_p(b, I32{}, std::integral_constant<int, 96>{});
      if (D == 64) return G == 32 ? by_p(b, I32{}, I64{}) : by_p(b, I64{}, I64{});
      return G == 32 ? by_p(b, I32{}, I128{}) : G == 64 ? by_p(b, I64{}, I128{}) : by_p(b, I128{}, I128{});
    };
    return bits == 8 ? by_g(std::integral_constant<int, 8>{}) : by_g(std::integral_constant<int, 4>{});
  };
  return dtype == KVQ_DTYPE_BF16 ? go(BF16{}) : go(F16{});
}

}  // namespace kvq
