// The decode kernel over the nodes of a tree of drafted tokens (tree.h): the rows of a KV head are its
// L nodes times its query heads. Quantized caches take the MULTI form whatever the rows are (its rounding of the
// value products is the smaller one); unquantized ones the plain form.

#include "decode_kernel.h"

namespace kvq {

template <typename T, int D, int BITS, int G, bool PAGED, bool NARROW>
static hipError_t launch_tree_t(const DecParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((decode_attn_kernel<T, D, BITS, 4, 2, PAGED, G, false, NARROW, BITS != 16, true>),
                     dim3(p.nunits * p.nsplit), dim3(256), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.nsplit == 1 || p.fused) return e;
  return launch_combine<T, D>(merge_params(p, DecCfg<D, BITS, G>::R), p.nunits / (p.Hkv * p.rowblocks), stream, p.dv);
}

template <typename T, int D, int BITS, int G, bool PAGED>
static hipError_t launch_tree_dims(const DecParams& p, hipStream_t stream) {
  if (p.dv == D) return launch_tree_t<T, D, BITS, G, PAGED, false>(p, stream);
  if constexpr (narrow_rows<D, BITS, G>()) return launch_tree_t<T, D, BITS, G, PAGED, true>(p, stream);
  return hipErrorInvalidValue;
}

hipError_t launch_decode_tree(const DecParams& p, int dtype, int D, int bits, int G, bool paged, hipStream_t stream) {
  if (bits == 16) {
    if (paged || D == 256) return hipErrorInvalidValue;
    auto go = [&](auto t) -> hipError_t {
      using T = decltype(t);
      return D == 128 ? launch_tree_dims<T, 128, 16, 64, false>(p, stream) : launch_tree_dims<T, 64, 16, 64, false>(p, stream);
    };
    return dtype == KVQ_DTYPE_BF16 ? go(BF16{}) : go(F16{});
  }
  return dispatch_quant(dtype, D, bits, G, [&](auto t, auto d, auto b, auto g) -> hipError_t {
    using T = decltype(t);
    constexpr int DD = decltype(d)::value, BB = decltype(b)::value, GG = decltype(g)::value;
    return paged ? launch_tree_dims<T, DD, BB, GG, true>(p, stream) : launch_tree_dims<T, DD, BB, GG, false>(p, stream);
  });
}

}  // namespace kvq
