// Reading a quantized cache back: x = scale * code + bias of every cached row, in the cache's type
// (kvq_dequantize, kvq_paged_dequantize). The counterpart of mx.dequantize.
//
// code * scale is exact in fp32 and the bias is added in one FMA, so the value is rounded once to fp32 and
// once to T. Bound by its bytes: D codes, their scales and biases read and 2 D bytes written per row. A thread takes
// 8 elements at a time (8, 4 or 2 bytes of codes, one 16-byte store).

#include "quantize_core.h"

namespace kvq {

struct ReadJob {
  const uint8_t* codes;
  const uint16_t* scales;
  const uint16_t* biases;
  int64_t c_b, c_h, c_s;  // bytes
  int64_t g_b, g_h, g_s;  // elements
  uint16_t* dst;
  int64_t d_b, d_h, d_l;
};

struct ReadMap {
  uint32_t total;  // 8-element chunks of a job
  int L, H, per_row;
  Div31 div_c, div_l, div_h;
  int64_t l0, row0;  // first row of the launch, and of the cache
  const int32_t* lens;  // rows of each sequence (paged), or null
};

// N chunks a thread, 256 apart, their loads issued together
template <typename T, int BITS, int G, int N>
__global__ __launch_bounds__(256) void dequantize_kernel(ReadJob job0, ReadJob job1, ReadMap m, PageMap pm) {
  const ReadJob job = blockIdx.y == 0 ? job0 : job1;
  Bytes<BITS> c[N];  // 8 codes are BITS bytes
  uint16_t s[N], b[N];
  uint16_t* dst[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const uint32_t t = (blockIdx.x * N + n) * 256u + threadIdx.x;
    dst[n] = nullptr;
    if (t >= m.total) continue;
    const uint32_t row = div31(t, m.div_c);
    const int chunk = (int)(t - row * (uint32_t)m.per_row);
    const uint32_t bh = div31(row, m.div_l);
    const int64_t l = m.l0 + (int64_t)(row - bh * (uint32_t)m.L);
    const uint32_t bb = div31(bh, m.div_h);
    const int64_t h = bh - bb * (uint32_t)m.H;
    int64_t page = bb, r = m.row0 + l;
    if (m.lens) {
      if (r >= m.lens[bb]) continue;  // rows behind the sequence are left as they are
      page = min(max(pm.table[(int64_t)bb * pm.table_stride + (r >> 6)], 0), pm.num_pages - 1);
      r &= 63;
    }
    c[n].load(job.codes + page * job.c_b + h * job.c_h + r * job.c_s + chunk * BITS);
    const int64_t g = page * job.g_b + h * job.g_h + r * job.g_s + 8 * chunk / G;
    s[n] = job.scales[g];
    b[n] = job.biases[g];
    dst[n] = job.dst + (int64_t)bb * job.d_b + h * job.d_h + l * job.d_l + 8 * chunk;
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (!dst[n]) continue;
    const float sf = to_float(s[n], T{}), bf = to_float(b[n], T{});
    u4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int bit = BITS * (2 * e + k);
        const uint32_t code = (c[n].w[bit / 32] >> (bit % 32)) & ((1u << BITS) - 1u);
        x[k] = __builtin_fmaf((float)code, sf, bf);
      }
      w[e] = (uint32_t)from_float(x[0], T{}) | ((uint32_t)from_float(x[1], T{}) << 16);
    }
    *(u4*)dst[n] = w;
  }
}

static ReadJob make_read(const kvq_qtensor* q, const kvq_rows* x) {
  ReadJob j{};
  j.codes = (const uint8_t*)q->codes;
  j.scales = (const uint16_t*)q->scales;
  j.biases = (const uint16_t*)q->biases;
  j.c_b = q->codes_stride_b * 4;
  j.c_h = q->codes_stride_h * 4;
  j.c_s = q->codes_stride_s * 4;
  j.g_b = q->sb_stride_b;
  j.g_h = q->sb_stride_h;
  j.g_s = q->sb_stride_s;
  j.dst = (uint16_t*)x->data;
  j.d_b = x->stride_b;
  j.d_h = x->stride_h;
  j.d_l = x->stride_l;
  return j;
}

template <typename T, int BITS, int G>
static hipError_t launch_read(const ReadJob& k, const ReadJob& v, int njobs, int B, int H, int64_t L, int D, int64_t row0,
                              const int32_t* lens, const PageMap& pm, hipStream_t stream) {
  // (the chunk index of a launch stays below 2^31: more rows take more launches)
  const int64_t per_l = (int64_t)B * H * (D / 8);
  if (per_l >= ((int64_t)1 << 31)) return hipErrorInvalidValue;
  const int64_t max_l = (((int64_t)1 << 31) - 1) / per_l;
  for (int64_t l0 = 0; l0 < L; l0 += max_l) {
    const int64_t n = L - l0 < max_l ? L - l0 : max_l;
    ReadMap m{};
    m.total = (uint32_t)(per_l * n);
    m.L = (int)n;
    m.H = H;
    m.per_row = D / 8;
    m.div_c = make_div31((uint32_t)m.per_row);
    m.div_l = make_div31((uint32_t)n);
    m.div_h = make_div31((uint32_t)H);
    m.l0 = l0;
    m.row0 = row0;
    m.lens = lens;
    // four chunks a thread where that still gives 4 workgroups a CU
    const unsigned blocks = (m.total + 255u) / 256u;
    if ((int64_t)blocks * njobs >= 4 * 1024)
      hipLaunchKernelGGL((dequantize_kernel<T, BITS, G, 4>), dim3((blocks + 3) / 4, njobs), dim3(256), 0, stream, k, v, m, pm);
    else
      hipLaunchKernelGGL((dequantize_kernel<T, BITS, G, 1>), dim3(blocks, njobs), dim3(256), 0, stream, k, v, m, pm);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_dequantize(const kvq_qtensor* k_src, const kvq_rows* k_dst, const kvq_qtensor* v_src, const kvq_rows* v_dst,
                             int num_pages, const int32_t* table, int64_t table_stride, const int32_t* lens, int64_t row0,
                             int B, int H, int64_t L, int D, int bits, int G, int dtype, hipStream_t stream) {
  const ReadJob k = make_read(k_src, k_dst), v = v_src ? make_read(v_src, v_dst) : k;
  const int njobs = v_src ? 2 : 1;
  const PageMap pm{table, table_stride, nullptr, num_pages};
  auto by_g = [&](auto t, auto b) -> hipError_t {
    using T = decltype(t);
    constexpr int BB = decltype(b)::value;
    if (G == 32) return launch_read<T, BB, 32>(k, v, njobs, B, H, L, D, row0, lens, pm, stream);
    return G == 64 ? launch_read<T, BB, 64>(k, v, njobs, B, H, L, D, row0, lens, pm, stream)
                   : launch_read<T, BB, 128>(k, v, njobs, B, H, L, D, row0, lens, pm, stream);
  };
  auto by_b = [&](auto t) -> hipError_t {
    if (bits == 2) return by_g(t, std::integral_constant<int, 2>{});
    return bits == 4 ? by_g(t, std::integral_constant<int, 4>{}) : by_g(t, std::integral_constant<int, 8>{});
  };
  return dtype == KVQ_DTYPE_BF16 ? by_b(BF16{}) : by_b(F16{});
}

}  // namespace kvq
