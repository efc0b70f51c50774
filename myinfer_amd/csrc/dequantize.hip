// Reading a quantized cache back: x = scale * code + bias of every cached row, in the cache's type
// (kvq_dequantize, kvq_paged_dequantize). The counterpart of mx.dequantize.
//
// code * scale is exact in fp32 and the bias is added in one FMA, so the value is rounded once to fp32 and
// once to T. Bound by its bytes: D codes, their scales and biases read and 2 D bytes written per row. A thread takes
// 8 elements at a time (8, 4 or 2 bytes of codes, one 16-byte store), a workgroup rows of one head, so that only a row's
// number within them is computed by the threads.
//
// The values leave by streaming stores: nobody reads them before the call ends, and they would turn the cached rows out
// of the L2 caches. 32768 rows of 8 heads of 128 dims in 8 bits, K and V (205 MB): 31 us, 6.6 TB/s, where a copy
// reaches 5.2 (ordinary stores 44, and each chunk finding its sequence and head by itself 45); pages of 8 sequences up to
// 8192 rows (308 MB) 55 us (75, 105), of 4 up to 1999 rows in 4 bits (31 MB) 9.1 (10.7, 12.1).

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
  int L, H, BH, per_row;  // rows of the launch; heads, and of all sequences; 8-element chunks of a row
  int rows, tiles;        // rows of a workgroup, workgroups of a head
  Div31 div_c, div_tiles, div_bh, div_h;
  int64_t l0, row0;  // first row of the launch, and of the cache
  const int32_t* lens;  // rows of each sequence (paged), or null
};

// A workgroup takes some rows of a head: N chunks a thread, 256 apart, their loads issued together
template <typename T, int BITS, int G, int N>
__global__ __launch_bounds__(256) void dequantize_kernel(ReadJob job0, ReadJob job1, ReadMap m, PageMap pm) {
  const int t0 = (int)div31(blockIdx.x, m.div_tiles), tile = (int)blockIdx.x - t0 * m.tiles;
  const int jb = (int)div31((uint32_t)t0, m.div_bh), bh = t0 - jb * m.BH;
  const int bb = (int)div31((uint32_t)bh, m.div_h), h = bh - bb * m.H;
  const ReadJob job = jb == 0 ? job0 : job1;
  const int64_t l = m.l0 + (int64_t)tile * m.rows, r0 = m.row0 + l;  // first rows, of the destination and the cache
  int nv = min(m.rows, m.L - tile * m.rows);
  if (m.lens) nv = (int)min((int64_t)nv, (int64_t)load_uniform_i32(m.lens, bb) - r0);  // rows behind the sequence stay
  const uint8_t* codes = job.codes + h * job.c_h;
  const uint16_t* scales = job.scales + h * job.g_h;
  const uint16_t* biases = job.biases + h * job.g_h;
  uint16_t* const out = job.dst + bb * job.d_b + h * job.d_h + l * job.d_l;
  Bytes<BITS> c[N];  // 8 codes are BITS bytes
  uint16_t s[N], b[N];
  int row[N], chunk[N], page[N];
  const int items = nv * m.per_row;  // (negative: none)
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int i = n * 256 + (int)threadIdx.x;
    row[n] = i < items ? (int)div31((uint32_t)i, m.div_c) : 0;
    chunk[n] = i - row[n] * m.per_row;
    page[n] = bb;
    if (m.lens && i < items) page[n] = pm.table[(int64_t)bb * pm.table_stride + ((r0 + row[n]) >> 6)];
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (n * 256 + (int)threadIdx.x >= items) continue;
    int64_t r = r0 + row[n];
    if (m.lens) {
      page[n] = min(max(page[n], 0), pm.num_pages - 1);
      r &= 63;
    }
    c[n].load(codes + page[n] * job.c_b + r * job.c_s + chunk[n] * BITS);
    const int64_t g = page[n] * job.g_b + r * job.g_s + 8 * chunk[n] / G;
    s[n] = scales[g];
    b[n] = biases[g];
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (n * 256 + (int)threadIdx.x >= items) continue;
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
    __builtin_nontemporal_store(w, (u4*)(out + row[n] * job.d_l + 8 * chunk[n]));
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
  ReadMap m{};
  m.H = H;
  m.BH = B * H;
  m.per_row = D / 8;
  m.div_c = make_div31((uint32_t)m.per_row);
  m.div_h = make_div31((uint32_t)H);
  m.div_bh = make_div31((uint32_t)m.BH);
  m.row0 = row0;
  m.lens = lens;
  // four chunks a thread where that still gives 4 workgroups a CU
  const int64_t heads = (int64_t)m.BH * njobs;
  const int n = heads * ((L + 1024 / m.per_row - 1) / (1024 / m.per_row)) >= 4 * 256 ? 4 : 1;
  m.rows = 256 * n / m.per_row;
  const int64_t max_l = (((int64_t)1 << 30) / heads) * m.rows;  // (workgroups of a launch: more rows take more launches)
  if (max_l <= 0) return hipErrorInvalidValue;
  for (int64_t l0 = 0; l0 < L; l0 += max_l) {
    m.l0 = l0;
    m.L = (int)(L - l0 < max_l ? L - l0 : max_l);
    m.tiles = (m.L + m.rows - 1) / m.rows;
    m.div_tiles = make_div31((uint32_t)m.tiles);
    const dim3 grid((unsigned)(heads * m.tiles)), block(256);
    if (n == 4)
      hipLaunchKernelGGL((dequantize_kernel<T, BITS, G, 4>), grid, block, 0, stream, k, v, m, pm);
    else
      hipLaunchKernelGGL((dequantize_kernel<T, BITS, G, 1>), grid, block, 0, stream, k, v, m, pm);
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
