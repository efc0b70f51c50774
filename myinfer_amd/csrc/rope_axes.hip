// Rotary embedding at positions given per row, over one or several axes (kvq_rope_axes), and fused with the
// quantize-append of a step's keys and values (kvq_rope_axes_append).
//
//   pair i of a row turns by  t = position[axis(i)][b][l] * scale * freq(i):
//   (x, y) -> (x cos t - y sin t, x sin t + y cos t)
//
// The angle is formed and reduced in double: position and frequency in fp32 leave an error of half an ulp of
// the angle, 2e-3 rad at position 32768, twice what rounding the result to fp16 costs. The rotation
// is in fp32, its products rounded before they are added, as in kvq_rope; the result is rounded to T.
//
// What bounds it: each row is read and written once (rotated in place, or read and stored quantized), and a pair's
// sine and cosine cost more than its rotation, so heads share them: in a thread's registers where rows are rotated in
// place, in a table in LDS where a workgroup quantizes some positions of several heads.
//
// Rotated in place (4096 tokens of 32 heads of 128 dims, 67 MB): 12.1 us with 4 heads a thread, 5.5 TB/s, the rate of a
// large copy; 13.3 with 2, 17.6 with 1, and 29.1 with the table, whose barrier each row waited for. At 1024 tokens
// 6.9 / 6.2 / 6.9 us with 4 / 2 / 1, at 16 tokens of 64 heads 5.9 / 4.7 / 5.8 (a launch takes 3.6).

#include "quantize_core.h"

namespace kvq {

constexpr int kAxesPairs = 128;    // pairs of a row at most
constexpr int kTableCells = 2048;  // (position, pair) cells of a workgroup's table: 16 KiB

struct AxesArgs {
  const int32_t* pos;
  int64_t pos_sa, pos_sb, pos_sl;
  int dims, pairs, traditional, axes;
  Div31 div_pairs;
  double freq[kAxesPairs];  // times the position scale
  alignas(8) uint8_t axis[kAxesPairs];
};

// sin and cos of an angle in radians: k pi/2 + t, |t| <= pi/4 (off by k 2^-54, nothing up to 2^31), and the
// Taylor series of t to t^9 and t^10 (remainders 1.8e-9 and 1.2e-10).
__device__ __forceinline__ float2 cos_sin(double angle) {
#pragma clang fp contract(off)
  const double k = __builtin_rint(angle * 0.63661977236758134308);
  const double td = __builtin_fma(-k, 1.57079632679489661923, angle);
  const float t = (float)td, tl = (float)(td - (double)t), z = t * t;
  float s = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(z, s, 8.3333333e-3f);
  s = __builtin_fmaf(z, s, -1.6666667e-1f);
  s = t + __builtin_fmaf(t * z, s, tl);
  float c = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = __builtin_fmaf(z, c, -1.3888889e-3f);
  c = __builtin_fmaf(z, c, 4.1666667e-2f);
  c = __builtin_fmaf(z, c, -0.5f);
  c = __builtin_fmaf(z, c, 1.0f);
  const int quadrant = (int)__builtin_fma(-4.0, __builtin_floor(k * 0.25), k);  // k mod 4
  const float a = quadrant & 1 ? c : s, b = quadrant & 1 ? s : c;
  return make_float2((quadrant + 1) & 2 ? -b : b, quadrant & 2 ? -a : a);
}

// (cos, sin) of the positions [l0, l0 + nl) of sequence b, [position][pair]
__device__ __forceinline__ void fill_table(const AxesArgs& r, int b, int l0, int nl, float2* tab) {
  for (int i = threadIdx.x; i < nl * r.pairs; i += 256) {
    const int l = (int)div31((uint32_t)i, r.div_pairs), pair = i - l * r.pairs;
    const int32_t p = r.pos[r.axis[pair] * r.pos_sa + b * r.pos_sb + (l0 + l) * r.pos_sl];
    tab[i] = cos_sin((double)p * r.freq[pair]);
  }
}

// The rows one workgroup takes: positions [l0, l0 + nl) of heads [h0, h0 + nh) of sequence b.
struct Rows {
  int b, l0, nl, h0, nh;
};
// How a launch's rows are cut: `per_pos` positions of `per_head` heads a workgroup, heads innermost.
struct RowCut {
  int per_pos, per_head, tiles, groups;  // of a sequence, of its heads
  Div31 div_groups, div_tiles;
  int blocks;  // workgroups in all
};
__device__ __forceinline__ Rows rows_of(const RowCut& c, int wg, int L, int H) {
  const int t = (int)div31((uint32_t)wg, c.div_groups), g = wg - t * c.groups;
  Rows r;
  r.b = (int)div31((uint32_t)t, c.div_tiles);
  r.l0 = (t - r.b * c.tiles) * c.per_pos;
  r.nl = min(c.per_pos, L - r.l0);
  r.h0 = g * c.per_head;
  r.nh = min(c.per_head, H - r.h0);
  return r;
}

struct RotateJob {
  uint16_t* x;
  int64_t s_b, s_h, s_l;
  int H, L, per_row, groups, heads;  // items (8 pairs each) of a row, groups of `heads` heads
  uint32_t items;                    // threads: a position's 8 pairs of a group of heads each
  Div31 div_row, div_l, div_groups;
  int blocks;
};

// Rotate rows in place. A thread takes 8 pairs of a position (split halves: dims [8j, +8) and [8j + dims/2, +8);
// interleaved: dims [16j, +16)) in NH heads, whose rows it loads first; their sines and cosines stay in its registers.
template <typename T, int NH>
__device__ __forceinline__ void rotate_rows(const RotateJob& job, const AxesArgs& r, uint32_t wg) {
#pragma clang fp contract(off)
  const uint32_t t = wg * 256 + threadIdx.x;
  if (t >= job.items) return;
  const uint32_t row = div31(t, job.div_row), j = t - row * job.per_row;
  const uint32_t bg = div31(row, job.div_l), l = row - bg * job.L;
  const uint32_t b = div31(bg, job.div_groups);
  const int h0 = (int)(bg - b * job.groups) * NH, nh = min(NH, job.H - h0);
  const int second = r.traditional ? 8 : r.dims / 2;
  uint16_t* const x = job.x + (int64_t)b * job.s_b + (int64_t)h0 * job.s_h + (int64_t)l * job.s_l + (r.traditional ? 16 : 8) * j;
  u4 lo[NH], hi[NH];
#pragma unroll
  for (int k = 0; k < NH; ++k) {
    const uint16_t* p = x + (int64_t)min(k, nh - 1) * job.s_h;
    lo[k] = *(const u4*)p;
    hi[k] = *(const u4*)(p + second);
  }
  float2 cs[8];
  {
    const int32_t* at = r.pos + (int64_t)b * r.pos_sb + (int64_t)l * r.pos_sl;
    int32_t pos[KVQ_MAX_AXES];
#pragma unroll
    for (int a = 0; a < KVQ_MAX_AXES; ++a) pos[a] = at[(int64_t)min(a, r.axes - 1) * r.pos_sa];
    const u2 axes = *(const u2*)(r.axis + 8 * j);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t a = (axes[e / 4] >> (8 * (e % 4))) & 0xffu;
      const int32_t q = a < 2 ? (a == 0 ? pos[0] : pos[1]) : (a == 2 ? pos[2] : pos[3]);
      cs[e] = cos_sin((double)q * r.freq[8 * j + e]);
    }
  }
#pragma unroll
  for (int k = 0; k < NH; ++k) {
    float a[16];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[2 * e] = to_float((uint16_t)(lo[k][e] & 0xffffu), T{});
      a[2 * e + 1] = to_float((uint16_t)(lo[k][e] >> 16), T{});
      a[8 + 2 * e] = to_float((uint16_t)(hi[k][e] & 0xffffu), T{});
      a[8 + 2 * e + 1] = to_float((uint16_t)(hi[k][e] >> 16), T{});
    }
    uint16_t o[16];
    auto turn = [&](int x0, int y0, int e) {
      const float u = a[x0] * cs[e].x - a[y0] * cs[e].y, v = a[x0] * cs[e].y + a[y0] * cs[e].x;
      o[x0] = from_float(u, T{});
      o[y0] = from_float(v, T{});
    };
    if (r.traditional) {
#pragma unroll
      for (int e = 0; e < 8; ++e) turn(2 * e, 2 * e + 1, e);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) turn(e, 8 + e, e);
    }
    if (k < nh) {
      uint16_t* p = x + (int64_t)k * job.s_h;
      u4 wl, wh;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wl[e] = (uint32_t)o[2 * e] | ((uint32_t)o[2 * e + 1] << 16);
        wh[e] = (uint32_t)o[8 + 2 * e] | ((uint32_t)o[8 + 2 * e + 1] << 16);
      }
      *(u4*)p = wl;
      *(u4*)(p + second) = wh;
    }
  }
}

template <typename T, int NH>
__global__ __launch_bounds__(256) void rope_axes_kernel(RotateJob job, AxesArgs r) {
  rotate_rows<T, NH>(job, r, blockIdx.x);
}

struct AppendJob {
  QuantJob k, v;
  int H, L, per_row;  // chunks of a row
  RowCut cut;
  Div31 div_chunks;
  int codes16, values;  // values: 1 if there are any
  int64_t row_offset;
  PageMap pm;
};

// Quantize rows, rotated first where `tab` is given. A chunk is EPT elements; its group's other chunks are in
// neighbouring lanes.
template <typename T, int BITS, int G, int EPT, bool ROTATE>
__device__ __forceinline__ void append_rows(const AppendJob& a, const QuantJob& job, const AxesArgs& r, const Rows& rows,
                                            float2* tab) {
#pragma clang fp contract(off)
  const int items = rows.nh * rows.nl * a.per_row, half = r.dims / 2;
  const uint32_t nl = (uint32_t)rows.nl;
  if constexpr (ROTATE) {
    fill_table(r, rows.b, rows.l0, rows.nl, tab);
    __syncthreads();
  }
  for (int i0 = 0; i0 < items; i0 += 256) {  // (whole groups stay together: a row holds whole groups)
    const int i = i0 + threadIdx.x;
    const bool active = i < items;
    const int row = active ? (int)div31((uint32_t)i, a.div_chunks) : 0;
    const int chunk = active ? i - row * a.per_row : 0;
    const int h = (int)((uint32_t)row / nl), l = row - h * rows.nl;
    const uint16_t* src = job.src + (int64_t)rows.b * job.s_b + (int64_t)(rows.h0 + h) * job.s_h + (int64_t)(rows.l0 + l) * job.s_l;
    float x[EPT], xp[EPT];
    u4 raw[EPT / 8], rawp[EPT / 8];
#pragma unroll
    for (int j = 0; j < EPT / 8; ++j) raw[j] = *(const u4*)(src + chunk * EPT + 8 * j);
    if constexpr (ROTATE) {
#pragma unroll
      for (int j = 0; j < EPT / 8; ++j) {
        const int d0 = chunk * EPT + 8 * j;
        if (!r.traditional && d0 < r.dims) rawp[j] = *(const u4*)(src + (d0 < half ? d0 + half : d0 - half));
      }
    }
#pragma unroll
    for (int j = 0; j < EPT / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[8 * j + 2 * e] = to_float((uint16_t)(raw[j][e] & 0xffffu), T{});
        x[8 * j + 2 * e + 1] = to_float((uint16_t)(raw[j][e] >> 16), T{});
      }
    if constexpr (ROTATE) {
#pragma unroll
      for (int j = 0; j < EPT / 8; ++j) {
        const int d0 = chunk * EPT + 8 * j;
        if (d0 >= r.dims) continue;
        float* y = x + 8 * j;
        if (r.traditional) {
          const float2* cs = tab + l * r.pairs + d0 / 2;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 t = cs[e];
            const float u = y[2 * e], v = y[2 * e + 1];
            y[2 * e] = to_float(from_float(u * t.x - v * t.y, T{}), T{});
            y[2 * e + 1] = to_float(from_float(u * t.y + v * t.x, T{}), T{});
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            xp[2 * e] = to_float((uint16_t)(rawp[j][e] & 0xffffu), T{});
            xp[2 * e + 1] = to_float((uint16_t)(rawp[j][e] >> 16), T{});
          }
          const bool first = d0 < half;
          const float2* cs = tab + l * r.pairs + (first ? d0 : d0 - half);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 t = cs[e];
            const float z = first ? y[e] * t.x - xp[e] * t.y : xp[e] * t.y + y[e] * t.x;
            y[e] = to_float(from_float(z, T{}), T{});
          }
        }
      }
    }
    Quantized<BITS, EPT> z;
    quantize_chunk<BITS, G, EPT>(x, active, z);
    if (active) store_quantized<T, BITS, G, EPT>(job, z, rows.b, rows.h0 + h, rows.l0 + l, chunk, a.row_offset, a.pm, a.codes16);
  }
}

// One launch for a step's rows: workgroups [0, append) the keys, then the values, then the queries.
template <typename T, int BITS, int G, int EPT>
__global__ __launch_bounds__(256) void rope_axes_append_kernel(AppendJob a, RotateJob q, AxesArgs r) {
  __shared__ float2 tab[kTableCells];
  int wg = (int)blockIdx.x;
  if (wg < a.cut.blocks) {
    append_rows<T, BITS, G, EPT, true>(a, a.k, r, rows_of(a.cut, wg, a.L, a.H), tab);
    return;
  }
  wg -= a.cut.blocks;
  if (a.values) {
    if (wg < a.cut.blocks) {
      append_rows<T, BITS, G, EPT, false>(a, a.v, r, rows_of(a.cut, wg, a.L, a.H), tab);
      return;
    }
    wg -= a.cut.blocks;
  }
  if (q.heads == 2)
    rotate_rows<T, 2>(q, r, (uint32_t)wg);
  else
    rotate_rows<T, 4>(q, r, (uint32_t)wg);
}

// ------------------------------------------------------------------------------------------
// Host side.

static AxesArgs make_axes(const kvq_axes* p) {
  AxesArgs r{};
  r.pos = p->positions;
  r.pos_sa = p->pos_stride_a;
  r.pos_sb = p->pos_stride_b;
  r.pos_sl = p->pos_stride_l;
  r.dims = p->dims;
  r.pairs = p->dims / 2;
  r.traditional = p->traditional;
  r.axes = p->axes;
  r.div_pairs = make_div31((uint32_t)r.pairs);
  int left[KVQ_MAX_AXES], count[KVQ_MAX_AXES] = {};
  for (int a = 0; a < p->axes; ++a) left[a] = p->sections[a];
  for (int i = 0, a = 0; i < r.pairs; ++i) {
    while (left[a] == 0) a = (a + 1) % p->axes;
    r.axis[i] = (uint8_t)a;
    --left[a];
    const double e = p->restart ? (double)count[a]++ / p->sections[a] : (double)i / r.pairs;
    r.freq[i] = (double)p->scale * pow((double)p->base, -e);
    if (p->interleaved) a = (a + 1) % p->axes;
  }
  return r;
}

// Rows of `per_row` items each, B sequences of L positions of H heads. Heads of a position share its sines, so a
// workgroup takes up to 32 of them; then as many positions as give it one item a thread, or four where that
// still leaves 2048 workgroups.
static RowCut cut_rows(int B, int H, int L, int per_row, int pairs) {
  RowCut c{};
  c.per_head = H < 32 ? H : 32;
  c.groups = (H + c.per_head - 1) / c.per_head;
  const int64_t items = (int64_t)B * H * L * per_row, one = (int64_t)c.per_head * per_row;
  const int64_t want = items / 1024 >= 2048 ? 1024 : 256;
  int64_t n = want / one;
  if (n > kTableCells / pairs) n = kTableCells / pairs;
  if (n > L) n = L;
  c.per_pos = n < 1 ? 1 : (int)n;
  c.tiles = (L + c.per_pos - 1) / c.per_pos;
  c.div_groups = make_div31((uint32_t)c.groups);
  c.div_tiles = make_div31((uint32_t)c.tiles);
  const int64_t blocks = (int64_t)B * c.tiles * c.groups;
  c.blocks = blocks < ((int64_t)1 << 29) ? (int)blocks : 0;
  return c;
}

constexpr int64_t kManyItems = 1 << 19;  // a head's 8 pairs; 4 heads a thread from here on (2048 tokens of 32 heads)

static RotateJob make_rotate(const kvq_rows* x, int B, int H, int L, int pairs) {
  RotateJob j{};
  j.x = (uint16_t*)x->data;
  j.s_b = x->stride_b;
  j.s_h = x->stride_h;
  j.s_l = x->stride_l;
  j.H = H;
  j.L = L;
  j.per_row = pairs / 8;
  const int64_t one = (int64_t)B * L * j.per_row;
  j.heads = one * H >= kManyItems ? 4 : 2;
  j.groups = (H + j.heads - 1) / j.heads;
  const int64_t items = one * j.groups;
  if (items >= (int64_t)1 << 31) return j;
  j.items = (uint32_t)items;
  j.blocks = (int)((items + 255) / 256);
  j.div_row = make_div31((uint32_t)j.per_row);
  j.div_l = make_div31((uint32_t)L);
  j.div_groups = make_div31((uint32_t)j.groups);
  return j;
}

hipError_t launch_rope_axes(const kvq_rows* x, const kvq_axes* rope, int B, int H, int L, int dtype, hipStream_t stream) {
  const AxesArgs r = make_axes(rope);
  const RotateJob j = make_rotate(x, B, H, L, r.pairs);
  if (!j.blocks) return hipErrorInvalidValue;
  auto go = [&](auto t) {
    using T = decltype(t);
    const dim3 grid(j.blocks), block(256);
    if (j.heads == 2)
      hipLaunchKernelGGL((rope_axes_kernel<T, 2>), grid, block, 0, stream, j, r);
    else
      hipLaunchKernelGGL((rope_axes_kernel<T, 4>), grid, block, 0, stream, j, r);
    return hipGetLastError();
  };
  return dtype == KVQ_DTYPE_BF16 ? go(BF16{}) : go(F16{});
}

template <typename T, int BITS, int G>
static hipError_t launch_append(AppendJob a, const RotateJob& q, const AxesArgs& r, int B, int D, hipStream_t stream) {
  // 32 elements a thread where that leaves enough of them, as in quantize.hip
  const bool wide = (int64_t)B * a.H * a.L * (D / 32) * (1 + a.values) >= 1024 * 256;
  a.per_row = D / (wide ? 32 : 8);
  a.div_chunks = make_div31((uint32_t)a.per_row);
  a.cut = cut_rows(B, a.H, a.L, a.per_row, r.pairs);
  if (!a.cut.blocks) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(a.cut.blocks * (1 + a.values) + q.blocks));
  if (wide)
    hipLaunchKernelGGL((rope_axes_append_kernel<T, BITS, G, 32>), grid, dim3(256), 0, stream, a, q, r);
  else
    hipLaunchKernelGGL((rope_axes_append_kernel<T, BITS, G, 8>), grid, dim3(256), 0, stream, a, q, r);
  return hipGetLastError();
}

hipError_t launch_rope_axes_append(const kvq_rows* k_src, const kvq_qtensor* k_dst, const kvq_rows* v_src,
                                   const kvq_qtensor* v_dst, const kvq_rows* q, int Hq, const kvq_axes* rope, int num_pages,
                                   const int32_t* table, int64_t table_stride, const int32_t* starts, int64_t row_offset,
                                   int B, int H, int L, int D, int bits, int G, int dtype, hipStream_t stream) {
  const AxesArgs r = make_axes(rope);
  AppendJob a{};
  a.k = make_job(k_src, k_dst);
  a.v = v_src ? make_job(v_src, v_dst) : a.k;
  a.values = v_src ? 1 : 0;
  a.H = H;
  a.L = L;
  a.row_offset = row_offset;
  a.pm = PageMap{table, table_stride, starts, num_pages};
  a.codes16 = 1;
  for (const QuantJob* j : {&a.k, &a.v}) a.codes16 &= (uintptr_t)j->codes % 16 == 0 && (j->c_b | j->c_h | j->c_s) % 4 == 0;
  RotateJob qj{};
  if (q) {
    qj = make_rotate(q, B, Hq, L, r.pairs);
    if (!qj.blocks) return hipErrorInvalidValue;
  }
  auto by_g = [&](auto t, auto b) -> hipError_t {
    using T = decltype(t);
    constexpr int BB = decltype(b)::value;
    if (G == 32) return launch_append<T, BB, 32>(a, qj, r, B, D, stream);
    return G == 64 ? launch_append<T, BB, 64>(a, qj, r, B, D, stream) : launch_append<T, BB, 128>(a, qj, r, B, D, stream);
  };
  auto by_b = [&](auto t) -> hipError_t {
    if (bits == 2) return by_g(t, std::integral_constant<int, 2>{});
    return bits == 4 ? by_g(t, std::integral_constant<int, 4>{}) : by_g(t, std::integral_constant<int, 8>{});
  };
  return dtype == KVQ_DTYPE_BF16 ? by_b(BF16{}) : by_b(F16{});
}

}  // namespace kvq
