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
// What bounds it: each row is read and written once (rotated in place, or read and stored quantized), and a
// pair's sine and cosine cost more than its rotation. A workgroup therefore takes some positions of
// several heads: it forms the sines and cosines of its positions once, into LDS, and every head's rows use them.

#include "quantize_core.h"

namespace kvq {

constexpr int kAxesPairs = 128;    // pairs of a row at most
constexpr int kTableCells = 2048;  // (position, pair) cells of a workgroup's table: 16 KiB

struct AxesArgs {
  const int32_t* pos;
  int64_t pos_sa, pos_sb, pos_sl;
  int dims, pairs, traditional;
  Div31 div_pairs;
  double freq[kAxesPairs];  // times the position scale
  uint8_t axis[kAxesPairs];
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
  int H;
  RowCut cut;
  Div31 div_items;  // items (8 pairs each) of a row
};

// Rotate rows in place: a thread takes 8 pairs of a row at a time (split halves: dims [8j, +8) and [8j + dims/2,
// +8); interleaved: dims [16j, +16)), the next item's loads issued before the present one is computed.
template <typename T>
__device__ __forceinline__ void rotate_rows(const RotateJob& job, const AxesArgs& r, const Rows& rows, float2* tab) {
#pragma clang fp contract(off)
  const int per_row = r.pairs / 8, items = rows.nh * rows.nl * per_row;
  const int second = r.traditional ? 8 : r.dims / 2;
  const uint32_t nl = (uint32_t)rows.nl;
  auto at = [&](int i, int& l, int& j) -> uint16_t* {
    const int row = (int)div31((uint32_t)i, job.div_items);
    j = i - row * per_row;
    const int h = (int)((uint32_t)row / nl);
    l = row - h * rows.nl;
    return job.x + (int64_t)rows.b * job.s_b + (int64_t)(rows.h0 + h) * job.s_h + (int64_t)(rows.l0 + l) * job.s_l +
           (r.traditional ? 16 : 8) * j;
  };
  int i = threadIdx.x, l = 0, j = 0;
  uint16_t* p = nullptr;
  u4 lo{}, hi{};
  if (i < items) {
    p = at(i, l, j);
    lo = *(const u4*)p;
    hi = *(const u4*)(p + second);
  }
  fill_table(r, rows.b, rows.l0, rows.nl, tab);
  __syncthreads();
  while (i < items) {
    const int ni = i + 256;
    uint16_t* np = nullptr;
    int n_l = 0, nj = 0;
    u4 nlo{}, nhi{};
    if (ni < items) {
      np = at(ni, n_l, nj);
      nlo = *(const u4*)np;
      nhi = *(const u4*)(np + second);
    }
    float a[16];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[2 * e] = to_float((uint16_t)(lo[e] & 0xffffu), T{});
      a[2 * e + 1] = to_float((uint16_t)(lo[e] >> 16), T{});
      a[8 + 2 * e] = to_float((uint16_t)(hi[e] & 0xffffu), T{});
      a[8 + 2 * e + 1] = to_float((uint16_t)(hi[e] >> 16), T{});
    }
    const float2* cs = tab + l * r.pairs + 8 * j;
    uint16_t o[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 t = cs[e];
      const float x = r.traditional ? a[2 * e] : a[e], y = r.traditional ? a[2 * e + 1] : a[8 + e];
      const uint16_t u = from_float(x * t.x - y * t.y, T{}), v = from_float(x * t.y + y * t.x, T{});
      if (r.traditional) {
        o[2 * e] = u;
        o[2 * e + 1] = v;
      } else {
        o[e] = u;
        o[8 + e] = v;
      }
    }
    u4 wl, wh;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      wl[e] = (uint32_t)o[2 * e] | ((uint32_t)o[2 * e + 1] << 16);
      wh[e] = (uint32_t)o[8 + 2 * e] | ((uint32_t)o[8 + 2 * e + 1] << 16);
    }
    *(u4*)p = wl;
    *(u4*)(p + second) = wh;
    i = ni;
    p = np;
    l = n_l;
    j = nj;
    lo = nlo;
    hi = nhi;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void rope_axes_kernel(RotateJob job, AxesArgs r, int L) {
  __shared__ float2 tab[kTableCells];
  rotate_rows<T>(job, r, rows_of(job.cut, (int)blockIdx.x, L, job.H), tab);
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
  rotate_rows<T>(q, r, rows_of(q.cut, wg, a.L, q.H), tab);
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

static RotateJob make_rotate(const kvq_rows* x, int B, int H, int L, int pairs) {
  RotateJob j{};
  j.x = (uint16_t*)x->data;
  j.s_b = x->stride_b;
  j.s_h = x->stride_h;
  j.s_l = x->stride_l;
  j.H = H;
  j.cut = cut_rows(B, H, L, pairs / 8, pairs);
  j.div_items = make_div31((uint32_t)(pairs / 8));
  return j;
}

hipError_t launch_rope_axes(const kvq_rows* x, const kvq_axes* rope, int B, int H, int L, int dtype, hipStream_t stream) {
  const AxesArgs r = make_axes(rope);
  const RotateJob j = make_rotate(x, B, H, L, r.pairs);
  if (!j.cut.blocks) return hipErrorInvalidValue;
  if (dtype == KVQ_DTYPE_BF16)
    hipLaunchKernelGGL((rope_axes_kernel<BF16>), dim3(j.cut.blocks), dim3(256), 0, stream, j, r, L);
  else
    hipLaunchKernelGGL((rope_axes_kernel<F16>), dim3(j.cut.blocks), dim3(256), 0, stream, j, r, L);
  return hipGetLastError();
}

template <typename T, int BITS, int G>
static hipError_t launch_append(AppendJob a, const RotateJob& q, const AxesArgs& r, int B, int D, hipStream_t stream) {
  // 32 elements a thread where that leaves enough of them, as in quantize.hip
  const bool wide = (int64_t)B * a.H * a.L * (D / 32) * (1 + a.values) >= 1024 * 256;
  a.per_row = D / (wide ? 32 : 8);
  a.div_chunks = make_div31((uint32_t)a.per_row);
  a.cut = cut_rows(B, a.H, a.L, a.per_row, r.pairs);
  if (!a.cut.blocks) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(a.cut.blocks * (1 + a.values) + q.cut.blocks));
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
    if (!qj.cut.blocks) return hipErrorInvalidValue;
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
