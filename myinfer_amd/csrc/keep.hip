// Keeping accepted rows (kvq_keep_rows): after drafted tokens were verified, row start + i of every cache array
// gets what row start + rows[i] held before the call.
//
// A thread owns one unit (16, 4 or 2 bytes, what the array's alignment allows) of a row's width in one (sequence,
// head) and moves it for every row, 16 rows at a time: their loads are all issued before the first store. No
// other thread touches that column, and an entry i below its index is not taken (rows[i] >= i holds
// for every ascending list), so a later load never meets a row that has been overwritten: no barrier, any
// list, in place. Bound by its launch and the latency of the index, page and data loads; the arrays of many
// layers go in one launch.

#include "launch.h"

namespace kvq {

constexpr int kKeepArrays = 192;  // arrays of a launch: 32 layers' codes, scales and biases of K and V
constexpr int kKeepKinds = 6;     // shapes and strides among them
constexpr int kKeepRows = 16;     // rows in flight

struct KeepKind {
  int64_t s_b, s_h, s_l;  // bytes (s_b of a paged array: its page stride)
  int width, unit;        // units of a row, bytes of a unit
};
struct KeepArgs {
  uint8_t* data[kKeepArrays];
  uint8_t kind[kKeepArrays];
  KeepKind kinds[kKeepKinds];
  const int32_t* rows;
  int64_t rows_sb;
  const int32_t* starts;
  int64_t start;
  const int32_t* table;
  int64_t table_stride;
  int num_pages, M, n, H, B;
};

template <typename U, bool PAGED>
__device__ __forceinline__ void move_rows(const KeepArgs& a, uint8_t* base, const KeepKind& k, int b, int64_t start) {
  const int32_t* rows = a.rows + (int64_t)b * a.rows_sb;
  const int32_t* table = PAGED ? a.table + (int64_t)b * a.table_stride : nullptr;
  // the address of a row, or null outside the sequence's pages
  auto at = [&](int64_t r) -> U* {
    if constexpr (PAGED) {
      if (r < 0 || (r >> 6) >= a.table_stride) return nullptr;
      const int pg = table[r >> 6];
      if (pg < 0 || pg >= a.num_pages) return nullptr;
      return (U*)(base + pg * k.s_b + (r & 63) * k.s_l);
    } else {
      return (U*)(base + r * k.s_l);
    }
  };
  for (int i0 = 0; i0 < a.M; i0 += kKeepRows) {
    U v[kKeepRows];
    U* dst[kKeepRows];
#pragma unroll
    for (int i = 0; i < kKeepRows; ++i) {
      const int at_i = i0 + i;
      const int r = at_i < a.M ? rows[at_i] : -1;
      dst[i] = nullptr;
      if (r <= at_i || r >= a.n) continue;  // (a row that stays needs no move)
      const U* src = at(start + r);
      U* d = at(start + at_i);
      if (!src || !d) continue;
      dst[i] = d;
      v[i] = *src;
    }
#pragma unroll
    for (int i = 0; i < kKeepRows; ++i)
      if (dst[i]) *dst[i] = v[i];
  }
}

struct alignas(16) Unit16 {
  uint32_t w[4];
};

template <bool PAGED>
__global__ __launch_bounds__(64) void keep_rows_kernel(KeepArgs a) {
  const KeepKind& k = a.kinds[a.kind[blockIdx.y]];
  const int b = blockIdx.z;
  const int t = blockIdx.x * 64 + threadIdx.x;
  const int h = t / k.width, u = t - h * k.width;
  if (h >= a.H) return;
  const int64_t start = a.starts ? a.starts[b] : a.start;
  uint8_t* base = a.data[blockIdx.y] + (PAGED ? 0 : b * k.s_b) + h * k.s_h + u * k.unit;
  if (k.unit == 16)
    move_rows<Unit16, PAGED>(a, base, k, b, start);
  else if (k.unit == 4)
    move_rows<uint32_t, PAGED>(a, base, k, b, start);
  else
    move_rows<uint16_t, PAGED>(a, base, k, b, start);
}

hipError_t launch_keep_rows(const kvq_row_array* arrays, int n_arrays, int num_pages, const int32_t* table,
                            int64_t table_stride, const int32_t* rows, int64_t rows_sb, const int32_t* starts, int64_t start,
                            int n, int M, int B, int H, hipStream_t stream) {
  int done = 0;
  while (done < n_arrays) {
    KeepArgs a{};
    a.rows = rows;
    a.rows_sb = rows_sb;
    a.starts = starts;
    a.start = start;
    a.table = table;
    a.table_stride = table_stride;
    a.num_pages = num_pages;
    a.M = M;
    a.n = n;
    a.H = H;
    a.B = B;
    int count = 0, kinds = 0, width = 0;
    for (; done < n_arrays && count < kKeepArrays; ++done, ++count) {
      const kvq_row_array& x = arrays[done];
      const int64_t all = (int64_t)(uintptr_t)x.data | x.stride_b | x.stride_h | x.stride_l | x.row_bytes;
      const int unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
      const KeepKind k{x.stride_b, x.stride_h, x.stride_l, (int)(x.row_bytes / unit), unit};
      int i = 0;
      for (; i < kinds; ++i)
        if (a.kinds[i].s_b == k.s_b && a.kinds[i].s_h == k.s_h && a.kinds[i].s_l == k.s_l && a.kinds[i].width == k.width &&
            a.kinds[i].unit == unit)
          break;
      if (i == kinds) {
        if (kinds == kKeepKinds) break;  // a launch of its own for the rest
        a.kinds[kinds++] = k;
      }
      a.data[count] = (uint8_t*)x.data;
      a.kind[count] = (uint8_t)i;
      width = k.width > width ? k.width : width;
    }
    const dim3 grid((unsigned)(((int64_t)H * width + 63) / 64), (unsigned)count, (unsigned)B);
    if (table)
      hipLaunchKernelGGL(keep_rows_kernel<true>, grid, dim3(64), 0, stream, a);
    else
      hipLaunchKernelGGL(keep_rows_kernel<false>, grid, dim3(64), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace kvq
