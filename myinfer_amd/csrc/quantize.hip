// Fused quantize-and-append: new K/V rows -> MLX-layout affine cache (codes, scales, biases).
//
// Algorithm (per group of G consecutive elements of a row), the affine quantizer of
// mx.quantize that mlx-lm's QuantizedKVCache.update_and_fetch applies to every appended row
// (reached from m5engine/attention.py:106-112 and the per-layer cache update):
//   xmax, xmin over the group in fp32; n = 2^bits - 1
//   s = max((xmax - xmin) / n, 1e-7), negated unless |xmin| > |xmax|
//   edge = |xmin| > |xmax| ? xmin : xmax;  q0 = rint(edge / s)
//   if q0 != 0: s = edge / q0, bias = edge   else bias = 0
//   code = clamp(rint((x - bias) / s), 0, n)          (fp32 s and bias, before rounding)
//   stored scale = T(s), bias = T(bias)               (round to nearest even)
// Every operation is IEEE fp32 with round-to-nearest-even (correctly rounded division, rint
// half-to-even), so codes, scales and biases are bit-identical to the CPU restatement.
//
// Thread mapping: one thread per 32 (large launches) or 8 consecutive elements, 16 bytes a load, all
// loads in flight at once; the threads of a group are neighbouring lanes and reduce min/max with
// DPP lane permutes. Grid.y selects the K or the V job of one launch. A large append is bound by its
// bytes and by instruction issue about equally: with codes of 16-byte aligned rows stored 16 bytes at a
// time and bytes made by v_cvt_pk_u8_f32 (clamp, conversion and insertion in one), 2048 rows of 4
// sequences of 16 heads of 128 dims, K and V in 8 bits (103 MB), went from 27.5 to 24.2 us (4.3 TB/s).
//
// RoPE (kvq_rope_quantize_append): the K job rotates its rows before quantizing, the way mlx-lm's
// attention layers rotate keys before the cache update and the reference's native kernel fuses
// the rotation with the KV write (native/src/kernels.metal:106-160). Pair i of a row at position
// p turns by angle = (p * scale) * freq_i, freq_i = 1 / base^(2i / dims), in fp32; the rotated
// value is rounded to T (what RoPE returns) before it is quantized. NeoX pairs (i, i + dims/2)
// are read by each thread from its own chunk and the partner chunk, so no lanes exchange data.

#include "quantize_core.h"

namespace kvq {

constexpr int kMaxRopePairs = 128;

// freq[i] = 1 / base^(2i / dims), computed once on the host in double precision and rounded to
// fp32, so that the angles do not depend on the device's pow (at position 1e5 one ulp of freq
// moves the angle by about 6e-3 rad).
struct RopeArgs {
  int dims, traditional;
  float scale;
  int64_t offset;
  float freq[kMaxRopePairs];
};

// The angle of pair `pair` at position `pos`.
__device__ __forceinline__ float rope_angle(const RopeArgs& r, int64_t pos, int pair) {
#pragma clang fp contract(off)
  return ((float)pos * r.scale) * r.freq[pair];
}

// cos and sin of N angles, the arithmetic that bounds a rotating append (its bytes take a third of its time).
// Below 2^26 an angle is k pi/2 + t, |t| <= pi/4, reduced in double (one FMA: off by k 2^-53 at most, below
// 5e-9 here), where the library's reduction of a large angle is a long integer sequence; then the Taylor
// series of sin and cos about 0 to t^9 and t^10 (remainders 1.8e-9 and 1.2e-10). Against sincosf, the append
// of 2048 rows of 8 heads of 256 dims went from 20.3 to 16.4 us (8 elements a thread). The low part of t
// that the float drops is added back to the sine.
template <int N>
__device__ __forceinline__ void rope_cs(const float (&ang)[N], float (&c)[N], float (&s)[N]) {
#pragma clang fp contract(off)
  bool far = false;
#pragma unroll
  for (int e = 0; e < N; ++e) far |= !(fabsf(ang[e]) < 0x1p26f);  // (and NaN)
  if (__builtin_expect(far, 0)) {
#pragma unroll
    for (int e = 0; e < N; ++e) sincosf(ang[e], &s[e], &c[e]);
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const double k = __builtin_rint((double)ang[e] * 0.63661977236758134308);
    const double td = __builtin_fma(-k, 1.57079632679489661923, (double)ang[e]);
    const float t = (float)td, tl = (float)(td - (double)t), z = t * t;
    float sn = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    sn = __builtin_fmaf(z, sn, 8.3333333e-3f);
    sn = __builtin_fmaf(z, sn, -1.6666667e-1f);
    sn = t + __builtin_fmaf(t * z, sn, tl);
    float cn = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    cn = __builtin_fmaf(z, cn, -1.3888889e-3f);
    cn = __builtin_fmaf(z, cn, 4.1666667e-2f);
    cn = __builtin_fmaf(z, cn, -0.5f);
    cn = __builtin_fmaf(z, cn, 1.0f);
    const int quadrant = (int)k;
    const float a = quadrant & 1 ? cn : sn, b = quadrant & 1 ? sn : cn;
    s[e] = quadrant & 2 ? -a : a;
    c[e] = (quadrant + 1) & 2 ? -b : b;
  }
}

static RopeArgs make_rope_args(const kvq_rope_params* p) {
  RopeArgs r{};
  r.dims = p->dims;
  r.traditional = p->traditional;
  r.scale = p->scale;
  r.offset = p->offset;
  for (int i = 0; i < p->dims / 2 && i < kMaxRopePairs; ++i)
    r.freq[i] = (float)(1.0 / pow((double)p->base, 2.0 * i / (double)p->dims));
  return r;
}

// Rotate the 8 values x of dims [d0, d0 + 8) of a row at position pos. For NeoX pairs, xp holds
// the 8 values at the partner dims (d0 -+ dims/2). Dims at or past r.dims pass through.
__device__ __forceinline__ void rope8(const RopeArgs& r, int64_t pos, int d0, float (&x)[8], const float (&xp)[8]) {
#pragma clang fp contract(off)
  if (d0 >= r.dims) return;
  if (r.traditional) {
    float ang[4], c[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ang[i] = rope_angle(r, pos, d0 / 2 + i);
    rope_cs(ang, c, sn);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * c[i] - b * sn[i];
      x[2 * i + 1] = a * sn[i] + b * c[i];
    }
  } else {
    const int half = r.dims / 2;
    const bool lo = d0 < half;
    float ang[8], c[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) ang[e] = rope_angle(r, pos, (lo ? d0 : d0 - half) + e);
    rope_cs(ang, c, sn);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = lo ? x[e] * c[e] - xp[e] * sn[e] : x[e] * c[e] + xp[e] * sn[e];
  }
}

// The rows [l0, l0 + L) of every (sequence, head) in one launch: thread t quantizes chunk
// t % per_row of row t / per_row (per_row = D / EPT), rows ordered (b, h, l); total < 2^31.
struct RowMap {
  uint32_t total, L, H, per_row;
  Div31 div_c, div_l, div_h;
  int64_t l0;
  int codes16;  // the code rows of both jobs are 16-byte aligned: 4 words a store
};

// EPT elements per thread (EPT / 8 16-byte loads in flight): 32 for launches large enough to fill
// the GPU several times over (fewer instructions per element), 8 for small, latency-bound ones.
template <typename T, int BITS, int G, bool ROPE, int EPT>
__global__ __launch_bounds__(256) void quantize_append_kernel(QuantJob job0, QuantJob job1, RowMap rm,
                                                              int64_t row_offset, RopeArgs rope, PageMap pm) {
#pragma clang fp contract(off)
  constexpr int kEPT = EPT;
  const QuantJob job = blockIdx.y == 0 ? job0 : job1;
  const uint32_t tid = blockIdx.x * 256u + threadIdx.x;
  const bool active = tid < rm.total;
  const uint32_t t = active ? tid : 0u;
  const uint32_t row = div31(t, rm.div_c);
  const int chunk = (int)(t - row * rm.per_row);
  const uint32_t bh = div31(row, rm.div_l);
  const int64_t l = rm.l0 + (int64_t)(row - bh * rm.L);  // the row's position among the appended rows
  const uint32_t b32 = div31(bh, rm.div_h);
  const int h = (int)(bh - b32 * rm.H);
  const int64_t b = b32;

  const uint16_t* srow = job.src + b * job.s_b + h * job.s_h + l * job.s_l;
  float x[kEPT];
  {
    u4 raw[kEPT / 8];  // every load in flight before any conversion
#pragma unroll
    for (int j = 0; j < kEPT / 8; ++j) raw[j] = *(const u4*)(srow + chunk * kEPT + 8 * j);
#pragma unroll
    for (int j = 0; j < kEPT / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[8 * j + 2 * i] = to_float((uint16_t)(raw[j][i] & 0xffffu), T{});
        x[8 * j + 2 * i + 1] = to_float((uint16_t)(raw[j][i] >> 16), T{});
      }
  }
  if constexpr (ROPE) {
    if (blockIdx.y == 0) {  // the K job
      const int half = rope.dims / 2;
      const int64_t pos = rope.offset + (pm.starts ? pm.starts[b] : 0) + l;
#pragma unroll
      for (int j = 0; j < kEPT / 8; ++j) {
        const int d0 = chunk * kEPT + 8 * j;
        float xs[8], xp[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) xs[i] = x[8 * j + i];
        if (!rope.traditional && d0 < rope.dims) load8<T>(srow + (d0 < half ? d0 + half : d0 - half), xp);
        rope8(rope, pos, d0, xs, xp);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[8 * j + i] = to_float(from_float(xs[i], T{}), T{});
      }
    }
  }
  Quantized<BITS, EPT> z;
  quantize_chunk<BITS, G, EPT>(x, active, z);
  if (!active) return;
  store_quantized<T, BITS, G, EPT>(job, z, b, h, l, chunk, row_offset, pm, rm.codes16);
}

template <typename T, int BITS, int G>
static hipError_t launch_quant(const QuantJob& k, const QuantJob& v, int njobs, int B, int H, int L, int D,
                               int64_t row_offset, const RopeArgs* rope, const PageMap& pm, hipStream_t stream) {
  // rows per launch: the thread index of every launch stays below 2^31 (more rows take more launches)
  // 32 elements per thread where that launch still has 2 workgroups per CU (512 in all), 4 with the rotation,
  // whose longer threads need more of them in flight: without it 1024 rows of 8 heads of 256 dims (8-bit, 512
  // workgroups) take 6.9 us at 8 elements and 5.3 at 32, with it 9.8 and 9.9, and 2048 rows 16.4 and 13.3
  const bool wide = (int64_t)B * H * L * (D / 32) * njobs >= (rope ? 1024 : 512) * 256;
  const int ept = wide ? 32 : 8;
  const int64_t per_l = (int64_t)B * H * (D / ept);
  if (per_l >= ((int64_t)1 << 31)) return hipErrorInvalidValue;
  const int64_t max_l = (((int64_t)1 << 31) - 1) / per_l;
  RowMap rm{};
  rm.H = (uint32_t)H;
  rm.div_h = make_div31((uint32_t)H);
  rm.per_row = (uint32_t)(D / ept);
  rm.codes16 = 1;
  for (const QuantJob* j : {&k, &v})
    if (j == &k || njobs > 1)
      rm.codes16 &= (uintptr_t)j->codes % 16 == 0 && (j->c_b | j->c_h | j->c_s) % 4 == 0;
  rm.div_c = make_div31(rm.per_row);
  for (int64_t l0 = 0; l0 < L; l0 += max_l) {
    const int64_t nl = L - l0 < max_l ? L - l0 : max_l;
    rm.L = (uint32_t)nl;
    rm.div_l = make_div31((uint32_t)nl);
    rm.total = (uint32_t)(per_l * nl);
    rm.l0 = l0;
    const unsigned blocks = (unsigned)((rm.total + 255u) / 256u);
    const RopeArgs ra = rope ? *rope : RopeArgs{};
    if (rope && wide)
      hipLaunchKernelGGL((quantize_append_kernel<T, BITS, G, true, 32>), dim3(blocks, njobs), dim3(256), 0, stream, k, v,
                         rm, row_offset, ra, pm);
    else if (rope)
      hipLaunchKernelGGL((quantize_append_kernel<T, BITS, G, true, 8>), dim3(blocks, njobs), dim3(256), 0, stream, k, v,
                         rm, row_offset, ra, pm);
    else if (wide)
      hipLaunchKernelGGL((quantize_append_kernel<T, BITS, G, false, 32>), dim3(blocks, njobs), dim3(256), 0, stream, k,
                         v, rm, row_offset, ra, pm);
    else
      hipLaunchKernelGGL((quantize_append_kernel<T, BITS, G, false, 8>), dim3(blocks, njobs), dim3(256), 0, stream, k,
                         v, rm, row_offset, ra, pm);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int BITS>
static hipError_t dispatch_group(int G, const QuantJob& k, const QuantJob& v, int njobs, int B, int H, int L, int D,
                                 int64_t row_offset, const RopeArgs* rope, const PageMap& pm, hipStream_t stream) {
  switch (G) {
    case 32: return launch_quant<T, BITS, 32>(k, v, njobs, B, H, L, D, row_offset, rope, pm, stream);
    case 64: return launch_quant<T, BITS, 64>(k, v, njobs, B, H, L, D, row_offset, rope, pm, stream);
    default: return launch_quant<T, BITS, 128>(k, v, njobs, B, H, L, D, row_offset, rope, pm, stream);
  }
}

template <typename T>
static hipError_t dispatch_bits(int bits, int G, const QuantJob& k, const QuantJob& v, int njobs, int B, int H, int L,
                                int D, int64_t row_offset, const RopeArgs* rope, const PageMap& pm, hipStream_t stream) {
  switch (bits) {
    case 2: return dispatch_group<T, 2>(G, k, v, njobs, B, H, L, D, row_offset, rope, pm, stream);
    case 4: return dispatch_group<T, 4>(G, k, v, njobs, B, H, L, D, row_offset, rope, pm, stream);
    default: return dispatch_group<T, 8>(G, k, v, njobs, B, H, L, D, row_offset, rope, pm, stream);
  }
}

hipError_t launch_quantize_append(const kvq_rows* k_src, const kvq_qtensor* k_dst, const kvq_rows* v_src,
                                  const kvq_qtensor* v_dst, const kvq_rope_params* rope, int64_t row_offset, int B, int H,
                                  int L, int D, int bits, int group_size, int dtype, hipStream_t stream) {
  QuantJob k = make_job(k_src, k_dst);
  QuantJob v = v_src ? make_job(v_src, v_dst) : k;
  const int njobs = v_src ? 2 : 1;
  RopeArgs ra{};
  if (rope) ra = make_rope_args(rope);
  const RopeArgs* rp = rope ? &ra : nullptr;
  const PageMap pm{nullptr, 0, nullptr, 0};
  if (dtype == KVQ_DTYPE_BF16)
    return dispatch_bits<BF16>(bits, group_size, k, v, njobs, B, H, L, D, row_offset, rp, pm, stream);
  return dispatch_bits<F16>(bits, group_size, k, v, njobs, B, H, L, D, row_offset, rp, pm, stream);
}

hipError_t launch_paged_quantize_append(const kvq_rows* k_src, const kvq_qtensor* k_pool, const kvq_rows* v_src,
                                        const kvq_qtensor* v_pool, int num_pages, const int32_t* table,
                                        int64_t table_stride, const int32_t* starts, int64_t row_offset,
                                        const kvq_rope_params* rope, int B, int H, int L, int D, int bits,
                                        int group_size, int dtype, hipStream_t stream) {
  QuantJob k = make_job(k_src, k_pool);
  QuantJob v = v_src ? make_job(v_src, v_pool) : k;
  const int njobs = v_src ? 2 : 1;
  RopeArgs ra{};
  if (rope) ra = make_rope_args(rope);
  const RopeArgs* rp = rope ? &ra : nullptr;
  const PageMap pm{table, table_stride, starts, num_pages};
  if (dtype == KVQ_DTYPE_BF16)
    return dispatch_bits<BF16>(bits, group_size, k, v, njobs, B, H, L, D, row_offset, rp, pm, stream);
  return dispatch_bits<F16>(bits, group_size, k, v, njobs, B, H, L, D, row_offset, rp, pm, stream);
}

// In-place RoPE: one thread per rotated pair of 8-value chunks (NeoX: dims [8j, +8) and
// [8j + dims/2, +8); interleaved: one chunk), so no thread reads what another writes.
template <typename T>
__global__ __launch_bounds__(256) void rope_kernel(uint16_t* x, int64_t s_b, int64_t s_h, int64_t s_l, int H, int L,
                                                   int64_t total, int per_row, RopeArgs r) {
  const int64_t tid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (tid >= total) return;
  const int j = (int)(tid % per_row);
  const int64_t row = tid / per_row;
  const int l = (int)(row % L), h = (int)((row / L) % H);
  const int64_t b = row / ((int64_t)L * H);
  uint16_t* xr = x + b * s_b + h * s_h + (int64_t)l * s_l;
  const int64_t pos = r.offset + l;
  auto store8 = [&](uint16_t* p, const float (&v)[8]) {
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)from_float(v[2 * i], T{}) | ((uint32_t)from_float(v[2 * i + 1], T{}) << 16);
    *(u4*)p = w;
  };
  float a[8], c[8];
  if (r.traditional) {
    load8<T>(xr + 8 * j, a);
    rope8(r, pos, 8 * j, a, c);
    store8(xr + 8 * j, a);
  } else {
    const int half = r.dims / 2;
    load8<T>(xr + 8 * j, a);
    load8<T>(xr + 8 * j + half, c);
    float a2[8], c2[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a2[i] = a[i];
      c2[i] = c[i];
    }
    rope8(r, pos, 8 * j, a2, c);         // first half: a * cos - c * sin
    rope8(r, pos, 8 * j + half, c2, a);  // second half: c * cos + a * sin
    store8(xr + 8 * j, a2);
    store8(xr + 8 * j + half, c2);
  }
}

hipError_t launch_rope(const kvq_rows* x, const kvq_rope_params* rope, int B, int H, int L, int dtype, hipStream_t stream) {
  const RopeArgs r = make_rope_args(rope);
  const int per_row = rope->traditional ? rope->dims / 8 : rope->dims / 16;
  const int64_t total = (int64_t)B * H * L * per_row;
  const int64_t blocks = (total + 255) / 256;
  if (dtype == KVQ_DTYPE_BF16)
    hipLaunchKernelGGL((rope_kernel<BF16>), dim3((unsigned)blocks), dim3(256), 0, stream, (uint16_t*)x->data,
                       x->stride_b, x->stride_h, x->stride_l, H, L, total, per_row, r);
  else
    hipLaunchKernelGGL((rope_kernel<F16>), dim3((unsigned)blocks), dim3(256), 0, stream, (uint16_t*)x->data,
                       x->stride_b, x->stride_h, x->stride_l, H, L, total, per_row, r);
  return hipGetLastError();
}

}  // namespace kvq
