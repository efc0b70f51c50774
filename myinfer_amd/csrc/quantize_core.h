// The affine quantizer on a thread's chunk of a row, and where the result goes: shared by the appends
// (quantize.hip, rope_axes.hip). The algorithm is stated in quantize.hip.
#pragma once

#include "common.h"
#include "launch.h"

namespace kvq {

template <typename T>
__device__ __forceinline__ void load8(const uint16_t* p, float (&x)[8]) {
  const u4 raw = *(const u4*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = to_float((uint16_t)(raw[i] & 0xffffu), T{});
    x[2 * i + 1] = to_float((uint16_t)(raw[i] >> 16), T{});
  }
}

struct QuantJob {
  const uint16_t* src;
  int64_t s_b, s_h, s_l;
  uint32_t* codes;
  uint16_t* scales;
  uint16_t* biases;
  int64_t c_b, c_h, c_s;
  int64_t g_b, g_h, g_s;
  int32_t* range_exp;  // the destination cache's range exponent (kvq_qtensor), or null
};

inline QuantJob make_job(const kvq_rows* src, const kvq_qtensor* dst) {
  QuantJob j;
  j.src = (const uint16_t*)src->data;
  j.s_b = src->stride_b;
  j.s_h = src->stride_h;
  j.s_l = src->stride_l;
  j.codes = dst->codes;
  j.scales = (uint16_t*)dst->scales;
  j.biases = (uint16_t*)dst->biases;
  j.c_b = dst->codes_stride_b;
  j.c_h = dst->codes_stride_h;
  j.c_s = dst->codes_stride_s;
  j.g_b = dst->sb_stride_b;
  j.g_h = dst->sb_stride_h;
  j.g_s = dst->sb_stride_s;
  j.range_exp = dst->range_exp;
  return j;
}

// The range exponent a group needs: the smallest E >= 0 with max(|b|, |b + n s|) <= 2^15 * 2^E,
// from the stored (rounded) scale and bias, whose dequantized values s * c + b (c in [0, n]) have
// their extremes at c = 0 and c = n.
__device__ __forceinline__ int group_range_exp(float s, float b, float n) {
#pragma clang fp contract(off)
  const float bound = fmaxf(fabsf(b), fabsf(b + n * s));
  if (!(bound > 32768.0f)) return 0;           // within range (or a NaN group, which no scale mends)
  if (__builtin_isinf(bound)) return 127;      // the largest exponent the kernels accept
  int k;
  const float m = frexpf(bound * (1.0f / 32768.0f), &k);  // bound / 2^15 = m 2^k, m in [0.5, 1)
  return m == 0.5f ? k - 1 : k;
}

// Paged destination: row r of sequence b goes to row r % 64 of page table[b][r / 64] (the job's
// batch strides are then page strides); r = starts[b] + l when `starts` is given, else
// row_offset + l. table == nullptr: the contiguous cache.
struct PageMap {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* starts;
  int num_pages;
};

// v of another lane by a DPP lane permutation: quad_perm [1, 0, 3, 2] and [2, 3, 0, 1] (the lane
// index XOR 1 and XOR 2), row_half_mirror (lane 7 - i of each 8) and row_mirror (15 - i of each 16)
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, false));
}
constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;

// Max and min over the TPG neighbouring lanes of a group (TPG a power of two up to 16): after the
// quad steps every lane of a quad holds its quad's value, so the mirrors exchange whole quads, then
// whole 8-lane halves.
template <int TPG>
__device__ __forceinline__ void group_minmax(float& mx, float& mn) {
  if constexpr (TPG >= 2) {
    mx = fmaxf(mx, dpp<kQuadXor1>(mx));
    mn = fminf(mn, dpp<kQuadXor1>(mn));
  }
  if constexpr (TPG >= 4) {
    mx = fmaxf(mx, dpp<kQuadXor2>(mx));
    mn = fminf(mn, dpp<kQuadXor2>(mn));
  }
  if constexpr (TPG >= 8) {
    mx = fmaxf(mx, dpp<kHalfMirror>(mx));
    mn = fminf(mn, dpp<kHalfMirror>(mn));
  }
  if constexpr (TPG >= 16) {
    mx = fmaxf(mx, dpp<kMirror>(mx));
    mn = fminf(mn, dpp<kMirror>(mn));
  }
}

// A thread's EPT elements quantized: the packed codes, and its group's scale and bias (fp32).
template <int BITS, int EPT>
struct Quantized {
  static constexpr int W = EPT * BITS / 32 > 0 ? EPT * BITS / 32 : 1;  // code words (2-bit, 8 elements: half a word)
  uint32_t packed[W];
  float s, bias;
};

// The G / EPT lanes of a group are neighbours. Inactive lanes take part in the exchange only.
template <int BITS, int G, int EPT>
__device__ __forceinline__ void quantize_chunk(const float (&x)[EPT], bool active, Quantized<BITS, EPT>& z) {
#pragma clang fp contract(off)
  constexpr int TPG = G / EPT;
  float mx = x[0], mn = x[0];
#pragma unroll
  for (int i = 1; i < EPT; ++i) {
    mx = fmaxf(mx, x[i]);
    mn = fminf(mn, x[i]);
  }
  group_minmax<TPG>(mx, mn);
  if (!active) return;

  constexpr float n_bins = (float)((1 << BITS) - 1);
  const bool neg = fabsf(mn) > fabsf(mx);
  float s = fmaxf((mx - mn) / n_bins, 1e-7f);
  s = neg ? s : -s;
  const float edge = neg ? mn : mx;
  const float q0 = rintf(edge / s);
  float bias = 0.0f;
  if (q0 != 0.0f) {
    s = edge / q0;
    bias = edge;
  }

  // code = rint((x - bias) / s) with the quotient rounded as the IEEE division rounds it. The
  // reciprocal estimate (v_rcp_f32, within 1 ulp) refined by one residual step gives q1 within one
  // ulp of that correctly rounded quotient, so rint(q1) can differ from its rint only when a
  // half-integer lies within one ulp. A thread with any quotient within 2 ulp (|q1| 2^-22) of a
  // half-integer, or of magnitude 2^21 or more, or not finite, divides all its elements exactly:
  // the codes stay bit-identical and the division is the rare path.
  constexpr int W = Quantized<BITS, EPT>::W;
  uint32_t packed[W];
  float low = 0.0f;  // 4 bits: the code before, the low nibble of its byte
  auto put = [&](int i, float c) {
    if constexpr (BITS == 8) {
      // one instruction clamps to [0, 255] (NaN to 0, as below), converts and inserts the byte
      packed[i / 4] = __builtin_amdgcn_cvt_pk_u8_f32(c, i % 4, i % 4 == 0 ? 0u : packed[i / 4]);
      return;
    }
    c = fminf(fmaxf(c, 0.0f), n_bins);
    if constexpr (BITS == 4) {  // a byte is low + 16 c, exact
      if (i % 2)
        packed[i / 8] = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_fmaf(c, 16.0f, low), i / 2 % 4,
                                                       i % 8 == 1 ? 0u : packed[i / 8]);
      low = c;
      return;
    }
    const int bit = i * BITS;
    if (bit % 32 == 0) packed[bit / 32] = 0u;
    packed[bit / 32] |= (uint32_t)c << (bit % 32);
  };
  const float rs = __builtin_amdgcn_rcpf(s);
  bool exact = false;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    const float a = x[i] - bias;
    const float qa = a * rs;
    const float q1 = __builtin_fmaf(__builtin_fmaf(-qa, s, a), rs, qa);
    const float c = rintf(q1);
    exact |= !(fabsf(q1 - c) < __builtin_fmaf(fabsf(q1), -0x1p-22f, 0.5f));
    put(i, c);
  }
  if (exact) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) put(i, rintf((x[i] - bias) / s));
  }
#pragma unroll
  for (int w = 0; w < W; ++w) z.packed[w] = packed[w];
  z.s = s;
  z.bias = bias;
}

// The chunk's codes and, from the group's first lane, its scale and bias to row l of the append.
template <typename T, int BITS, int G, int EPT>
__device__ __forceinline__ void store_quantized(const QuantJob& job, const Quantized<BITS, EPT>& z, int64_t b, int h, int64_t l,
                                                int chunk, int64_t row_offset, const PageMap& pm, int codes16) {
  constexpr int W = Quantized<BITS, EPT>::W, TPG = G / EPT;
  constexpr float n_bins = (float)((1 << BITS) - 1);
  const auto& packed = z.packed;
  const float s = z.s, bias = z.bias;
  int64_t drow = row_offset + l, bb = b;
  if (pm.table) {
    const int64_t r = (pm.starts ? (int64_t)pm.starts[b] : row_offset) + l;
    if (r < 0 || (r >> 6) >= pm.table_stride) return;  // a row outside the sequence's table is dropped
    // A table entry outside the pool (such as a -1 "unallocated" sentinel) drops the row too:
    // clamping it would write into a page that may belong to another sequence.
    const int pg = pm.table[b * pm.table_stride + (r >> 6)];
    if (pg < 0 || pg >= pm.num_pages) return;
    bb = pg;
    drow = r & 63;
  }
  uint32_t* cdst = job.codes + bb * job.c_b + h * job.c_h + drow * job.c_s;
  if constexpr (EPT * BITS < 32) {  // 2-bit, 8 elements: 16 bits; two neighbouring threads share a word
    const uint32_t other = (uint32_t)__builtin_amdgcn_ds_bpermute((__lane_id() ^ 1) << 2, (int)packed[0]);
    if ((chunk & 1) == 0) cdst[chunk / 2] = packed[0] | (other << 16);
  } else if (W % 4 == 0 && codes16) {  // 16-byte aligned rows
#pragma unroll
    for (int w = 0; w + 3 < W; w += 4)
      *(u4*)(cdst + chunk * W + w) = u4{packed[w], packed[w + 1], packed[w + 2], packed[w + 3]};
  } else if constexpr (BITS == 8) {  // 8-byte aligned (checked on the host)
#pragma unroll
    for (int w = 0; w < W; w += 2) *(u2*)(cdst + chunk * W + w) = u2{packed[w], packed[w + 1]};
  } else {
#pragma unroll
    for (int w = 0; w < W; ++w) cdst[chunk * W + w] = packed[w];
  }
  if (chunk % TPG == 0) {
    const int64_t gi = bb * job.g_b + h * job.g_h + drow * job.g_s + chunk / TPG;
    const uint16_t sT = from_float(s, T{}), bT = from_float(bias, T{});
    job.scales[gi] = sT;
    job.biases[gi] = bT;
    if (job.range_exp) {
      const int e = group_range_exp(to_float(sT, T{}), to_float(bT, T{}), n_bins);
      if (e > 0) atomicMax(job.range_exp, e);
    }
  }
}

}  // namespace kvq
