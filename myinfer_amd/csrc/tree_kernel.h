// Attention of a tree's query rows over a quantized or an unquantized cache, for some tens of rows of a KV head
// (a drafted tree's nodes times the query heads of a GQA group), head_dim 64 or 128.
//
//   out = softmax(scale * q K^T + M) V, M by the tree (tree.h); K = sK * codesK + bK, V = sV * codesV + bV
//
// The decode kernel's 16 MFMA columns hold 8 rows (128 dims, groups of 64) and the prefill kernel's workgroups compute
// 256 rows whether they are there or not: between them neither is near the time of the keys' bytes. Here:
//  * A workgroup serves 32 rows of one (sequence, KV head) over a range of keys; its 4 waves take 32-key tiles in
//    turn, each through a ring of its own (buffer->LDS DMA, as the decode kernel), so no barrier stands in the
//    key loop and two workgroups fit a CU.
//  * S^T = K Q^T with v_mfma_f32_32x32x16: lane n is key n and dequantizes its half row straight from the raw tile
//    into the A operand (its group's scale and bias are two registers); no dequantized tile is written to LDS.
//    The lane halves take halves of the row (dims hh D/2 + 8j in k-step j), which the query operand follows.
//  * Every lane then holds 16 scores of one row: maximum and sum are lane-local, and the packed probabilities are the
//    B operand of O^T = V^T P^T.
//  * V^T: lane n owns dims (D/32) n .. of 8 keys a k-step; byte permutes (4 bits: masks) pair neighbouring keys, and
//    packed FMAs apply their scales and biases, which the wave's lanes converted once per tile into a small table.
//  * Splits are merged as the decode kernel's are: up to 4 by the last to finish, more by combine_kernel.
// Operands and roundings are the prefill kernel's: q times a power of two in fp16 (exact), K and V dequantized to fp16
// (a bf16 cache's times 2^-E), probabilities in fp16, everything else in fp32; an unquantized cache runs in its own
// type. E follows from the scales and biases of the tile itself (K) or of the wave's tiles so far (V), 0 while they fit
// fp16: the cache's range word is not needed, so pages without one do not have to fall back on the decode kernel.
//
// Measured with the merge (decode kernel / here / prefill kernel, us): 8 KV heads over 32768 keys of 128 dims in 8 bits
// (75 MB, 14.5 us as a copy), 32 rows 38.7 / 31.3 / 51.0, 64 rows 64.5 / 32.7 / 50.8, 128 rows 116 / 48.8 / 53.6;
// 8 sequences of 6144 keys in 4 bits, 64 rows 68.9 / 40.3 / 71.8. Bound by the vector ALUs, 75% busy at 512 rows: a tile
// is about 320 vector instructions (16 of them exponentials, four times as long) and 80 scalar ones beside 24 MFMAs;
// calls of few tiles a wave (the second, 12) spend as long again before and after them. Blocks of 64 rows
// (dequantized once for two) came to 35.0 us at 64 rows, 47.3 at 128: one wave a SIMD then hides less than the second
// block saves. tree_kernel_of (capi.hip) has the rule between the three.

#pragma once

#include <math.h>

#include <type_traits>

#include "decode_kernel.h"
#include "dma.h"

namespace kvq {

constexpr int kTW = 4;  // waves

template <int D, int BITS, int G>
struct TreeCfg {
  static constexpr bool DENSE = BITS == 16;
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  static constexpr int NG = DENSE ? 1 : D / G;
  static constexpr int KSTEPS = D / 16;
  static constexpr int DPL = D / 32;           // dims a lane owns in V^T, and its 32-dim blocks
  static constexpr int ROWB = D * BITS / 8;    // bytes of a row's codes
  static constexpr int CPR = ROWB / 16;        // 16-byte chunks of a row
  static constexpr int HC = CPR / 2;           // ... of a lane's half
  static constexpr int TB = kTile * ROWB;
  static constexpr int CI = TB / 1024;         // DMA instructions of a K (or V) tile
  static constexpr int RPI = 64 / CPR;         // rows of one
  // scales and biases: cell 32 g + key (4 bytes, the value in the low half) of each of sK, bK, sV, bV; one DMA fills
  // 64 cells, two groups of 32 keys
  static constexpr int NSB = DENSE ? 0 : NG > 2 ? NG / 2 : 1;
  static constexpr int AS = 256 * NSB;
  static constexpr int SLOT = 2 * TB + 4 * AS;
  static constexpr int IPT = 2 * CI + 4 * NSB;  // DMA instructions of a tile
  // A lane half reads chunk c of 32 rows at once: rows 32 / CPR apart share banks (512 bytes), so they hold it at
  // distinct positions c ^ swz(row).
  static constexpr __host__ __device__ int swz(int r) { return (r / (32 / CPR)) % CPR; }
  // the dequantizing kernels' table of a tile's V scales and biases: fp16 [2][NG][32] per wave
  static constexpr int TAB = DENSE ? 0 : 2 * NG * 32 * 2;
  static constexpr int R = 32;        // query rows
  static constexpr int ORow = D + 4;  // floats of a row in the waves' merge (rows shift by 4 banks)
  static constexpr int SLOTS = 2;     // ring slots of a wave
  static constexpr int RING = kTW * SLOTS * SLOT;
  static constexpr int EPI = kTW * R * (ORow + 2) * 4;
  static constexpr int LDS = (RING + kTW * TAB) > EPI ? RING + kTW * TAB : EPI;
  static constexpr int MINWG = 2 * LDS + 16 <= 160 * 1024 ? 2 : 1;
};

// N bytes at an LDS address as a register (1, 2 or 4 bytes) or two.
template <int N>
struct VRaw;
template <>
struct VRaw<1> {
  uint32_t w;
  __device__ __forceinline__ void load(const uint8_t* p) { w = *p; }
};
template <>
struct VRaw<2> {
  uint32_t w;
  __device__ __forceinline__ void load(const uint8_t* p) { w = *(const uint16_t*)p; }
};
template <>
struct VRaw<4> {
  uint32_t w;
  __device__ __forceinline__ void load(const uint8_t* p) { w = *(const uint32_t*)p; }
};
template <>
struct VRaw<8> {
  u2 w;
  __device__ __forceinline__ void load(const uint8_t* p) { w = *(const u2*)p; }
};

__device__ __forceinline__ h2 as_h2(uint32_t x) { return __builtin_bit_cast(h2, x); }
__device__ __forceinline__ uint32_t as_u32(h2 x) { return __builtin_bit_cast(uint32_t, x); }

// The two code bytes of a word that `sel` picks times scales plus biases: 1024 + c is exact in fp16, the FMA rounds once.
__device__ __forceinline__ uint32_t dequant_bytes(uint32_t bytes, uint32_t sel, uint32_t s2, uint32_t b2) {
  const h2 x = as_h2(perm(0x64646464u, bytes, sel)) - h2{(_Float16)1024.0f, (_Float16)1024.0f};
  return as_u32(x * as_h2(s2) + as_h2(b2));
}

// 4-bit codes of a word's two halves, nibbles 0 .. 3 of each: out[i] is the pair of nibbles i, dequantized. In the mantissa
// of 1024 a nibble at bits 4 .. 7 counts 16 times: (1024 + 16 c) / 16 - 64 is c, exact.
__device__ __forceinline__ void dequant_nibbles(uint32_t w, uint32_t s2, uint32_t b2, uint32_t (&out)[4]) {
  constexpr uint32_t M = 0x64006400u;
  const h2 one = {(_Float16)-1024.0f, (_Float16)-1024.0f}, six = {(_Float16)0.0625f, (_Float16)0.0625f},
           off = {(_Float16)-64.0f, (_Float16)-64.0f};
  const uint32_t w8 = w >> 8;
  const h2 c[4] = {as_h2((w & 0x000F000Fu) | M) + one, as_h2((w & 0x00F000F0u) | M) * six + off,
                   as_h2((w8 & 0x000F000Fu) | M) + one, as_h2((w8 & 0x00F000F0u) | M) * six + off};
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = as_u32(c[i] * as_h2(s2) + as_h2(b2));
}

template <typename T>
__device__ __forceinline__ _Float16 operand_half(uint32_t cell, float m) {
  if constexpr (T::id == KVQ_DTYPE_BF16) return (_Float16)(__uint_as_float(cell << 16) * m);
  return __builtin_bit_cast(_Float16, (uint16_t)cell);
}

// The larger of |bias| and |bias + top code * scale|: what a group's values are bounded by.
template <int BITS>
__device__ __forceinline__ float group_bound(uint32_t s_cell, uint32_t b_cell) {
  const float s = __uint_as_float(s_cell << 16), b = __uint_as_float(b_cell << 16);
  return fmaxf(fabsf(b), fabsf(fmaf((float)((1 << BITS) - 1), s, b)));
}

constexpr float kHalfSafe = 32768.0f;  // operands stay within it (the rounding of a value next to 65504 may not)

// The smallest e >= 0 with every lane's bound <= 2^15 2^e (bounds that are NaN ask for nothing).
__device__ __forceinline__ int bound_exponent(float bound) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) bound = fmaxf(bound, __shfl_xor(bound, m));
  int e = 0;
  if (bound > kHalfSafe) {
    const float f = frexpf(bound * (1.0f / kHalfSafe), &e);  // bound <= 2^15 2^e
    if (f == 0.5f) --e;
    e = min(max(e, 0), 127);
    if (bound == INFINITY) e = 127;
  }
  return e;
}

// Keys of a workgroup: the sequence's keys from `base` in whole tiles, an even share for each split that is a multiple of
// the waves' tiles.
struct TreeSplit {
  int begin, end;
};
__device__ __forceinline__ TreeSplit tree_split(const DecParams& p, int S_b, int split) {
  const int base = p.window > 0 ? max(0, S_b - p.L - p.window + 1) & ~(kTile - 1) : 0;
  const int tiles = (S_b - base + kTile - 1) / kTile;
  const int per = (tiles + p.nsplit - 1) / p.nsplit;
  const int chunk = (per + kTW - 1) / kTW * (kTW * kTile);
  TreeSplit s;
  s.begin = base + split * chunk;
  s.end = min(s.begin + chunk, S_b);
  return s;
}

template <typename T, int D, int BITS, int G, bool PAGED>
__global__ __launch_bounds__(kTW * 64, (TreeCfg<D, BITS, G>::MINWG)) void tree_attn_kernel(DecParams p) {
  using C = TreeCfg<D, BITS, G>;
  using OT = typename std::conditional<C::DENSE, T, F16>::type;  // operand type
  __shared__ __align__(16) uint8_t smem[C::LDS];
  __shared__ unsigned s_prev;
  const int lane = __lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, hh = lane >> 5;

  // ---- workgroup -> (sequence, KV head), split, row block: the row blocks of one key range are neighbours
  const int wg0 = blockIdx.x;
  const int wg = p.xcd_remap ? (wg0 % kXcds) * ((p.nunits * p.nsplit) / kXcds) + wg0 / kXcds : wg0;
  const int t0 = (int)div31((uint32_t)wg, p.d_rowblocks);
  const int rb = wg - t0 * p.rowblocks;
  const int bk = (int)div31((uint32_t)t0, p.d_nsplit);
  const int split = t0 - bk * p.nsplit;
  const int unit = bk * p.rowblocks + rb;
  const int b = (int)div31((uint32_t)bk, p.d_hkv);
  const int kvh = bk - b * p.Hkv;
  const int S_b = p.seq_lens ? min(max(load_uniform_i32(p.seq_lens, b), 0), p.S) : p.S;
  const TreeSplit ks = tree_split(p, S_b, split);
  const int ntile = ks.end > ks.begin ? (ks.end - ks.begin + kTile - 1) / kTile : 0;
  const int nmine = ntile > wave ? (ntile - wave + kTW - 1) / kTW : 0;  // tiles wave, wave + kTW, ...

  // ---- this lane's row (MFMA column n) and its raw query half
  const int first = S_b - p.L;  // the tree's first row
  const int row = rb * C::R + n;
  const bool row_ok = row < p.nrows;
  const int rq = (int)div31((uint32_t)row, p.d_l);
  const int hq = kvh * p.rep + (row_ok ? rq : 0);
  const int lq = row_ok ? row - rq * p.L : 0;
  const uint16_t* qrow = p.q + (int64_t)b * p.q_sb + (int64_t)hq * p.q_sh + (int64_t)lq * p.q_sl + hh * (D / 2);
  u4 qop[C::KSTEPS];
#pragma unroll
  for (int j = 0; j < C::KSTEPS; ++j) qop[j] = *(const u4*)(qrow + 8 * j);
  TreeRow node;
  node.load(p.tree, b, lq, first);
  const int lo_r = p.window > 0 ? max(0, first + node.depth - p.window + 1) : 0;

  // ---- tile stream
  const uint8_t* kbase = p.kc + (int64_t)kvh * p.kc_sh + (PAGED ? 0 : (int64_t)b * p.kc_sb);
  const uint8_t* vbase = p.vc + (int64_t)kvh * p.vc_sh + (PAGED ? 0 : (int64_t)b * p.vc_sb);
  const uint16_t* sbase[4] = {p.ks, p.kb, p.vs, p.vb};
  if constexpr (!C::DENSE) {
#pragma unroll
    for (int a = 0; a < 4; ++a)
      sbase[a] += (int64_t)kvh * (a < 2 ? p.ksb_sh : p.vsb_sh) + (PAGED ? 0 : (int64_t)b * (a < 2 ? p.ksb_sb : p.vsb_sb));
  }
  uint32_t dk[C::CI], dv[C::CI], dsk[C::NSB > 0 ? C::NSB : 1], dsv[C::NSB > 0 ? C::NSB : 1];
#pragma unroll
  for (int c = 0; c < C::CI; ++c) {
    const int r = c * C::RPI + lane / C::CPR, cc = lane % C::CPR;
    dk[c] = (uint32_t)(r * p.kc_ss + 16 * (cc ^ C::swz(r)));
    dv[c] = (uint32_t)(r * p.vc_ss + 16 * cc);
  }
#pragma unroll
  for (int h = 0; h < C::NSB; ++h) {
    const int g = C::NG >= 2 ? 2 * h + hh : 0;
    dsk[h] = (uint32_t)(2 * (n * p.ksb_ss + g));
    dsv[h] = (uint32_t)(2 * (n * p.vsb_ss + g));
  }
  uint8_t* const ring = smem + wave * (C::SLOTS * C::SLOT);
  const uint32_t ring_lds = lds_addr(ring);
  const int last = max(nmine - 1, 0);
  auto tile_k0 = [&](int i) { return ks.begin + kTile * (wave + kTW * min(i, last)); };
  // a paged tile lies in one 64-row page, read one tile ahead (clamped to the pool); its resources span the page's valid
  // rows, so rows past S_b read as zero either way
  auto page_of = [&](int k0) -> int {
    const int pi = min(k0, max(S_b - 1, 0)) >> 6;
    return __builtin_amdgcn_readfirstlane(min(max(p.table[(int64_t)b * p.table_stride + pi], 0), p.num_pages - 1));
  };
  int pg_next = PAGED ? page_of(tile_k0(0)) : 0;
  auto issue = [&](int i) __attribute__((always_inline)) {  // past the last tile it is loaded again
    const int k0 = __builtin_amdgcn_readfirstlane(tile_k0(i));
    const uint32_t slot = ring_lds + (uint32_t)((i % C::SLOTS) * C::SLOT);
    const uint8_t *kp = kbase, *vp = vbase;
    const uint16_t* sp[4] = {sbase[0], sbase[1], sbase[2], sbase[3]};
    int nv = S_b, r0 = k0;
    if constexpr (PAGED) {
      const int pg = pg_next;
      pg_next = page_of(tile_k0(i + 1));
      nv = __builtin_amdgcn_readfirstlane(max(min(64, S_b - (k0 & ~63)), 0));
      r0 = k0 & 63;
      kp += (int64_t)pg * p.kc_sb;
      vp += (int64_t)pg * p.vc_sb;
      if constexpr (!C::DENSE) {
#pragma unroll
        for (int a = 0; a < 4; ++a) sp[a] += (int64_t)pg * (a < 2 ? p.ksb_sb : p.vsb_sb);
      }
    }
    const __amdgpu_buffer_rsrc_t kr = make_rsrc(kp, (uint32_t)((int64_t)nv * p.kc_ss));
    const __amdgpu_buffer_rsrc_t vr = make_rsrc(vp, (uint32_t)((int64_t)nv * p.vc_ss));
#pragma unroll
    for (int c = 0; c < C::CI; ++c) dma_b128(kr, slot + 1024 * c, dk[c], (uint32_t)(r0 * p.kc_ss));
#pragma unroll
    for (int c = 0; c < C::CI; ++c) dma_b128(vr, slot + C::TB + 1024 * c, dv[c], (uint32_t)(r0 * p.vc_ss));
    if constexpr (!C::DENSE) {
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int64_t ss = a < 2 ? p.ksb_ss : p.vsb_ss;
        const __amdgpu_buffer_rsrc_t r = make_rsrc(sp[a], (uint32_t)(2 * nv * ss));
#pragma unroll
        for (int h = 0; h < C::NSB; ++h)
          dma_b16(r, slot + 2 * C::TB + C::AS * a + 256 * h, a < 2 ? dsk[h] : dsv[h], (uint32_t)(2 * r0 * ss));
      }
    }
  };
  if (nmine > 0) {
#pragma unroll
    for (int j = 0; j < C::SLOTS; ++j) issue(j);
  }

  // ---- query operand
  float inv2 = p.scale_log2;
  if constexpr (!C::DENSE) {
    float qmax = 0.0f;
#pragma unroll
    for (int j = 0; j < C::KSTEPS; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qmax = fmaxf(qmax, fmaxf(fabsf(to_float((uint16_t)(qop[j][i] & 0xffffu), T{})),
                                 fabsf(to_float((uint16_t)(qop[j][i] >> 16), T{}))));
    qmax = max_xor32(qmax);
    int e = 0;
    if (qmax > 0.0f) frexpf(qmax, &e);
    const int qe = 14 - e;  // |q| 2^qe < 2^14, exact
    const float qmul = ldexpf(1.0f, qe);
    inv2 = ldexpf(inv2, -qe);
#pragma unroll
    for (int j = 0; j < C::KSTEPS; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qop[j][i] = pack_f16x2(to_float((uint16_t)(qop[j][i] & 0xffffu), T{}) * qmul,
                               to_float((uint16_t)(qop[j][i] >> 16), T{}) * qmul);
    if constexpr (BITS == 4) {  // the dims in the order of dequant_nibbles
#pragma unroll
      for (int j = 0; j < C::KSTEPS; ++j) {
        const u4 q = qop[j];
        qop[j] = u4{perm(q[2], q[0], 0x05040100u), perm(q[2], q[0], 0x07060302u), perm(q[3], q[1], 0x05040100u),
                    perm(q[3], q[1], 0x07060302u)};
      }
    }
  }

  const int lo_all = p.window > 0 ? max(0, S_b - p.window) : 0;
  float m_run = -INFINITY, l_run = 0.0f;
  constexpr bool kRange = !C::DENSE && T::id == KVQ_DTYPE_BF16;  // values may leave the fp16 range
  int ev = 0;                   // V's exponent so far (uniform)
  float vmul = 1.0f, vback = 1.0f, vlimit = kHalfSafe;  // 2^-ev, 2^ev, 2^15 2^ev
  f16v oacc[C::DPL];
#pragma unroll
  for (int db = 0; db < C::DPL; ++db) oacc[db] = f16v{};
  uint32_t off_k[C::HC];
#pragma unroll
  for (int c = 0; c < C::HC; ++c) off_k[c] = (uint32_t)(n * C::ROWB + 16 * ((C::HC * hh + c) ^ C::swz(n)));
  constexpr int VB = C::DPL * BITS / 8;  // bytes of a lane's dims of a V row
  const uint32_t off_v = (uint32_t)(C::TB + 4 * hh * C::ROWB + n * VB);
  constexpr int KG = C::DENSE ? 1 : C::NG > 2 ? 2 : 1;  // scale groups of a lane's half row
  const int kg0 = C::DENSE ? 0 : hh * (D / 2) / G;
  const int vg = C::DENSE ? 0 : C::DPL * n / G;  // the group of the lane's V dims
  uint8_t* const tab = smem + C::RING + wave * C::TAB;

  for (int i = 0; i < nmine; ++i) {
    const uint8_t* sl = ring + (i % C::SLOTS) * C::SLOT;
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"((C::SLOTS - 1) * C::IPT) : "memory");  // tile i has landed
    // ---- the tile's operands into registers
    uint32_t kcell[2][KG] = {};
    float kmul = 1.0f, inv2t = inv2;
    if constexpr (!C::DENSE) {
      const uint32_t* cells = (const uint32_t*)(sl + 2 * C::TB);
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        kcell[0][g] = cells[32 * (kg0 + g) + n];
        kcell[1][g] = cells[C::AS / 4 + 32 * (kg0 + g) + n];
      }
      if constexpr (kRange) {
        float kb = 0.0f, vb = 0.0f;
#pragma unroll
        for (int g = 0; g < KG; ++g) kb = fmaxf(kb, group_bound<BITS>(kcell[0][g], kcell[1][g]));
#pragma unroll
        for (int h = 0; h < C::NSB; ++h) {
          const int c = 64 * h + (C::NG >= 2 ? 32 * hh : 0) + n;
          vb = fmaxf(vb, group_bound<BITS>(cells[2 * C::AS / 4 + c], cells[3 * C::AS / 4 + c]));
        }
        if (__builtin_amdgcn_ballot_w64(kb > kHalfSafe) != 0) {
          const int ek = bound_exponent(kb);
          kmul = ldexpf(1.0f, -ek);
          inv2t = ldexpf(inv2, ek);
        }
        if (__builtin_amdgcn_ballot_w64(vb > vlimit) != 0) {
          const int e = max(bound_exponent(vb), ev);
          const float f = ldexpf(1.0f, ev - e);
#pragma unroll
          for (int db = 0; db < C::DPL; ++db)
#pragma unroll
            for (int x = 0; x < 16; ++x) oacc[db][x] *= f;
          ev = e;
          vmul = ldexpf(1.0f, -ev);
          vback = ldexpf(1.0f, ev);
          vlimit = ldexpf(kHalfSafe, min(ev, 112));  // (past it every finite bound is within)
        }
      }
      // V's, converted once: lane -> group 2 h + hh of key n
#pragma unroll
      for (int h = 0; h < C::NSB; ++h) {
        if (C::NG >= 2 || hh == 0) {
          const int c = 64 * h + 32 * hh + n;
          const _Float16 s = operand_half<T>(cells[2 * C::AS / 4 + c], vmul), bi = operand_half<T>(cells[3 * C::AS / 4 + c], vmul);
          *(_Float16*)(tab + 2 * c) = s;
          *(_Float16*)(tab + 2 * (32 * C::NG + c)) = bi;
        }
      }
    }
    u4 kraw[C::HC];
#pragma unroll
    for (int c = 0; c < C::HC; ++c) kraw[c] = *(const u4*)(sl + off_k[c]);
    VRaw<VB> vraw[2][8];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) vraw[t][e].load(sl + off_v + (16 * t + 8 * (e >> 2) + (e & 3)) * C::ROWB);
    u2 vs[2][2], vb[2][2];  // scales and biases of the 8 keys of k-step t: keys 16 t + 4 hh .. + 3, and + 8
    if constexpr (!C::DENSE) {
      // (a wave's LDS operations keep their order; the compiler's must too, across the types)
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = 16 * t + 8 * h + 4 * hh;
          vs[t][h] = *(const u2*)(tab + 2 * (32 * vg + key));
          vb[t][h] = *(const u2*)(tab + 2 * (32 * (C::NG + vg) + key));
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot is free
    issue(i + C::SLOTS);

    // ---- scores
    f16v s = f16v{};
    {
      uint32_t ks2[KG], kb2[KG];
      if constexpr (!C::DENSE) {
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          const _Float16 a = operand_half<T>(kcell[0][g], kmul), c = operand_half<T>(kcell[1][g], kmul);
          ks2[g] = as_u32(h2{a, a});
          kb2[g] = as_u32(h2{c, c});
        }
      }
#pragma unroll
      for (int j = 0; j < C::KSTEPS; ++j) {
        u4 a;
        if constexpr (C::DENSE) {
          a = kraw[j];
        } else {
          const int g = KG == 2 ? (8 * j) / 32 : 0;
          if constexpr (BITS == 8) {
            const uint32_t w0 = kraw[j / 2][2 * (j % 2)], w1 = kraw[j / 2][2 * (j % 2) + 1];
            a = u4{dequant_bytes(w0, 0x04010400u, ks2[g], kb2[g]), dequant_bytes(w0, 0x04030402u, ks2[g], kb2[g]),
                   dequant_bytes(w1, 0x04010400u, ks2[g], kb2[g]), dequant_bytes(w1, 0x04030402u, ks2[g], kb2[g])};
          } else {
            uint32_t x[4];  // dims (0, 4), (1, 5), (2, 6), (3, 7)
            dequant_nibbles(kraw[j / 4][j % 4], ks2[g], kb2[g], x);
            a = u4{x[0], x[1], x[2], x[3]};
          }
        }
        s = mfma_32x32x16(a, qop[j], s, OT{});
      }
    }
    // value i: key k0 + 8 (i / 4) + 4 hh + i % 4
    const int k0 = ks.begin + kTile * (wave + kTW * i);
    if (!(k0 >= lo_all && k0 + kTile <= first)) {
      const uint32_t seen = node.keys(k0) >> (4 * hh);
      const int lo = lo_r - k0 - 4 * hh;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int c = 8 * (e >> 2) + (e & 3);
        if (c < lo || !((seen >> c) & 1u)) s[e] = -INFINITY;
      }
    }
    // ---- V^T operands of k-step t, block db (its row n is dim DPL n + db)
    u4 vop[2][C::DPL];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        if constexpr (BITS == 16) {
          const VRaw<VB>&x = vraw[t][2 * a], &y = vraw[t][2 * a + 1];
          if constexpr (C::DPL == 4) {
#pragma unroll
            for (int db = 0; db < 4; ++db)
              vop[t][db][a] = perm(y.w[db >> 1], x.w[db >> 1], (db & 1) ? 0x07060302u : 0x05040100u);
          } else {
            vop[t][0][a] = perm(y.w, x.w, 0x05040100u);
            vop[t][1][a] = perm(y.w, x.w, 0x07060302u);
          }
        } else {
          const uint32_t s2 = vs[t][a >> 1][a & 1], b2 = vb[t][a >> 1][a & 1], x = vraw[t][2 * a].w, y = vraw[t][2 * a + 1].w;
          if constexpr (BITS == 8) {  // two keys' codes of two dims as bytes: (x d0, y d0, x d1, y d1)
#pragma unroll
            for (int d = 0; d < C::DPL; d += 2) {
              const uint32_t xy = perm(y, x, d == 0 ? 0x05010400u : 0x07030602u);
              vop[t][d][a] = dequant_bytes(xy, 0x04010400u, s2, b2);
              vop[t][d + 1][a] = dequant_bytes(xy, 0x04030402u, s2, b2);
            }
          } else {  // DPL nibbles of each
            uint32_t v4[4];
            dequant_nibbles(x | (y << 16), s2, b2, v4);
#pragma unroll
            for (int d = 0; d < C::DPL; ++d) vop[t][d][a] = v4[d];
          }
        }
      }
    // ---- softmax, and O^T += V^T P^T
    float tm = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) tm = fmaxf(tm, s[e]);
    tm = max_xor32(tm) * inv2t;
    if (__builtin_amdgcn_ballot_w64(tm > m_run + kSlack) != 0) {
      const float m_new = tm > m_run + kSlack ? fmaxf(m_run, tm) : m_run;
      const float corr = m_new == m_run ? 1.0f : exp2_fast(m_run - m_new);
      l_run *= corr;
#pragma unroll
      for (int db = 0; db < C::DPL; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[db][e] *= corr;
      m_run = m_new;
    }
    const float nm = m_run == -INFINITY ? 0.0f : -m_run;
    u4 pop[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const float p0 = exp2_fast(fmaf(s[8 * t + 2 * a], inv2t, nm));
        const float p1 = exp2_fast(fmaf(s[8 * t + 2 * a + 1], inv2t, nm));
        pop[t][a] = pack2(p0, p1, OT{});
        l_run = add_pair(pop[t][a], l_run, OT{});
      }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int db = 0; db < C::DPL; ++db) oacc[db] = mfma_32x32x16(vop[t][db], pop[t], oacc[db], OT{});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load lands in the ring once it is used below
  // ---- merge the waves
  float* const w_o = (float*)smem;                   // [wave][row][ORow]
  float* const w_m = w_o + kTW * C::R * C::ORow;     // [wave][row]
  float* const w_l = w_m + kTW * C::R;
  __syncthreads();
  {
    const bool here = node.depth >= 0;  // an absent node sees nothing
    const float l_wave = add_xor32(l_run);
    const int at = wave * C::R + n;
    if (hh == 0) {
      w_m[at] = here ? m_run : -INFINITY;
      w_l[at] = here ? l_wave : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float* dst = w_o + at * C::ORow + C::DPL * (8 * (e >> 2) + 4 * hh + (e & 3));
      if constexpr (C::DPL == 4) {
        *(f4*)dst = f4{oacc[0][e] * vback, oacc[1][e] * vback, oacc[2][e] * vback, oacc[3][e] * vback};
      } else {
        *(float2*)dst = make_float2(oacc[0][e] * vback, oacc[1][e] * vback);
      }
    }
  }
  __syncthreads();
  constexpr int NPT = C::R * D / 4 / (kTW * 64);  // float4s of a partial per thread
  const bool single = p.nsplit == 1;
  auto out_row = [&](int rr) -> uint16_t* {
    const int rw = rb * C::R + rr;
    if (rw >= p.nrows) return nullptr;
    const int q = (int)div31((uint32_t)rw, p.d_l);
    return p.out + (int64_t)b * p.o_sb + (int64_t)(kvh * p.rep + q) * p.o_sh + (int64_t)(rw - q * p.L) * p.o_sl;
  };
  auto write_out = [&](uint16_t* dst, f4 o, float inv) {
    u2 w;
    w[0] = (uint32_t)from_float(o[0] * inv, T{}) | ((uint32_t)from_float(o[1] * inv, T{}) << 16);
    w[1] = (uint32_t)from_float(o[2] * inv, T{}) | ((uint32_t)from_float(o[3] * inv, T{}) << 16);
    *(u2*)dst = w;
  };
  const __amdgpu_buffer_rsrc_t ro = make_rsrc(p.part_o + (int64_t)unit * p.nsplit * (C::R * D), (uint32_t)(p.nsplit * C::R * D * 4));
  const __amdgpu_buffer_rsrc_t rm = make_rsrc(p.part_ml + (int64_t)unit * p.nsplit * (2 * C::R), (uint32_t)(p.nsplit * C::R * 8));
#pragma unroll
  for (int it = 0; it < NPT; ++it) {
    const int i4 = threadIdx.x + it * (kTW * 64), rr = 4 * i4 / D, d0 = 4 * i4 % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kTW; ++w) M = fmaxf(M, w_m[w * C::R + rr]);
    f4 o = {0, 0, 0, 0};
    float l = 0.0f;
    if (M != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kTW; ++w) {
        const float mw = w_m[w * C::R + rr];
        if (mw == -INFINITY) continue;
        const float f = exp2_fast(mw - M);
        o += f * *(const f4*)&w_o[(w * C::R + rr) * C::ORow + d0];
        l += f * w_l[w * C::R + rr];
      }
    }
    if (single) {
      uint16_t* dst = out_row(rr);
      if (dst) write_out(dst + d0, o, l > 0.0f ? 1.0f / l : 0.0f);
    } else if (p.fused) {
      store_agent_b128(ro, 16 * i4 + split * (C::R * D * 4), o);
      if (d0 == 0) store_agent_b64(rm, 8 * rr + split * (C::R * 8), make_float2(M, l));
    } else {
      const int64_t pi = ((int64_t)unit * p.nsplit + split) * C::R + rr;
      *(f4*)(p.part_o + pi * D + d0) = o;
      if (d0 == 0) ((float2*)p.part_ml)[pi] = make_float2(M, l);
    }
  }
  if (single || !p.fused) return;

  // ---- few splits: the last of the unit to finish merges them (decode_kernel.h says why this order is enough)
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) s_prev = __hip_atomic_fetch_add(&p.counters[unit], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_prev != (unsigned)(p.nsplit - 1)) return;
  if (threadIdx.x == 0) __hip_atomic_store(&p.counters[unit], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const int last_split = p.nsplit - 1;
#pragma unroll
  for (int it = 0; it < NPT; ++it) {
    const int i4 = threadIdx.x + it * (kTW * 64), rr = 4 * i4 / D, d0 = 4 * i4 % D;
    f4 po[kFewSplits];
    float2 mv[kFewSplits];
#pragma unroll
    for (int u = 0; u < kFewSplits; ++u) {
      const int su = min(u, last_split);
      po[u] = load_agent_b128(ro, 16 * i4, su * (C::R * D * 4));
      mv[u] = load_agent_b64(rm, 8 * rr, su * (C::R * 8));
    }
    float M = -INFINITY;
#pragma unroll
    for (int u = 0; u < kFewSplits; ++u)
      if (u <= last_split && mv[u].y > 0.0f) M = fmaxf(M, mv[u].x);
    f4 acc = {0, 0, 0, 0};
    float l = 0.0f;
#pragma unroll
    for (int u = 0; u < kFewSplits; ++u) {
      const float w = (u <= last_split && mv[u].y > 0.0f) ? exp2_fast(mv[u].x - M) : 0.0f;
      acc += w * po[u];
      l += w * mv[u].y;
    }
    uint16_t* dst = out_row(rr);
    if (dst) write_out(dst + d0, acc, l > 0.0f ? 1.0f / l : 0.0f);
  }
}

}  // namespace kvq
