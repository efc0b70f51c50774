// C ABI of libkvq.so: argument validation, error reporting, dispatch to the kernel launchers.
// Every check runs on the host before any HIP call, so a rejected call touches no device state.

#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>

#include <mutex>

#include "launch.h"
#include "merge.h"

// Scratch of kvq_decode_attn_static: device memory the library owns, one copy per GPU, held until
// the process ends. In host code `scratch` is a host-side stand-in for the symbol, not a device
// address: the kernels get the per-device address hipGetSymbolAddress returns (static_scratch
// below), never the name.
static __device__ __align__(256) uint8_t scratch[KVQ_STATIC_SCRATCH_BYTES];

// Zero `n` words (the scratch's arrival counters, once per device). A kernel rather than
// hipMemsetAsync, so that a caller may capture the first call into a HIP graph.
__global__ void zero_words_kernel(uint32_t* p, size_t n) {
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) p[i] = 0u;
}

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int ok() {
  g_err[0] = '\0';
  return KVQ_OK;
}

int hip_status(hipError_t e, const char* what) {
  if (e == hipSuccess) return ok();
  return fail(KVQ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p % a) == 0; }

int check_dtype(int dtype) {
  if (dtype != KVQ_DTYPE_F16 && dtype != KVQ_DTYPE_BF16) return fail(KVQ_ERR_INVALID, "dtype %d is not f16 (0) or bf16 (1)", dtype);
  return KVQ_OK;
}

int check_qtensor(const kvq_qtensor* t, const char* name) {
  if (!t) return fail(KVQ_ERR_INVALID, "%s descriptor is NULL", name);
  if (!t->codes || !t->scales || !t->biases) return fail(KVQ_ERR_INVALID, "%s has a NULL codes/scales/biases pointer", name);
  if (t->codes_stride_b < 0 || t->codes_stride_h < 0 || t->codes_stride_s <= 0 || t->sb_stride_b < 0 ||
      t->sb_stride_h < 0 || t->sb_stride_s <= 0)
    return fail(KVQ_ERR_INVALID, "%s has a negative or zero stride", name);
  if (!aligned(t->scales, 2) || !aligned(t->biases, 2)) return fail(KVQ_ERR_INVALID, "%s scales/biases are not 2-byte aligned", name);
  return KVQ_OK;
}

int check_rows(const kvq_rows* r, const char* name, int D, bool vec16) {
  if (!r || !r->data) return fail(KVQ_ERR_INVALID, "%s is NULL", name);
  if (r->stride_b < 0 || r->stride_h < 0 || r->stride_l < 0) return fail(KVQ_ERR_INVALID, "%s has a negative stride", name);
  if (vec16) {
    if (!aligned(r->data, 16) || r->stride_b % 8 || r->stride_h % 8 || r->stride_l % 8 || D % 8)
      return fail(KVQ_ERR_INVALID, "%s must be 16-byte aligned with strides that are multiples of 8 elements", name);
  } else if (!aligned(r->data, 2)) {
    return fail(KVQ_ERR_INVALID, "%s is not 2-byte aligned", name);
  }
  return KVQ_OK;
}

// Rows that are rotated in place or written out have an address of their own each: of a broadcast tensor the result
// would depend on the order of the workgroups.
int check_own_rows(const kvq_rows* r, const char* name, int B, int H, int L) {
  if ((B > 1 && !r->stride_b) || (H > 1 && !r->stride_h) || (L > 1 && !r->stride_l))
    return fail(KVQ_ERR_INVALID, "%s is written: its rows must not share their memory (a stride is 0)", name);
  return KVQ_OK;
}

// The index of the first array whose address an earlier one has, or -1 (-2: no memory for the look). A hash table of
// addresses, half full at most: a call with 192 arrays takes 8.3 us with it and without.
int repeated_array(const kvq_row_array* arrays, int n) {
  constexpr size_t kSmall = 512;
  uintptr_t small[kSmall] = {};
  size_t slots = kSmall;
  while (slots < 2 * (size_t)n) slots *= 2;
  uintptr_t* big = slots > kSmall ? (uintptr_t*)calloc(slots, sizeof(uintptr_t)) : nullptr;
  if (slots > kSmall && !big) return -2;
  uintptr_t* table = big ? big : small;
  int found = -1;
  for (int i = 0; i < n && found < 0; ++i) {
    const uintptr_t p = (uintptr_t)arrays[i].data;
    size_t at = (size_t)(((uint64_t)p * 0x9E3779B97F4A7C15ull) >> 32) & (slots - 1);  // (the golden ratio's multiplicative hash)
    while (table[at] && table[at] != p) at = (at + 1) & (slots - 1);
    if (table[at]) found = i;
    table[at] = p;
  }
  free(big);
  return found;
}

// Shared checks of the attention entry points (shape, dtype, scale, window, queries, output).
int check_attn_common(const kvq_rows* q, const kvq_rows* out, int B, int Hq, int Hkv, int L, int D, int S, int dtype,
                      float scale, int window) {
  int rc;
  if ((rc = check_dtype(dtype))) return rc;
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || L <= 0 || S <= 0) return fail(KVQ_ERR_INVALID, "B, Hq, Hkv, L and S must be positive (got %d, %d, %d, %d, %d)", B, Hq, Hkv, L, S);
  if (Hq % Hkv) return fail(KVQ_ERR_INVALID, "Hq=%d is not a multiple of Hkv=%d", Hq, Hkv);
  if (window < 0) return fail(KVQ_ERR_INVALID, "window must be >= 0, got %d", window);
  if (!isfinite(scale)) return fail(KVQ_ERR_INVALID, "scale is not finite");
  if ((rc = check_rows(q, "queries", D, true))) return rc;
  if ((rc = check_rows(out, "out", D, false))) return rc;
  // every attention kernel writes 4 output elements (8 bytes) at a time
  if (!aligned(out->data, 8) || out->stride_b % 4 || out->stride_h % 4 || out->stride_l % 4)
    return fail(KVQ_ERR_INVALID, "out must be 8-byte aligned with strides that are multiples of 4 elements");
  return KVQ_OK;
}

// Head dimensions 64, 128 and 256 have kernels of their own width; any other multiple of 8 up to 256
// runs at the next width (kvq::decode_kernel_dim), for every query length: on the decode kernel, or
// for unquantized rows past 128 dims on the head_dim-256 kernel. Quantized rows of 96 dims have a
// prefill kernel too (prefill_serves_96).
bool native_dim(int D) { return D == 64 || D == 128 || D == 256; }

int check_head_dim(int D, const char* what) {
  if (D > 0 && D % 8 == 0 && D <= 256) return KVQ_OK;
  return fail(KVQ_ERR_UNSUPPORTED, "%s supports head_dim 64, 128, 256 and other multiples of 8 up to 256, got %d", what,
              D);
}

int check_workspace(size_t ws_needed, void* workspace, size_t workspace_bytes) {
  if (!workspace || workspace_bytes < ws_needed)
    return fail(KVQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", ws_needed, workspace ? workspace_bytes : (size_t)0);
  if (!aligned(workspace, 256)) return fail(KVQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  return KVQ_OK;
}

// Scale-group sizes the attention kernels are built for: 32, 64 and 128, at most the kernel width and
// at least a quarter of it (a decode lane's quarter of a row lies in one group), dividing D.
int check_attn_group(int group_size, int D) {
  const int Dk = kvq::decode_kernel_dim(D);
  if ((group_size != 32 && group_size != 64 && group_size != 128) || group_size > Dk || 4 * group_size < Dk ||
      D % group_size)
    return fail(KVQ_ERR_UNSUPPORTED,
                "attention supports group_size 32, 64 and 128 dividing head_dim (%d) and between %d/4 and %d, got %d",
                D, Dk, Dk, group_size);
  return KVQ_OK;
}

// Everything check_attn checks but the workspace.
int check_attn_args(const kvq_rows* q, const kvq_qtensor* k, const kvq_qtensor* v, const kvq_rows* out, int B, int Hq,
                    int Hkv, int L, int D, int S, int bits, int group_size, int dtype, float scale, int window) {
  int rc;
  if ((rc = check_attn_common(q, out, B, Hq, Hkv, L, D, S, dtype, scale, window))) return rc;
  if (bits != 4 && bits != 8) return fail(KVQ_ERR_UNSUPPORTED, "attention supports 4- and 8-bit caches, got bits=%d", bits);
  if ((rc = check_attn_group(group_size, D))) return rc;
  if ((rc = check_qtensor(k, "keys"))) return rc;
  if ((rc = check_qtensor(v, "values"))) return rc;
  const int64_t row_words = (int64_t)D * bits / 32;
  for (const kvq_qtensor* t : {k, v}) {
    if (!aligned(t->codes, 16) || (t->codes_stride_s * 4) % 16 || (t->codes_stride_h * 4) % 16 || (t->codes_stride_b * 4) % 16)
      return fail(KVQ_ERR_INVALID, "codes must be 16-byte aligned with 16-byte-multiple row, head and batch strides");
    if (t->codes_stride_s < row_words) return fail(KVQ_ERR_INVALID, "codes row stride %lld is smaller than D*bits/32=%lld", (long long)t->codes_stride_s, (long long)row_words);
    if (t->sb_stride_s < D / group_size)
      return fail(KVQ_ERR_INVALID, "scales row stride %lld is smaller than D/group=%d", (long long)t->sb_stride_s, D / group_size);
    // a row narrower than its kernel reads the next row's first groups past its own: they must be
    // rows of the cache, not padding
    if (D < kvq::decode_kernel_dim(D) && t->sb_stride_s != D / group_size)
      return fail(KVQ_ERR_UNSUPPORTED, "head_dim %d needs scale and bias rows of exactly D/group=%d elements, got a stride "
                  "of %lld", D, D / group_size, (long long)t->sb_stride_s);
    // the kernels address each (sequence, KV head)'s rows with 32-bit byte offsets
    if ((int64_t)S * t->codes_stride_s * 4 > (int64_t)UINT32_MAX || (int64_t)S * t->sb_stride_s * 2 > (int64_t)UINT32_MAX)
      return fail(KVQ_ERR_UNSUPPORTED, "attention needs S times each row stride within 4 GiB (S=%d)", S);
  }
  return KVQ_OK;
}

int check_attn(const kvq_rows* q, const kvq_qtensor* k, const kvq_qtensor* v, const kvq_rows* out, int B, int Hq,
               int Hkv, int L, int D, int S, int bits, int group_size, int dtype, float scale, int window,
               size_t ws_needed, void* workspace, size_t workspace_bytes) {
  int rc;
  if ((rc = check_attn_args(q, k, v, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale, window))) return rc;
  return check_workspace(ws_needed, workspace, workspace_bytes);
}

// Attention over an unquantized cache: K and V are strided T rows like the queries.
int check_attn_dense(const kvq_rows* q, const kvq_rows* k, const kvq_rows* v, const kvq_rows* out, int B, int Hq,
                     int Hkv, int L, int D, int S, int dtype, float scale, int window, size_t ws_needed,
                     void* workspace, size_t workspace_bytes) {
  int rc;
  if ((rc = check_attn_common(q, out, B, Hq, Hkv, L, D, S, dtype, scale, window))) return rc;
  if ((rc = check_rows(k, "keys", D, true))) return rc;
  if ((rc = check_rows(v, "values", D, true))) return rc;
  // a key row narrower than its kernel reads the next row's first elements past its own: they must
  // be a row of the cache, not padding
  if (D < kvq::decode_kernel_dim(D) && k->stride_l != D)
    return fail(KVQ_ERR_UNSUPPORTED, "head_dim %d needs key rows of exactly D elements, got a stride of %lld", D,
                (long long)k->stride_l);
  for (const kvq_rows* t : {k, v}) {
    if (t->stride_l < D) return fail(KVQ_ERR_INVALID, "K/V row stride %lld is smaller than D=%d", (long long)t->stride_l, D);
    // the kernels address each (sequence, KV head)'s rows with 32-bit byte offsets
    if ((int64_t)S * t->stride_l * 2 > (int64_t)UINT32_MAX)
      return fail(KVQ_ERR_UNSUPPORTED, "attention needs S times the K/V row stride within 4 GiB (S=%d)", S);
  }
  return check_workspace(ws_needed, workspace, workspace_bytes);
}

int check_quantize(const kvq_rows* k_src, const kvq_qtensor* k_dst, const kvq_rows* v_src, const kvq_qtensor* v_dst,
                   int64_t row_offset, int B, int H, int L, int D, int bits, int group_size, int dtype, bool read = false) {
  int rc;
  if ((rc = check_dtype(dtype))) return rc;
  if (bits != 2 && bits != 4 && bits != 8) return fail(KVQ_ERR_UNSUPPORTED, "bits must be 2, 4 or 8, got %d", bits);
  if (group_size != 32 && group_size != 64 && group_size != 128)
    return fail(KVQ_ERR_UNSUPPORTED, "group_size must be 32, 64 or 128, got %d", group_size);
  if (B < 0 || H < 0 || L < 0 || D <= 0) return fail(KVQ_ERR_INVALID, "negative shape (B=%d H=%d L=%d D=%d)", B, H, L, D);
  if (D % group_size) return fail(KVQ_ERR_INVALID, "D=%d is not a multiple of group_size=%d", D, group_size);
  if (row_offset < 0) return fail(KVQ_ERR_INVALID, "row_offset must be >= 0");
  // (reading back, the rows are the destination)
  const char *kr = read ? "k_dst" : "k_src", *kq = read ? "k_src" : "k_dst", *vr = read ? "v_dst" : "v_src", *vq = read ? "v_src" : "v_dst";
  if ((v_src == nullptr) != (v_dst == nullptr)) return fail(KVQ_ERR_INVALID, "v_src and v_dst must both be given or both be NULL");
  if ((rc = check_rows(k_src, kr, D, true))) return rc;
  if ((rc = check_qtensor(k_dst, kq))) return rc;
  if (v_src) {
    if ((rc = check_rows(v_src, vr, D, true))) return rc;
    if ((rc = check_qtensor(v_dst, vq))) return rc;
  }
  if (read && (rc = check_own_rows(k_src, kr, B, H, L))) return rc;
  if (read && v_src && (rc = check_own_rows(v_src, vr, B, H, L))) return rc;
  const int64_t row_words = (int64_t)D * bits / 32;
  for (const kvq_qtensor* t : {k_dst, v_dst}) {
    if (!t) continue;
    if (t->codes_stride_s < row_words) return fail(KVQ_ERR_INVALID, "codes row stride is smaller than D*bits/32");
    if (bits == 8 && (!aligned(t->codes, 8) || t->codes_stride_s % 2 || t->codes_stride_h % 2 || t->codes_stride_b % 2))
      return fail(KVQ_ERR_INVALID, "8-bit codes must be 8-byte aligned with even word strides");
    if (t->sb_stride_s < D / group_size) return fail(KVQ_ERR_INVALID, "scales row stride is smaller than D/group_size");
  }
  return KVQ_OK;
}

// A paged pool described by a kvq_qtensor whose batch strides are page strides: pages of
// KVQ_PAGE_ROWS rows per head, head-major within a page.
int check_pool(const kvq_qtensor* t, const char* name, int H, int D, int bits, int group_size, int num_pages) {
  int rc;
  if ((rc = check_qtensor(t, name))) return rc;
  if (num_pages <= 0) return fail(KVQ_ERR_INVALID, "num_pages must be positive, got %d", num_pages);
  const int64_t row_words = (int64_t)D * bits / 32, groups = D / group_size;
  if (t->codes_stride_s < row_words || t->sb_stride_s < groups)
    return fail(KVQ_ERR_INVALID, "%s row strides are smaller than one row", name);
  if (D < kvq::decode_kernel_dim(D) && t->sb_stride_s != groups)
    return fail(KVQ_ERR_UNSUPPORTED, "head_dim %d needs %s scale and bias rows of exactly D/group=%lld elements", D, name,
                (long long)groups);
  if (t->codes_stride_h < KVQ_PAGE_ROWS * t->codes_stride_s || t->sb_stride_h < KVQ_PAGE_ROWS * t->sb_stride_s ||
      t->codes_stride_b < H * t->codes_stride_h || t->sb_stride_b < H * t->sb_stride_h)
    return fail(KVQ_ERR_INVALID, "%s is not [num_pages][H][%d][row]: its strides overlap", name, KVQ_PAGE_ROWS);
  return KVQ_OK;
}

int check_table(const int32_t* table, int64_t table_stride, int64_t rows_needed) {
  if (!table) return fail(KVQ_ERR_INVALID, "block_table is NULL");
  if (table_stride <= 0) return fail(KVQ_ERR_INVALID, "table_stride must be positive");
  if ((rows_needed + KVQ_PAGE_ROWS - 1) / KVQ_PAGE_ROWS > table_stride)
    return fail(KVQ_ERR_INVALID, "table_stride %lld pages cannot hold %lld rows", (long long)table_stride,
                (long long)rows_needed);
  return KVQ_OK;
}

// The address of this device's copy of `scratch`, looked up once per device (with the device
// current) by hipGetSymbolAddress; the first call on a device also zeroes its arrival counters on
// `stream` (every later call leaves them at zero).
constexpr int kMaxDevices = 64;
struct ScratchSlot {
  std::once_flag once;
  void* ptr = nullptr;
  hipError_t err = hipSuccess;
};
ScratchSlot g_scratch[kMaxDevices];

int static_scratch(hipStream_t stream, void** out) {
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return hip_status(e, "hipGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(KVQ_ERR_UNSUPPORTED, "device %d is beyond the %d the library tracks", dev, kMaxDevices);
  ScratchSlot& s = g_scratch[dev];
  std::call_once(s.once, [&] {
    void* p = nullptr;
    s.err = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (s.err != hipSuccess) return;
    const size_t words = kvq::kCounterBytes / 4;
    hipLaunchKernelGGL(zero_words_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, stream, (uint32_t*)p, words);
    s.err = hipGetLastError();
    if (s.err == hipSuccess) s.ptr = p;
  });
  if (!s.ptr) return hip_status(s.err != hipSuccess ? s.err : hipErrorInvalidSymbol, "static scratch set-up");
  *out = s.ptr;
  return KVQ_OK;
}

int check_rope(const kvq_rope_params* r, int D) {
  if (!r) return fail(KVQ_ERR_INVALID, "rope descriptor is NULL");
  if (r->dims <= 0 || r->dims > D || r->dims > 256 || r->dims % 16)
    return fail(KVQ_ERR_UNSUPPORTED, "rope dims must be a positive multiple of 16, at most D=%d and 256, got %d", D,
                r->dims);
  if (!(r->base > 0.0f) || !isfinite(r->base)) return fail(KVQ_ERR_INVALID, "rope base must be positive and finite");
  if (!isfinite(r->scale)) return fail(KVQ_ERR_INVALID, "rope scale is not finite");
  if (r->offset < 0) return fail(KVQ_ERR_INVALID, "rope offset must be >= 0");
  return KVQ_OK;
}

int check_axes(const kvq_axes* r, int D) {
  if (!r) return fail(KVQ_ERR_INVALID, "rope descriptor is NULL");
  if (r->dims <= 0 || r->dims > D || r->dims > 256 || r->dims % 16)
    return fail(KVQ_ERR_UNSUPPORTED, "rope dims must be a positive multiple of 16, at most D=%d and 256, got %d", D,
                r->dims);
  if (r->axes < 1 || r->axes > KVQ_MAX_AXES)
    return fail(KVQ_ERR_UNSUPPORTED, "rope needs 1 to %d position axes, got %d", KVQ_MAX_AXES, r->axes);
  int64_t pairs = 0;
  for (int a = 0; a < r->axes; ++a) {
    if (r->sections[a] < 1) return fail(KVQ_ERR_INVALID, "rope section %d has %d pairs: at least 1 is needed", a, r->sections[a]);
    pairs += r->sections[a];
  }
  if (pairs != r->dims / 2)
    return fail(KVQ_ERR_INVALID, "rope sections hold %lld pairs, dims %d have %d", (long long)pairs, r->dims, r->dims / 2);
  if (!(r->base > 0.0) || !isfinite(r->base)) return fail(KVQ_ERR_INVALID, "rope base must be positive and finite");
  if (!isfinite(r->scale)) return fail(KVQ_ERR_INVALID, "rope scale is not finite");
  if (!r->positions) return fail(KVQ_ERR_INVALID, "rope positions are NULL");
  if (!aligned(r->positions, 4) || r->pos_stride_a < 0 || r->pos_stride_b < 0 || r->pos_stride_l < 0)
    return fail(KVQ_ERR_INVALID, "rope positions must be 4-byte aligned with non-negative strides");
  return KVQ_OK;
}

}  // namespace

extern "C" {

int kvq_abi_version(void) { return KVQ_ABI_VERSION; }

const char* kvq_last_error(void) { return g_err; }

int kvq_quantize_append(const kvq_rows* k_src, const kvq_qtensor* k_dst, const kvq_rows* v_src,
                        const kvq_qtensor* v_dst, int64_t row_offset, int B, int H, int L, int D, int bits,
                        int group_size, int dtype, void* stream) {
  int rc;
  if ((rc = check_quantize(k_src, k_dst, v_src, v_dst, row_offset, B, H, L, D, bits, group_size, dtype))) return rc;
  if (B == 0 || H == 0 || L == 0) return ok();
  return hip_status(kvq::launch_quantize_append(k_src, k_dst, v_src, v_dst, nullptr, row_offset, B, H, L, D, bits,
                                                group_size, dtype, (hipStream_t)stream),
                    "quantize_append launch");
}

int kvq_rope(const kvq_rows* x, const kvq_rope_params* rope, int B, int H, int L, int D, int dtype, void* stream) {
  int rc;
  if ((rc = check_dtype(dtype))) return rc;
  if (B < 0 || H < 0 || L < 0 || D <= 0 || D % 8) return fail(KVQ_ERR_INVALID, "bad shape (B=%d H=%d L=%d D=%d)", B, H, L, D);
  if ((rc = check_rope(rope, D))) return rc;
  if ((rc = check_rows(x, "x", D, true))) return rc;
  if (B == 0 || H == 0 || L == 0) return ok();
  return hip_status(kvq::launch_rope(x, rope, B, H, L, dtype, (hipStream_t)stream), "rope launch");
}

int kvq_rope_quantize_append(const kvq_rows* k_src, const kvq_qtensor* k_dst, const kvq_rows* v_src,
                             const kvq_qtensor* v_dst, const kvq_rope_params* rope, int64_t row_offset, int B, int H, int L,
                             int D, int bits, int group_size, int dtype, void* stream) {
  int rc;
  if ((rc = check_rope(rope, D))) return rc;
  if ((rc = check_quantize(k_src, k_dst, v_src, v_dst, row_offset, B, H, L, D, bits, group_size, dtype))) return rc;
  if (B == 0 || H == 0 || L == 0) return ok();
  return hip_status(kvq::launch_quantize_append(k_src, k_dst, v_src, v_dst, rope, row_offset, B, H, L, D, bits,
                                                group_size, dtype, (hipStream_t)stream),
                    "rope_quantize_append launch");
}

int kvq_paged_quantize_append(const kvq_rows* k_src, const kvq_qtensor* k_pool, const kvq_rows* v_src,
                              const kvq_qtensor* v_pool, int num_pages, const int32_t* block_table,
                              int64_t table_stride, const int32_t* starts, int64_t row_offset,
                              const kvq_rope_params* rope, int B, int H, int L, int D, int bits, int group_size,
                              int dtype, void* stream) {
  int rc;
  if ((rc = check_quantize(k_src, k_pool, v_src, v_pool, row_offset, B, H, L, D, bits, group_size, dtype))) return rc;
  if ((rc = check_pool(k_pool, "k_pool", H, D, bits, group_size, num_pages))) return rc;
  if (v_pool && (rc = check_pool(v_pool, "v_pool", H, D, bits, group_size, num_pages))) return rc;
  if ((rc = check_table(block_table, table_stride, starts ? 1 : row_offset + L))) return rc;
  if (rope && (rc = check_rope(rope, D))) return rc;
  if (B == 0 || H == 0 || L == 0) return ok();
  return hip_status(kvq::launch_paged_quantize_append(k_src, k_pool, v_src, v_pool, num_pages, block_table, table_stride,
                                                      starts, row_offset, rope, B, H, L, D, bits, group_size, dtype,
                                                      (hipStream_t)stream),
                    "paged_quantize_append launch");
}

int kvq_rope_axes(const kvq_rows* x, const kvq_axes* rope, int B, int H, int L, int D, int dtype, void* stream) {
  int rc;
  if ((rc = check_dtype(dtype))) return rc;
  if (B < 0 || H < 0 || L < 0 || D <= 0 || D % 8) return fail(KVQ_ERR_INVALID, "bad shape (B=%d H=%d L=%d D=%d)", B, H, L, D);
  if ((rc = check_axes(rope, D))) return rc;
  if ((rc = check_rows(x, "x", D, true))) return rc;
  if ((rc = check_own_rows(x, "x", B, H, L))) return rc;
  if (B == 0 || H == 0 || L == 0) return ok();
  return hip_status(kvq::launch_rope_axes(x, rope, B, H, L, dtype, (hipStream_t)stream), "rope_axes launch");
}

int kvq_rope_axes_append(const kvq_rows* k_src, const kvq_qtensor* k_dst, const kvq_rows* v_src, const kvq_qtensor* v_dst,
                         const kvq_rows* q, int Hq, const kvq_axes* rope, int num_pages, const int32_t* block_table,
                         int64_t table_stride, const int32_t* starts, int64_t row_offset, int B, int H, int L, int D,
                         int bits, int group_size, int dtype, void* stream) {
  int rc;
  if ((rc = check_axes(rope, D))) return rc;
  if ((rc = check_quantize(k_src, k_dst, v_src, v_dst, row_offset, B, H, L, D, bits, group_size, dtype))) return rc;
  if (q) {
    if (Hq < 0) return fail(KVQ_ERR_INVALID, "negative shape (Hq=%d)", Hq);
    if ((rc = check_rows(q, "queries", D, true))) return rc;
    if ((rc = check_own_rows(q, "queries", B, Hq, L))) return rc;
  }
  if (block_table) {
    if ((rc = check_pool(k_dst, "k_pool", H, D, bits, group_size, num_pages))) return rc;
    if (v_dst && (rc = check_pool(v_dst, "v_pool", H, D, bits, group_size, num_pages))) return rc;
    if ((rc = check_table(block_table, table_stride, starts ? 1 : row_offset + L))) return rc;
  } else if (starts) {
    return fail(KVQ_ERR_INVALID, "starts need a block table");
  }
  if (B == 0 || L == 0 || H == 0) return ok();
  return hip_status(kvq::launch_rope_axes_append(k_src, k_dst, v_src, v_dst, Hq > 0 ? q : nullptr, Hq, rope, num_pages,
                                                 block_table, table_stride, starts, row_offset, B, H, L, D, bits, group_size,
                                                 dtype, (hipStream_t)stream),
                    "rope_axes_append launch");
}

int kvq_dequantize(const kvq_qtensor* k_src, const kvq_rows* k_dst, const kvq_qtensor* v_src, const kvq_rows* v_dst,
                   int64_t row_offset, int B, int H, int L, int D, int bits, int group_size, int dtype, void* stream) {
  int rc;
  if ((rc = check_quantize(k_dst, k_src, v_dst, v_src, row_offset, B, H, L, D, bits, group_size, dtype, true))) return rc;
  if (B == 0 || H == 0 || L == 0) return ok();
  return hip_status(kvq::launch_dequantize(k_src, k_dst, v_src, v_dst, 0, nullptr, 0, nullptr, row_offset, B, H, L, D, bits,
                                           group_size, dtype, (hipStream_t)stream),
                    "dequantize launch");
}

int kvq_paged_dequantize(const kvq_qtensor* k_pool, const kvq_rows* k_dst, const kvq_qtensor* v_pool, const kvq_rows* v_dst,
                         int num_pages, const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens, int B,
                         int H, int L, int D, int bits, int group_size, int dtype, void* stream) {
  int rc;
  if ((rc = check_quantize(k_dst, k_pool, v_dst, v_pool, 0, B, H, L, D, bits, group_size, dtype, true))) return rc;
  if ((rc = check_pool(k_pool, "k_pool", H, D, bits, group_size, num_pages))) return rc;
  if (v_pool && (rc = check_pool(v_pool, "v_pool", H, D, bits, group_size, num_pages))) return rc;
  if ((rc = check_table(block_table, table_stride, L))) return rc;
  if (!seq_lens) return fail(KVQ_ERR_INVALID, "seq_lens is NULL");
  if (B == 0 || H == 0 || L == 0) return ok();
  return hip_status(kvq::launch_dequantize(k_pool, k_dst, v_pool, v_dst, num_pages, block_table, table_stride, seq_lens, 0, B,
                                           H, L, D, bits, group_size, dtype, (hipStream_t)stream),
                    "paged_dequantize launch");
}

int kvq_keep_rows(const kvq_row_array* arrays, int n_arrays, int num_pages, const int32_t* block_table, int64_t table_stride,
                  const int32_t* rows, int64_t rows_stride_b, const int32_t* starts, int64_t start, int n, int M, int B,
                  int H, void* stream) {
  if (n_arrays < 0 || n < 0 || M < 0 || B < 0 || H < 0)
    return fail(KVQ_ERR_INVALID, "negative shape (arrays=%d n=%d M=%d B=%d H=%d)", n_arrays, n, M, B, H);
  if (M > n) return fail(KVQ_ERR_INVALID, "%d rows cannot be kept of %d", M, n);
  if (B > 65535) return fail(KVQ_ERR_UNSUPPORTED, "a batch of at most 65535, got %d", B);
  if (n_arrays > 0 && !arrays) return fail(KVQ_ERR_INVALID, "arrays is NULL");
  if (!rows || !aligned(rows, 4) || !aligned(starts, 4) || rows_stride_b < 0)
    return fail(KVQ_ERR_INVALID, "rows must not be NULL, rows and starts 4-byte aligned, with a non-negative batch stride");
  if (start < 0) return fail(KVQ_ERR_INVALID, "start must be >= 0");
  if (block_table) {
    if (!aligned(block_table, 4) || table_stride <= 0 || num_pages <= 0)
      return fail(KVQ_ERR_INVALID, "block_table must be 4-byte aligned, table_stride and num_pages positive");
  } else if (starts) {
    return fail(KVQ_ERR_INVALID, "starts need a block table");
  }
  for (int i = 0; i < n_arrays; ++i) {
    const kvq_row_array& a = arrays[i];
    if (!a.data) return fail(KVQ_ERR_INVALID, "array %d has a NULL pointer", i);
    if (a.stride_b < 0 || a.stride_h < 0 || a.stride_l <= 0 || a.row_bytes <= 0)
      return fail(KVQ_ERR_INVALID, "array %d has a negative or zero stride or width", i);
    if (!aligned(a.data, 2) || (a.stride_b | a.stride_h | a.stride_l | a.row_bytes) & 1)
      return fail(KVQ_ERR_INVALID, "array %d has an odd address, stride or width", i);
    if (a.stride_l < a.row_bytes || a.row_bytes > 65536)
      return fail(KVQ_ERR_INVALID, "array %d: rows of %lld bytes every %lld", i, (long long)a.row_bytes, (long long)a.stride_l);
    if (((block_table ? num_pages : B) > 1 && !a.stride_b) || (H > 1 && !a.stride_h))
      return fail(KVQ_ERR_INVALID, "array %d is broadcast: its rows share their memory", i);
  }
  const int twice = repeated_array(arrays, n_arrays);
  if (twice >= 0) return fail(KVQ_ERR_INVALID, "array %d is named twice: its rows would move twice", twice);
  if (twice != -1) return fail(KVQ_ERR_INVALID, "out of host memory for %d arrays", n_arrays);
  if (n_arrays == 0 || M == 0 || B == 0 || H == 0) return ok();
  return hip_status(kvq::launch_keep_rows(arrays, n_arrays, num_pages, block_table, table_stride, rows, rows_stride_b, starts,
                                          start, n, M, B, H, (hipStream_t)stream),
                    "keep_rows launch");
}

size_t kvq_decode_workspace_size(int B, int Hq, int Hkv, int L, int D, int S, int window) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || L <= 0 || S <= 0 || D <= 0 || D > 256 || D % 8 || window < 0) return 0;
  // one size serves every cache format: the quantized (8-, 4-bit) and the unquantized (16) plans
  // and every scale-group size (the group sets the query rows per workgroup)
  const int Dk = kvq::decode_kernel_dim(D);
  size_t n = 0;
  for (int bits : {8, 16})  // (4 bits plan as 8 do; every unquantized plan is that of group 64)
    for (int G : {32, 64, 128}) {
      if (G > Dk || 4 * G < Dk || (bits == 16 && (Dk > 128 || G != 64))) continue;
      const size_t x = kvq::decode_workspace_bytes(B, Hq, Hkv, L, D, S, window, bits, G);
      n = x > n ? x : n;
    }
  if (window == 0 && Hq % Hkv == 0) {  // calls under a general mask may run on the prefill kernel
    const size_t x = kvq::prefill_masked_bytes(B, Hq, Hkv, L, D, S);
    n = x > n ? x : n;
  }
  if (Dk == 256) {  // unquantized rows past 128 dims run through the head_dim-256 kernel
    const size_t x = kvq::wide_workspace_bytes(B, Hq, Hkv, L, Dk, S, window);
    n = x > n ? x : n;
  }
  return n;
}

int kvq_decode_attn(const kvq_rows* q, const kvq_qtensor* k, const kvq_qtensor* v, const int32_t* seq_lens,
                    const kvq_rows* out, int B, int Hq, int Hkv, int L, int D, int S, int bits, int group_size,
                    int dtype, float scale, int causal, int window, void* workspace, size_t workspace_bytes,
                    void* stream) {
  if (check_head_dim(D, "decode")) return KVQ_ERR_UNSUPPORTED;
  int rc = check_attn(q, k, v, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale, window,
                      kvq_decode_workspace_size(B, Hq, Hkv, L, D, S, window), workspace, workspace_bytes);
  if (rc) return rc;
  return hip_status(kvq::launch_decode(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale,
                                       causal, window, workspace, (hipStream_t)stream),
                    "decode_attn launch");
}

int kvq_decode_attn_static(const kvq_rows* q, const kvq_qtensor* k, const kvq_qtensor* v, const int32_t* seq_lens,
                           const kvq_rows* out, int B, int Hq, int Hkv, int L, int D, int S, int bits, int group_size,
                           int dtype, float scale, int causal, int window, void* stream) {
  if (check_head_dim(D, "decode")) return KVQ_ERR_UNSUPPORTED;
  int rc = check_attn_args(q, k, v, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale, window);
  if (rc) return rc;
  // the scratch has to hold this call's own plan (its format and group size), not the largest plan
  // any cache format could need at these shapes
  const size_t need = kvq::decode_workspace_bytes(B, Hq, Hkv, L, D, S, window, bits, group_size);
  if (need > (size_t)KVQ_STATIC_SCRATCH_BYTES)
    return fail(KVQ_ERR_WORKSPACE, "this call needs %zu bytes of scratch; the static scratch holds %zu (use kvq_decode_attn "
                "with a workspace)", need, (size_t)KVQ_STATIC_SCRATCH_BYTES);
  void* ws = nullptr;
  if ((rc = static_scratch((hipStream_t)stream, &ws))) return rc;
  return hip_status(kvq::launch_decode(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale,
                                       causal, window, ws, (hipStream_t)stream),
                    "decode_attn_static launch");
}

size_t kvq_prefill_workspace_size(int B, int Hq, int Hkv, int L, int D, int S, int window) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || L <= 0 || S <= 0 || window < 0 || Hq % Hkv) return 0;
  if (!native_dim(D)) {  // the decode kernel serves, or at 96 dims the prefill kernel (prefill_serves_96)
    const size_t n = kvq_decode_workspace_size(B, Hq, Hkv, L, D, S, window);
    return D == 96 && n ? std::max(n, kvq::prefill_workspace_bytes(B, Hq, Hkv, L, D, S, window)) : n;
  }
  if (D == 256) return kvq::wide_workspace_bytes(B, Hq, Hkv, L, D, S, window);
  return kvq::prefill_workspace_bytes(B, Hq, Hkv, L, D, S, window);
}

// The prefill kernel loads two scale groups of a row at once when a row has several: scale and
// bias rows then have to be 4-byte aligned.
static int check_prefill_sb(const kvq_qtensor* k, const kvq_qtensor* v, int D, int group_size) {
  if (D / group_size < 2) return KVQ_OK;
  for (const kvq_qtensor* t : {k, v})
    if (!aligned(t->scales, 4) || !aligned(t->biases, 4) || (t->sb_stride_s | t->sb_stride_h | t->sb_stride_b) & 1)
      return fail(KVQ_ERR_INVALID, "prefill with %d scale groups per row needs 4-byte aligned scales and biases with "
                  "even row, head and batch (page) strides", D / group_size);
  return KVQ_OK;
}

// Whether a quantized head_dim-96 prefill call runs on the prefill kernel. A decode pass serves 4 query
// rows (group 32) and its time grows with them, the prefill kernel's is flat up to a row block of 256:
// 8 KV heads, 8 bits, 64 rows (16 decode passes) 14.8 us against 21.7 at 2048 keys, 38.5 against 48.1
// at 8192 and 130 against 155 at 32768, 48 rows of 12 passes up to even; a 1999-token prompt of 32 heads
// 1276 us on the decode kernel, 53 on the prefill kernel. So the line is at 64 rows. The calls that
// the prefill kernel cannot take as the decode kernel does stay there too: output rows that are not
// 16-byte aligned, and a bf16 cache without range words, whose values may leave the fp16 operands.
static bool prefill_serves_96(const kvq_qtensor* k, const kvq_qtensor* v, const kvq_rows* out, int Hq, int Hkv, int L,
                              int D, int dtype) {
  if (D != 96 || (int64_t)(Hq / Hkv) * L <= 64) return false;
  if (dtype == KVQ_DTYPE_BF16 && (!k->range_exp || !v->range_exp)) return false;
  return aligned(out->data, 16) && !((out->stride_b | out->stride_h | out->stride_l) % 8);
}

int kvq_prefill_attn(const kvq_rows* q, const kvq_qtensor* k, const kvq_qtensor* v, const int32_t* seq_lens,
                     const kvq_rows* out, int B, int Hq, int Hkv, int L, int D, int S, int bits, int group_size,
                     int dtype, float scale, int causal, int window, void* workspace, size_t workspace_bytes,
                     void* stream) {
  if (check_head_dim(D, "prefill")) return KVQ_ERR_UNSUPPORTED;
  int rc = check_attn(q, k, v, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale, window,
                      kvq_prefill_workspace_size(B, Hq, Hkv, L, D, S, window), workspace, workspace_bytes);
  if (rc) return rc;
  const bool at96 = prefill_serves_96(k, v, out, Hq, Hkv, L, D, dtype);
  if (!native_dim(D) && !at96)
    return hip_status(kvq::launch_decode(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale,
                                         causal, window, workspace, (hipStream_t)stream),
                      "prefill_attn launch (the decode kernel, head_dim other than 64/128/256)");
  if (D == 256)
    return hip_status(kvq::launch_wide(q, k, v, seq_lens, out, B, Hq, Hkv, L, S, bits, group_size, dtype, scale, causal,
                                       window, workspace, (hipStream_t)stream),
                      "prefill_attn launch (head_dim 256)");
  if ((rc = check_rows(out, "out", D, true))) return rc;  // rows are stored 16 bytes at a time
  if (!at96 && (rc = check_prefill_sb(k, v, D, group_size))) return rc;
  return hip_status(kvq::launch_prefill(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale,
                                        causal, window, workspace, (hipStream_t)stream),
                    "prefill_attn launch");
}

// Attention over paged pools: the quantized checks with the pool geometry and the block table.
static int check_paged_attn(const kvq_rows* q, const kvq_qtensor* k, const kvq_qtensor* v, int num_pages,
                            const int32_t* table, int64_t table_stride, const kvq_rows* out, int B, int Hq, int Hkv,
                            int L, int D, int S, int bits, int group_size, int dtype, float scale, int window,
                            size_t ws_needed, void* workspace, size_t workspace_bytes) {
  int rc;
  if ((rc = check_attn_common(q, out, B, Hq, Hkv, L, D, S, dtype, scale, window))) return rc;
  if (bits != 4 && bits != 8) return fail(KVQ_ERR_UNSUPPORTED, "attention supports 4- and 8-bit caches, got bits=%d", bits);
  if ((rc = check_attn_group(group_size, D))) return rc;
  if ((rc = check_pool(k, "k_pool", Hkv, D, bits, group_size, num_pages))) return rc;
  if ((rc = check_pool(v, "v_pool", Hkv, D, bits, group_size, num_pages))) return rc;
  for (const kvq_qtensor* t : {k, v})
    if (!aligned(t->codes, 16) || (t->codes_stride_s * 4) % 16 || (t->codes_stride_h * 4) % 16 || (t->codes_stride_b * 4) % 16)
      return fail(KVQ_ERR_INVALID, "codes must be 16-byte aligned with 16-byte-multiple row, head and page strides");
  if ((rc = check_table(table, table_stride, S))) return rc;
  return check_workspace(ws_needed, workspace, workspace_bytes);
}

int kvq_paged_decode_attn(const kvq_rows* q, const kvq_qtensor* k_pool, const kvq_qtensor* v_pool, int num_pages,
                          const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens,
                          const kvq_rows* out, int B, int Hq, int Hkv, int L, int D, int S, int bits, int group_size,
                          int dtype, float scale, int causal, int window, void* workspace, size_t workspace_bytes,
                          void* stream) {
  if (check_head_dim(D, "decode")) return KVQ_ERR_UNSUPPORTED;
  int rc = check_paged_attn(q, k_pool, v_pool, num_pages, block_table, table_stride, out, B, Hq, Hkv, L, D, S, bits,
                            group_size, dtype, scale, window, kvq_decode_workspace_size(B, Hq, Hkv, L, D, S, window),
                            workspace, workspace_bytes);
  if (rc) return rc;
  return hip_status(kvq::launch_decode_paged(q, k_pool, v_pool, num_pages, block_table, table_stride, seq_lens, out, B,
                                             Hq, Hkv, L, D, S, bits, group_size, dtype, scale, causal, window,
                                             workspace, (hipStream_t)stream),
                    "paged_decode_attn launch");
}

int kvq_paged_prefill_attn(const kvq_rows* q, const kvq_qtensor* k_pool, const kvq_qtensor* v_pool, int num_pages,
                           const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens,
                           const kvq_rows* out, int B, int Hq, int Hkv, int L, int D, int S, int bits, int group_size,
                           int dtype, float scale, int causal, int window, void* workspace, size_t workspace_bytes,
                           void* stream) {
  if (check_head_dim(D, "prefill")) return KVQ_ERR_UNSUPPORTED;
  int rc = check_paged_attn(q, k_pool, v_pool, num_pages, block_table, table_stride, out, B, Hq, Hkv, L, D, S, bits,
                            group_size, dtype, scale, window, kvq_prefill_workspace_size(B, Hq, Hkv, L, D, S, window),
                            workspace, workspace_bytes);
  if (rc) return rc;
  const bool at96 = prefill_serves_96(k_pool, v_pool, out, Hq, Hkv, L, D, dtype);
  if (!native_dim(D) && !at96)
    return hip_status(kvq::launch_decode_paged(q, k_pool, v_pool, num_pages, block_table, table_stride, seq_lens, out,
                                               B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale, causal, window,
                                               workspace, (hipStream_t)stream),
                      "paged_prefill_attn launch (the decode kernel, head_dim other than 64/128/256)");
  if (D == 256)
    return hip_status(kvq::launch_wide_paged(q, k_pool, v_pool, num_pages, block_table, table_stride, seq_lens, out, B,
                                             Hq, Hkv, L, S, bits, group_size, dtype, scale, causal, window, workspace,
                                             (hipStream_t)stream),
                      "paged_prefill_attn launch (head_dim 256)");
  if ((rc = check_rows(out, "out", D, true))) return rc;  // rows are stored 16 bytes at a time
  if (!at96 && (rc = check_prefill_sb(k_pool, v_pool, D, group_size))) return rc;
  return hip_status(kvq::launch_prefill_paged(q, k_pool, v_pool, num_pages, block_table, table_stride, seq_lens, out, B,
                                              Hq, Hkv, L, D, S, bits, group_size, dtype, scale, causal, window,
                                              workspace, (hipStream_t)stream),
                    "paged_prefill_attn launch");
}

int kvq_decode_attn_dense(const kvq_rows* q, const kvq_rows* k, const kvq_rows* v, const int32_t* seq_lens,
                          const kvq_rows* out, int B, int Hq, int Hkv, int L, int D, int S, int dtype, float scale,
                          int causal, int window, void* workspace, size_t workspace_bytes, void* stream) {
  if (check_head_dim(D, "unquantized decode")) return KVQ_ERR_UNSUPPORTED;
  int rc = check_attn_dense(q, k, v, out, B, Hq, Hkv, L, D, S, dtype, scale, window,
                            kvq_decode_workspace_size(B, Hq, Hkv, L, D, S, window), workspace, workspace_bytes);
  if (rc) return rc;
  if (D > 128)
    return hip_status(kvq::launch_wide_dense(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, dtype, scale, causal, window,
                                             workspace, (hipStream_t)stream),
                      "decode_attn_dense launch (the head_dim-256 kernel)");
  return hip_status(kvq::launch_decode_dense(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, dtype, scale, causal, window,
                                             workspace, (hipStream_t)stream),
                    "decode_attn_dense launch");
}

// A general mask: a known kind, a pointer aligned to its element, non-negative strides (the key
// stride is 1 by definition).
static int check_mask(const kvq_mask* m) {
  if (!m || !m->data) return fail(KVQ_ERR_INVALID, "mask and mask->data must not be NULL");
  if (m->kind < KVQ_MASK_BOOL || m->kind > KVQ_MASK_F32) return fail(KVQ_ERR_INVALID, "unknown mask kind %d", m->kind);
  const uintptr_t el = m->kind == KVQ_MASK_BOOL ? 1 : m->kind == KVQ_MASK_F32 ? 4 : 2;
  if (!aligned(m->data, el)) return fail(KVQ_ERR_INVALID, "mask data is not aligned to its %zu-byte elements", (size_t)el);
  if (m->stride_b < 0 || m->stride_kvh < 0 || m->stride_rep < 0 || m->stride_l < 0)
    return fail(KVQ_ERR_INVALID, "mask strides must be non-negative");
  return KVQ_OK;
}

// Whether a call under a general mask runs on the prefill kernel: enough query rows per KV head, a head
// dim it has, rows it can store, a cache whose values its operands hold (a bf16 cache needs its range
// words), and over a quantized cache a boolean mask (the tile loop's scalar registers hold no more than
// that reading). The others stay on the decode kernel.
static bool masked_on_prefill(const kvq_qtensor* k, const kvq_qtensor* v, const kvq_rows* out, int B, int Hq, int Hkv, int L,
                              int D, int S, int group_size, int dtype, const kvq_mask* mask, size_t ws_bytes) {
  if (!kvq::prefill_masked_rows(B, Hq, Hkv, L, D, S)) return false;
  const bool rows16 = aligned(out->data, 16) && !((out->stride_b | out->stride_h | out->stride_l) % 8);
  if (!k) {
    if (D != 64 && (D != 128 || !rows16)) return false;
  } else {
    if (mask->kind != KVQ_MASK_BOOL) return false;
    if ((D != 64 && D != 96 && D != 128) || !rows16) return false;
    if (D != 96 && check_prefill_sb(k, v, D, group_size)) return false;
    if (dtype == KVQ_DTYPE_BF16 && (!k->range_exp || !v->range_exp)) return false;
  }
  return kvq::prefill_masked_fits(B, Hq, Hkv, L, D, S, mask, ws_bytes);
}

int kvq_masked_on_prefill(int B, int Hq, int Hkv, int L, int D, int S) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || L <= 0 || S <= 0 || Hq % Hkv) return 0;
  return kvq::prefill_masked_rows(B, Hq, Hkv, L, D, S) ? 1 : 0;
}

int kvq_decode_attn_masked(const kvq_rows* q, const kvq_qtensor* k, const kvq_qtensor* v, const kvq_rows* out, int B,
                           int Hq, int Hkv, int L, int D, int S, int bits, int group_size, int dtype, float scale,
                           const kvq_mask* mask, void* workspace, size_t workspace_bytes, void* stream) {
  if (check_head_dim(D, "decode")) return KVQ_ERR_UNSUPPORTED;
  const size_t ws = kvq_decode_workspace_size(B, Hq, Hkv, L, D, S, 0);
  int rc = check_attn(q, k, v, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale, 0, ws, workspace,
                      workspace_bytes);
  if (rc || (rc = check_mask(mask))) return rc;
  if (masked_on_prefill(k, v, out, B, Hq, Hkv, L, D, S, group_size, dtype, mask, ws))
    return hip_status(kvq::launch_prefill_masked(q, k, v, nullptr, nullptr, out, B, Hq, Hkv, L, D, S, bits, group_size,
                                                 dtype, scale, mask, workspace, ws, (hipStream_t)stream),
                      "decode_attn_masked launch (the prefill kernel)");
  return hip_status(kvq::launch_decode(q, k, v, nullptr, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale, 0, 0,
                                       workspace, (hipStream_t)stream, mask),
                    "decode_attn_masked launch");
}

int kvq_decode_attn_dense_masked(const kvq_rows* q, const kvq_rows* k, const kvq_rows* v, const kvq_rows* out, int B,
                                 int Hq, int Hkv, int L, int D, int S, int dtype, float scale, const kvq_mask* mask,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (check_head_dim(D, "masked unquantized attention")) return KVQ_ERR_UNSUPPORTED;
  const size_t ws = kvq_decode_workspace_size(B, Hq, Hkv, L, D, S, 0);
  int rc = check_attn_dense(q, k, v, out, B, Hq, Hkv, L, D, S, dtype, scale, 0, ws, workspace, workspace_bytes);
  if (rc || (rc = check_mask(mask))) return rc;
  if (D > 128)  // unquantized rows past 128 dims run through the head_dim-256 kernel
    return hip_status(kvq::launch_wide_dense(q, k, v, nullptr, out, B, Hq, Hkv, L, D, S, dtype, scale, 0, 0, workspace,
                                             (hipStream_t)stream, mask),
                      "decode_attn_dense_masked launch (the head_dim-256 kernel)");
  if (masked_on_prefill(nullptr, nullptr, out, B, Hq, Hkv, L, D, S, 64, dtype, mask, ws))
    return hip_status(kvq::launch_prefill_masked(q, nullptr, nullptr, k, v, out, B, Hq, Hkv, L, D, S, 16, 64, dtype, scale,
                                                 mask, workspace, ws, (hipStream_t)stream),
                      "decode_attn_dense_masked launch (the prefill kernel)");
  return hip_status(kvq::launch_decode_dense(q, k, v, nullptr, out, B, Hq, Hkv, L, D, S, dtype, scale, 0, 0, workspace,
                                             (hipStream_t)stream, mask),
                    "decode_attn_dense_masked launch");
}

// ---- trees of drafted tokens

int kvq_draft_tree(const int32_t* parents, int64_t parents_stride_b, int B, int L, uint32_t* bits, int32_t* depths,
                   const int32_t* starts, int64_t start, int32_t* positions, void* stream) {
  if (!parents || !bits || !depths) return fail(KVQ_ERR_INVALID, "parents, bits and depths must not be NULL");
  if (B < 0 || L < 0) return fail(KVQ_ERR_INVALID, "negative shape (B=%d L=%d)", B, L);
  if (L > KVQ_TREE_MAX_NODES || B > 65535)
    return fail(KVQ_ERR_UNSUPPORTED, "a tree has at most %d nodes and a batch 65535 trees, got %d and %d", KVQ_TREE_MAX_NODES, L, B);
  if (parents_stride_b < 0) return fail(KVQ_ERR_INVALID, "parents have a negative batch stride");
  if (!aligned(parents, 4) || !aligned(bits, 4) || !aligned(depths, 4) || !aligned(starts, 4) || !aligned(positions, 4))
    return fail(KVQ_ERR_INVALID, "parents, bits, depths, starts and positions must be 4-byte aligned");
  if (B == 0 || L == 0) return ok();
  return hip_status(kvq::launch_draft_tree(parents, parents_stride_b, B, L, bits, depths, starts, start, positions,
                                           (hipStream_t)stream),
                    "draft_tree launch");
}

static int check_tree(const kvq_tree* t, int L, float scale, int window) {
  // (the kernels hide keys before they scale)
  if (!(scale > 0.0f)) return fail(KVQ_ERR_INVALID, "tree attention needs a positive scale, got %g", (double)scale);
  if (!t || !t->bits || !t->depths) return fail(KVQ_ERR_INVALID, "tree, tree->bits and tree->depths must not be NULL");
  if (!aligned(t->bits, 4) || !aligned(t->depths, 4) || t->bits_stride_b < 0 || t->depths_stride_b < 0)
    return fail(KVQ_ERR_INVALID, "tree bits and depths must be 4-byte aligned with non-negative batch strides");
  if (L > KVQ_TREE_MAX_NODES) return fail(KVQ_ERR_UNSUPPORTED, "a tree has at most %d nodes, got L=%d", KVQ_TREE_MAX_NODES, L);
  // an ancestor is then never outside the window of its descendants
  if (window > 0 && window < L) return fail(KVQ_ERR_UNSUPPORTED, "a tree of %d nodes needs a window of at least as many keys, got %d", L, window);
  return KVQ_OK;
}

// The kernel of a tree call by its sizes: the one whose time is estimated the lowest. rows: a KV head's query rows.
//   decode: a launch, 25 us (64 dims 18, unquantized 12.5; 96 dims 30; 256 dims 35) for a million keys of a pass of 16 G / D
//           rows (D the kernel's width), and 2.5 for 512 workgroups of it (unquantized 64 dims none);
//   rows:   its plan's model (tree_attn.hip), 64 and 128 dims;
//   prefill: a launch or two and 130 us (64 dims 85, 96 dims 100) for a million keys of a block of 256 rows; 256 dims:
//           145 of 128 rows.
// Over 260 random calls the choice came to 1.6% more than the best of the three on average (a choice by rows and keys
// alone 5%), 41% at most. us, decode / rows / prefill (128 dims, groups of 64, 8 bits, 8 KV heads unless said):
//   20 rows,  4106 keys   11.5 /  13.8 /  22    32 rows, 8 sequences of 4096, 4 bits  32.5 / 26.2 / 53.0
//   24 rows, 16384 keys   20.1 /  25.8 /  32    64 rows, 8 sequences of 6144, 4 bits  68.9 / 40.3 / 71.8
//   64 rows,  4096 keys   14.5 /  13.8 /  21   128 rows, 32768 keys                    116 / 48.8 / 53.6
//   64 rows,  8192 keys   21.6 /  18.7 /  25   192 rows, 32768 keys                    215 / 65.7 / 56.4
//  256 rows,  2048 keys   20.6 /  20.7 /  24   256 rows, 32768 keys                    215 / 79.9 / 59.6
//  124 rows of 64 unquantized dims, 4 sequences of 2047: 11.0 / 11.9 / 22; 44 rows of 64 dims, 64 units of 19345: 105 / 60 / 111
//  928 unquantized rows, 32 units of 265: 90 / 39.5 / 19.3
// At 96 and 256 dims, of two, 1.2% and 1.9% above the better over 70 random calls each (choices by rows and passes 16% and
// 5%, 334% and 104% at most).
enum class TreeKernel { kDecode, kRows, kPrefill };
static TreeKernel tree_kernel_of(int B, int Hq, int Hkv, int L, int D, int S, int bits, int group_size, int window) {
  const bool dense = bits == 16;
  const int64_t rows = (int64_t)(Hq / Hkv) * L, units = (int64_t)B * Hkv;
  const int64_t keys = window > 0 ? std::min((int64_t)S, (int64_t)window + L) : S;
  if ((D != 64 && D != 96 && D != 128 && D != 256) || (dense && D != 64 && D != 128) || rows <= 8) return TreeKernel::kDecode;
  const int64_t per = std::max(16 * (int64_t)group_size / (D == 96 ? 128 : D), (int64_t)1), passes = (rows + per - 1) / per;
  const int64_t block = D == 256 ? 128 : 256, blocks = (rows + block - 1) / block;
  const float work = (float)(units * keys) * 1e-6f;
  const float pass_us = D == 256 ? 35.0f : D == 128 ? 25.0f : D == 96 ? 30.0f : dense ? 12.5f : 18.0f;
  const float block_us = D == 256 ? 145.0f : D == 128 ? 130.0f : D == 96 ? 100.0f : 85.0f;
  const float decode = 7.5f + pass_us * work * passes + (D == 64 && dense ? 0.0f : 2.5f / 512) * (float)(units * passes);
  const float prefill = (D == 256 ? 16.0f : 14.5f) + block_us * work * blocks;
  if (D == 96 || D == 256) return decode <= prefill ? TreeKernel::kDecode : TreeKernel::kPrefill;
  const float mine = kvq::tree_rows_time(B, Hq, Hkv, L, D, S, window, bits);
  return decode <= mine && decode <= prefill ? TreeKernel::kDecode : mine <= prefill ? TreeKernel::kRows : TreeKernel::kPrefill;
}

int kvq_tree_kernel(int B, int Hq, int Hkv, int L, int D, int S, int bits, int group_size, int window) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || L <= 0 || S <= 0 || D <= 0 || window < 0 || group_size <= 0 || Hq % Hkv) return 0;
  if (bits == 16) group_size = 64;
  return (int)tree_kernel_of(B, Hq, Hkv, L, D, S, bits, group_size, window);
}

// ... and after: what the prefill kernel cannot take (a bf16 cache without range words, output or scale rows that are not
// aligned for it) runs on the rows kernel, of a width that has none on the decode kernel.
static TreeKernel tree_kernel_for(const kvq_qtensor* k, const kvq_qtensor* v, const kvq_rows* out, int B, int Hq, int Hkv,
                                  int L, int D, int S, int bits, int group_size, int dtype, int window) {
  const TreeKernel t = tree_kernel_of(B, Hq, Hkv, L, D, S, bits, group_size, window);
  if (t != TreeKernel::kPrefill) return t;
  bool ok = !k || dtype != KVQ_DTYPE_BF16 || (k->range_exp && v->range_exp);
  if (D != 256) {
    const bool rows16 = aligned(out->data, 16) && !((out->stride_b | out->stride_h | out->stride_l) % 8);
    ok = ok && (rows16 || (!k && D == 64)) && (!k || D == 96 || check_prefill_sb(k, v, D, group_size) == KVQ_OK);
  }
  return ok ? t : D == 64 || D == 128 ? TreeKernel::kRows : TreeKernel::kDecode;
}

size_t kvq_tree_workspace_size(int B, int Hq, int Hkv, int L, int D, int S, int window) {
  size_t n = kvq_decode_workspace_size(B, Hq, Hkv, L, D, S, window);
  if (n == 0 || Hq % Hkv) return 0;
  if (D == 64 || D == 96 || D == 128) n = std::max(n, kvq::prefill_tree_bytes(B, Hq, Hkv, L, D, S, window));
  if (D == 64 || D == 128) n = std::max(n, kvq::tree_rows_bytes(B, Hq, Hkv, L, D, S, window));
  return n;  // (the decode size covers the head_dim-256 kernel)
}

int kvq_tree_attn(const kvq_rows* q, const kvq_qtensor* k, const kvq_qtensor* v, const int32_t* seq_lens,
                  const kvq_rows* out, int B, int Hq, int Hkv, int L, int D, int S, int bits, int group_size, int dtype,
                  float scale, const kvq_tree* tree, int window, void* workspace, size_t workspace_bytes, void* stream) {
  if (check_head_dim(D, "tree attention")) return KVQ_ERR_UNSUPPORTED;
  int rc = check_attn(q, k, v, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale, window,
                      kvq_tree_workspace_size(B, Hq, Hkv, L, D, S, window), workspace, workspace_bytes);
  if (rc || (rc = check_tree(tree, L, scale, window))) return rc;
  const TreeKernel kernel = tree_kernel_for(k, v, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, window);
  hipError_t e;
  if (kernel != TreeKernel::kPrefill) {
    e = kvq::launch_decode(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale, 0, window, workspace,
                           (hipStream_t)stream, nullptr, tree, kernel == TreeKernel::kRows);
  } else if (D == 256) {
    e = kvq::launch_wide(q, k, v, seq_lens, out, B, Hq, Hkv, L, S, bits, group_size, dtype, scale, 0, window, workspace,
                         (hipStream_t)stream, tree);
  } else {
    e = kvq::launch_prefill(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, scale, 0, window, workspace,
                            (hipStream_t)stream, tree);
  }
  return hip_status(e, "tree_attn launch");
}

int kvq_paged_tree_attn(const kvq_rows* q, const kvq_qtensor* k_pool, const kvq_qtensor* v_pool, int num_pages,
                        const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens, const kvq_rows* out,
                        int B, int Hq, int Hkv, int L, int D, int S, int bits, int group_size, int dtype, float scale,
                        const kvq_tree* tree, int window, void* workspace, size_t workspace_bytes, void* stream) {
  if (check_head_dim(D, "tree attention")) return KVQ_ERR_UNSUPPORTED;
  int rc = check_paged_attn(q, k_pool, v_pool, num_pages, block_table, table_stride, out, B, Hq, Hkv, L, D, S, bits,
                            group_size, dtype, scale, window, kvq_tree_workspace_size(B, Hq, Hkv, L, D, S, window),
                            workspace, workspace_bytes);
  if (rc || (rc = check_tree(tree, L, scale, window))) return rc;
  if (!seq_lens) return fail(KVQ_ERR_INVALID, "seq_lens is NULL");
  const TreeKernel kernel = tree_kernel_for(k_pool, v_pool, out, B, Hq, Hkv, L, D, S, bits, group_size, dtype, window);
  hipError_t e;
  if (kernel != TreeKernel::kPrefill) {
    e = kvq::launch_decode_paged(q, k_pool, v_pool, num_pages, block_table, table_stride, seq_lens, out, B, Hq, Hkv, L, D, S,
                                 bits, group_size, dtype, scale, 0, window, workspace, (hipStream_t)stream, tree,
                                 kernel == TreeKernel::kRows);
  } else if (D == 256) {
    e = kvq::launch_wide_paged(q, k_pool, v_pool, num_pages, block_table, table_stride, seq_lens, out, B, Hq, Hkv, L, S, bits,
                               group_size, dtype, scale, 0, window, workspace, (hipStream_t)stream, tree);
  } else {
    e = kvq::launch_prefill_paged(q, k_pool, v_pool, num_pages, block_table, table_stride, seq_lens, out, B, Hq, Hkv, L, D, S,
                                  bits, group_size, dtype, scale, 0, window, workspace, (hipStream_t)stream, tree);
  }
  return hip_status(e, "paged_tree_attn launch");
}

int kvq_tree_attn_dense(const kvq_rows* q, const kvq_rows* k, const kvq_rows* v, const int32_t* seq_lens,
                        const kvq_rows* out, int B, int Hq, int Hkv, int L, int D, int S, int dtype, float scale,
                        const kvq_tree* tree, int window, void* workspace, size_t workspace_bytes, void* stream) {
  if (check_head_dim(D, "unquantized tree attention")) return KVQ_ERR_UNSUPPORTED;
  int rc = check_attn_dense(q, k, v, out, B, Hq, Hkv, L, D, S, dtype, scale, window,
                            kvq_tree_workspace_size(B, Hq, Hkv, L, D, S, window), workspace, workspace_bytes);
  if (rc || (rc = check_tree(tree, L, scale, window))) return rc;
  const TreeKernel kernel = tree_kernel_for(nullptr, nullptr, out, B, Hq, Hkv, L, D, S, 16, 64, dtype, window);
  hipError_t e;
  if (D > 128) {  // unquantized rows past 128 dims run through the head_dim-256 kernel
    e = kvq::launch_wide_dense(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, dtype, scale, 0, window, workspace,
                               (hipStream_t)stream, nullptr, tree);
  } else if (kernel == TreeKernel::kPrefill) {
    e = kvq::launch_prefill_dense(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, dtype, scale, 0, window, workspace,
                                  (hipStream_t)stream, tree);
  } else {
    e = kvq::launch_decode_dense(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, dtype, scale, 0, window, workspace,
                                 (hipStream_t)stream, nullptr, tree, kernel == TreeKernel::kRows);
  }
  return hip_status(e, "tree_attn_dense launch");
}

int kvq_prefill_attn_dense(const kvq_rows* q, const kvq_rows* k, const kvq_rows* v, const int32_t* seq_lens,
                           const kvq_rows* out, int B, int Hq, int Hkv, int L, int D, int S, int dtype, float scale,
                           int causal, int window, void* workspace, size_t workspace_bytes, void* stream) {
  if (check_head_dim(D, "unquantized prefill")) return KVQ_ERR_UNSUPPORTED;
  int rc = check_attn_dense(q, k, v, out, B, Hq, Hkv, L, D, S, dtype, scale, window,
                            kvq_prefill_workspace_size(B, Hq, Hkv, L, D, S, window), workspace, workspace_bytes);
  if (rc) return rc;
  if (D > 128 && D < 256)
    return hip_status(kvq::launch_wide_dense(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, dtype, scale, causal, window,
                                             workspace, (hipStream_t)stream),
                      "prefill_attn_dense launch (the head_dim-256 kernel)");
  if (!native_dim(D))
    return hip_status(kvq::launch_decode_dense(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, dtype, scale, causal, window,
                                               workspace, (hipStream_t)stream),
                      "prefill_attn_dense launch (the decode kernel, head_dim other than 64/128/256)");
  if (D == 256)
    return hip_status(kvq::launch_wide_dense(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, dtype, scale, causal, window,
                                             workspace, (hipStream_t)stream),
                      "prefill_attn_dense launch (head_dim 256)");
  if (D == 128 && (rc = check_rows(out, "out", D, true))) return rc;  // rows are stored 16 bytes at a time
  return hip_status(kvq::launch_prefill_dense(q, k, v, seq_lens, out, B, Hq, Hkv, L, D, S, dtype, scale, causal, window,
                                              workspace, (hipStream_t)stream),
                    "prefill_attn_dense launch");
}

}  // extern "C"
