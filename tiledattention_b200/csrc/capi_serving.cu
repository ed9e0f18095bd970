// C ABI of the operators around a decoder's attention: rotary positions, the write into the
// paged 8-bit cache and attention over it. Argument checks and launches; see
// include/tiledattention_b200.h for the contracts.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstdio>

#include "capi_internal.h"
#include "kv8.h"
#include "rotary.h"
#include "tiledattention_b200.h"

namespace {

// Multiprocessors of the current device (looked up once per device); 0 on failure.
int sm_count() {
  static int cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64) {
    const int known = __atomic_load_n(&cached[dev], __ATOMIC_RELAXED);
    if (known) return known;
  }
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) __atomic_store_n(&cached[dev], n, __ATOMIC_RELAXED);
  return n;
}

bool is_16bit(int dtype) { return dtype == TA_DTYPE_F16 || dtype == TA_DTYPE_BF16; }

bool aligned(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Bytes, a power of two up to 16, that divide the base and the outer strides (of dims with more than
// one entry) of 16-bit values.
int rows_alignment(const void* p, const int64_t* st, int64_t n0, int64_t n1, int64_t n2) {
  uint64_t bits = reinterpret_cast<uintptr_t>(p) | 16;
  const int64_t n[3] = {n0, n1, n2};
  for (int i = 0; i < 3; ++i)
    if (n[i] != 1) bits |= static_cast<uint64_t>(st[i]) * 2;
  return static_cast<int>(bits & (~bits + 1));
}
bool rows_aligned(const void* p, const int64_t* st, int64_t n0, int64_t n1, int64_t n2) {
  return rows_alignment(p, st, n0, n1, n2) == 16;
}

int launched(cudaError_t err, const char* what) {
  if (err == cudaSuccess) return TA_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(err));
  return ta_capi_fail(TA_ERR_CUDA, buf);
}

// Checks shared by the two cache operators.
int check_cache(const void* k_pages, const void* v_pages, const float* k_scale,
                const float* v_scale, int num_pages, int page, const int* table,
                int64_t table_stride, int table_width, int B, int Hkv, int T, int D) {
  if (!k_pages || !v_pages || !k_scale || !v_scale || !table)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (B <= 0 || Hkv <= 0 || T <= 0 || num_pages <= 0 || table_width <= 0)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT,
                        "B, Hkv, T, num_pages and table_width must be positive");
  if (D < 16 || D > 256 || D % 16 != 0)
    return ta_capi_fail(TA_ERR_UNSUPPORTED_DIM,
                        "head dim of the 8-bit cache: a multiple of 16 up to 256");
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "page size must be 16, 32, 64 or 128");
  if (static_cast<int64_t>(table_width) * page > 0x7fffffffll)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "table_width * page must be below 2^31");
  if (table_stride < table_width && B > 1)
    return ta_capi_fail(TA_ERR_LAYOUT, "page table rows overlap");
  if (static_cast<int64_t>(num_pages) * Hkv > 0x7fffffffll)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "num_pages * Hkv must be below 2^31");
  if (Hkv > 65535) return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "too many heads");
  if (!aligned(k_pages, 16) || !aligned(v_pages, 16))
    return ta_capi_fail(TA_ERR_LAYOUT, "cache pages must be 16-byte aligned");
  return TA_OK;
}

// Map of the cache's pages as (D, page, P * Hkv) bytes with boxes of `rows` tokens; columns from
// D on read as zeros.
int make_pages_map(CUtensorMap* map, const void* pages, int D, int page, int64_t planes, int rows) {
  const auto enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ta_capi_tensor_map_encoder());
  if (!enc) return ta_capi_fail(TA_ERR_DRIVER, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(page),
                              static_cast<cuuint64_t>(planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(D) * page};
  const cuuint32_t box[3] = {D <= 64 ? 64u : 128u, static_cast<cuuint32_t>(rows), 1};
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(pages), dims,
                         strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         D <= 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TA_OK
                           : ta_capi_fail(TA_ERR_LAYOUT, "cuTensorMapEncodeTiled rejected the cache");
}

int64_t workspace_bytes_of(int B, int Hq, int Hkv, int T, int D, int sms) {
  const int64_t rows = static_cast<int64_t>(Hq / Hkv) * T;
  if (rows >= (1 << 24) || Hq / Hkv > ta::kv8::kMaxGroup) return 0;
  return static_cast<int64_t>(ta::kv8::uses_chunk(static_cast<int>(rows), D)
                                  ? ta::kv8::chunk_workspace_bytes(D, sms)
                                  : ta::kv8::attend_workspace_bytes(B, Hq, Hkv, T, D, sms));
}

}  // namespace

namespace ta {
namespace kv8 {
// Many rows fill the chunk kernel's tiles of 128; few rows are served by the other kernel, whose time
// grows with each 32 rows (16 above head dim 128) while the chunk kernel's stays. Measured, few-row
// kernel and chunk kernel, 16 sequences of 8192, 8 cache heads: head dim 128, 32 rows
// 108 and 173 us, 40 rows 184 and 174; head dim 256, 48 rows 272 and 274 us, 64 rows 382 and 275.
// A single short sequence loses by it (2048 tokens, 2 cache heads, head dim 128, 40 rows: 20 and 25 us).
bool uses_chunk(int rows, int D) { return rows > (D > 128 ? 48 : 32); }
}  // namespace kv8
}  // namespace ta

extern "C" {

int ta_rotary(const void* q, void* q_out, const int64_t* q_strides, const int64_t* q_out_strides,
              int Hq, const void* k, void* k_out, const int64_t* k_strides,
              const int64_t* k_out_strides, int Hk, int B, int S, int D, int rotary_dim,
              const void* positions, int positions_64, const int64_t* position_strides,
              const double* inv_freq, int interleaved, int inverse, float magnitude, int dtype,
              void* stream) {
  TaNvtxRange nvtx_range("ta_rotary");
  ta_capi_clear_error();
  if (!q || !q_out || !q_strides || !q_out_strides || !positions || !position_strides || !inv_freq)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "null pointer argument");
  if ((k != nullptr) != (Hk > 0) ||
      (k && (!k_out || !k_strides || !k_out_strides)))
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "k: pointers and a head count, or neither");
  if (B <= 0 || Hq <= 0 || Hk < 0 || S <= 0 || D <= 0)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "B, H, S, D must be positive");
  if (rotary_dim < 2 || rotary_dim > D || rotary_dim % 2 != 0)
    return ta_capi_fail(TA_ERR_UNSUPPORTED_DIM, "rotary dims: an even number from 2 to the head dim");
  if (!is_16bit(dtype)) return ta_capi_fail(TA_ERR_UNSUPPORTED_DTYPE, "rotary: fp16 or bf16");
  if (!std::isfinite(magnitude))
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "magnitude must be finite");
  if (q_strides[3] != 1 || q_out_strides[3] != 1 ||
      (k && (k_strides[3] != 1 || k_out_strides[3] != 1)))
    return ta_capi_fail(TA_ERR_LAYOUT, "rotary: head-dim stride must be 1");
  const int rc = ta_capi_check_device();
  if (rc) return rc;
  ta::RotaryParams p{};
  p.t[0] = {q, q_out, q_strides[0], q_strides[1], q_strides[2],
            q_out_strides[0], q_out_strides[1], q_out_strides[2], Hq};
  int alignment = std::min(rows_alignment(q, q_strides, B, Hq, S),
                           rows_alignment(q_out, q_out_strides, B, Hq, S));
  if (k) {
    p.t[1] = {k, k_out, k_strides[0], k_strides[1], k_strides[2],
              k_out_strides[0], k_out_strides[1], k_out_strides[2], Hk};
    alignment = std::min({alignment, rows_alignment(k, k_strides, B, Hk, S),
                          rows_alignment(k_out, k_out_strides, B, Hk, S)});
  }
  p.positions = positions;
  p.pos_sb = position_strides[0];
  p.pos_ss = position_strides[1];
  p.inv_freq = inv_freq;
  p.B = B;
  p.S = S;
  p.D = D;
  p.half = rotary_dim / 2;
  p.pos64 = positions_64 != 0;
  p.interleaved = interleaved != 0;
  p.inverse = inverse != 0;
  p.bf16 = dtype == TA_DTYPE_BF16;
  p.magnitude = magnitude;
  return launched(ta::launch_rotary(p, alignment, sm_count(), static_cast<cudaStream_t>(stream)),
                  "rotary launch failed");
}

int ta_kv8_append(const void* k, const void* v, const int64_t* k_strides, const int64_t* v_strides,
                  void* k_pages, void* v_pages, float* k_scale, float* v_scale, int num_pages,
                  int page, const int* table, int64_t table_stride, int table_width,
                  const int* starts, const int* counts, int B, int Hkv, int T, int D, int dtype,
                  unsigned int* dev_status, void* stream) {
  TaNvtxRange nvtx_range("ta_kv8_append");
  ta_capi_clear_error();
  if (!k || !v || !k_strides || !v_strides || !starts)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "null pointer argument");
  int rc = check_cache(k_pages, v_pages, k_scale, v_scale, num_pages, page, table, table_stride,
                       table_width, B, Hkv, T, D);
  if (rc) return rc;
  if (!is_16bit(dtype)) return ta_capi_fail(TA_ERR_UNSUPPORTED_DTYPE, "k, v: fp16 or bf16");
  if (k_strides[3] != 1 || v_strides[3] != 1 || !rows_aligned(k, k_strides, B, Hkv, T) ||
      !rows_aligned(v, v_strides, B, Hkv, T))
    return ta_capi_fail(TA_ERR_LAYOUT,
                        "k, v: unit head-dim stride, base and strides multiples of 16 bytes");
  if ((rc = ta_capi_check_device())) return rc;
  ta::kv8::AppendParams p{};
  p.x[0] = k;
  p.x[1] = v;
  const int64_t* st[2] = {k_strides, v_strides};
  for (int i = 0; i < 2; ++i) {
    p.sb[i] = st[i][0];
    p.sh[i] = st[i][1];
    p.ss[i] = st[i][2];
  }
  p.pages[0] = static_cast<uint8_t*>(k_pages);
  p.pages[1] = static_cast<uint8_t*>(v_pages);
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.table = table;
  p.table_stride = table_stride;
  p.starts = starts;
  p.counts = counts;
  p.status = dev_status;
  p.B = B;
  p.Hkv = Hkv;
  p.T = T;
  p.D = D;
  p.page = page;
  p.width = table_width;
  p.num_pages = num_pages;
  p.bf16 = dtype == TA_DTYPE_BF16;
  return launched(ta::kv8::launch_append(p, static_cast<cudaStream_t>(stream)),
                  "cache append launch failed");
}

int64_t ta_sdpa_kv8_workspace(int B, int Hq, int Hkv, int T, int D) {
  ta_capi_clear_error();
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || D <= 0 || D > 256 || Hq % Hkv != 0) return 0;
  return workspace_bytes_of(B, Hq, Hkv, T, D, sm_count());
}

int ta_sdpa_kv8(const void* q, const int64_t* q_strides, void* o, const int64_t* o_strides,
                float* lse, const void* k_pages, const void* v_pages, const float* k_scale,
                const float* v_scale, int num_pages, int page, const int* table,
                int64_t table_stride, int table_width, const int* lengths, const int* counts,
                int B, int Hq, int Hkv, int T, int D, int dtype, int causal, float scale,
                void* workspace, int64_t workspace_bytes, unsigned int* dev_status, void* stream) {
  TaNvtxRange nvtx_range("ta_sdpa_kv8");
  ta_capi_clear_error();
  if (!q || !o || !q_strides || !o_strides || !lengths)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "null pointer argument");
  int rc = check_cache(k_pages, v_pages, k_scale, v_scale, num_pages, page, table, table_stride,
                       table_width, B, Hkv, T, D);
  if (rc) return rc;
  if (Hq <= 0 || Hq % Hkv != 0)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "query heads must be a multiple of the cache's heads");
  if (Hq / Hkv > ta::kv8::kMaxGroup)
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "at most 256 query heads per cache head");
  if (static_cast<int64_t>(Hq / Hkv) * T >= (1 << 24))
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "too many query rows per cache head");
  if (!workspace) return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "null workspace");
  if (!is_16bit(dtype)) return ta_capi_fail(TA_ERR_UNSUPPORTED_DTYPE, "q: fp16 or bf16");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "scale must be a positive finite number");
  if (q_strides[3] != 1 || o_strides[3] != 1 || !rows_aligned(q, q_strides, B, Hq, T) ||
      !rows_aligned(o, o_strides, B, Hq, T))
    return ta_capi_fail(TA_ERR_LAYOUT,
                        "q, o: unit head-dim stride, base and strides multiples of 16 bytes");
  if ((rc = ta_capi_check_device())) return rc;
  const int sms = sm_count();
  if (!aligned(workspace, 16) ||
      workspace_bytes < workspace_bytes_of(B, Hq, Hkv, T, D, sms))
    return ta_capi_fail(TA_ERR_INVALID_ARGUMENT, "workspace too small or not 16-byte aligned");
  ta::kv8::AttendParams p{};
  p.q = q;
  p.q_sb = q_strides[0];
  p.q_sh = q_strides[1];
  p.q_ss = q_strides[2];
  p.o = o;
  p.o_sb = o_strides[0];
  p.o_sh = o_strides[1];
  p.o_ss = o_strides[2];
  p.lse = lse;
  p.pages[0] = static_cast<const uint8_t*>(k_pages);
  p.pages[1] = static_cast<const uint8_t*>(v_pages);
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.table = table;
  p.table_stride = table_stride;
  p.lengths = lengths;
  p.counts = counts;
  p.status = dev_status;
  p.part_o = static_cast<float*>(workspace);
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.T = T;
  p.D = D;
  p.page = page;
  p.page_shift = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  p.width = table_width;
  p.num_pages = num_pages;
  p.bf16 = dtype == TA_DTYPE_BF16;
  p.causal = causal != 0;
  p.group = Hq / Hkv;
  p.group_recip = ta::kv8::group_reciprocal(p.group);
  p.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  if (ta::kv8::uses_chunk(p.group * T, D))
    return launched(ta::kv8::launch_chunk(p, sms, static_cast<cudaStream_t>(stream)),
                    "cache attention launch failed");
  CUtensorMap map_k, map_v;
  const int box = page < ta::kv8::kKeysPerStep ? page : ta::kv8::kKeysPerStep;
  const int64_t planes = static_cast<int64_t>(num_pages) * Hkv;
  if ((rc = make_pages_map(&map_k, k_pages, D, page, planes, box)) ||
      (rc = make_pages_map(&map_v, v_pages, D, page, planes, box)))
    return rc;
  return launched(ta::kv8::launch_attend(p, map_k, map_v, sms, static_cast<cudaStream_t>(stream)),
                  "cache attention launch failed");
}

}  // extern "C"
