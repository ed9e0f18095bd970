// The paged 8-bit key/value cache: what the kernels that write it (kv8_append.cu) and read it
// (sdpa_kv8*.cu) share. Host-callable parts are checked on the CPU (tests/native/kv8_check.cu).
//
// Pages [P, Hkv, page, D] of e4m3, D a multiple of 16 up to 256, page 16, 32, 64 or 128; one
// float32 scale for each (page, head). What is written here has scales 2^e, e in [kScaleExpMin,
// kScaleExpMax]: powers of two cost an e4m3 value nothing (its own exponent does the rest) and make
// every product with a scale exact. Caches made elsewhere may have any scale of that range. The range
// keeps 2^(difference of two exponents) inside float32.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ta {
namespace kv8 {

constexpr int kScaleExpMin = -50;
constexpr int kScaleExpMax = 50;

// Least e with amax <= 448 * 2^e (448 = 1.75 * 2^8 is e4m3's largest value), held in range;
// amax_bits: the bits of a finite float32 >= 0. Zero (a page of zeros) gives the least e.
__host__ __device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23) - 127;
  const int up = (amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0;
  const int need = e - 8 + up;
  return need < kScaleExpMin ? kScaleExpMin : (need > kScaleExpMax ? kScaleExpMax : need);
}

// Exponent of a stored scale, held in range whatever the bits are.
__host__ __device__ __forceinline__ int stored_exponent(uint32_t scale_bits) {
  const int e = static_cast<int>((scale_bits >> 23) & 0xffu) - 127;
  return e < kScaleExpMin ? kScaleExpMin : (e > kScaleExpMax ? kScaleExpMax : e);
}

// A stored scale's bits with its exponent held in range and no sign: itself for every scale from
// 2^kScaleExpMin up to below 2^(kScaleExpMax + 1).
__host__ __device__ __forceinline__ uint32_t held_scale(uint32_t scale_bits) {
  return static_cast<uint32_t>(stored_exponent(scale_bits) + 127) << 23 | (scale_bits & 0x7fffffu);
}

// A page id from the table, or -1 where the slot or the id is outside its range.
__host__ __device__ __forceinline__ int checked_page(const int32_t* table_row, int64_t slot,
                                                     int width, int num_pages) {
  if (slot < 0 || slot >= width) return -1;
  const int id = table_row[slot];
  return id >= 0 && id < num_pages ? id : -1;
}

// Tokens start .. start + count of one sequence that fall into table slot `slot`: rows
// [row0, row1) of its page are written from token t0 on; row0 rows before them are kept.
struct SlotSpan {
  int row0, row1;
  int64_t t0;
};
__host__ __device__ __forceinline__ SlotSpan slot_span(int64_t start, int64_t count, int64_t slot,
                                                       int page) {
  const int64_t first = slot * page;
  const int64_t lo = start > first ? start : first;
  const int64_t hi = start + count < first + page ? start + count : first + page;
  if (hi <= lo) return {0, 0, 0};
  return {static_cast<int>(lo - first), static_cast<int>(hi - first), lo - start};
}

// Pages that T > 0 tokens touch at most.
__host__ __device__ __forceinline__ int64_t slots_for(int T, int page) {
  return (static_cast<int64_t>(T) + page - 2) / page + 1;
}

struct AppendParams {
  const void* x[2];               // k, v: [B, Hkv, T, D], 16-bit
  int64_t sb[2], sh[2], ss[2];    // element strides (dim stride 1)
  uint8_t* pages[2];
  float* scale[2];
  const int32_t* table;           // [B, width] int32, row stride table_stride
  int64_t table_stride;
  const int32_t* starts;          // [B]
  const int32_t* counts;          // [B] or null (all T)
  unsigned int* status;
  int B, Hkv, T, D, page, width, num_pages, bf16;
};

cudaError_t launch_append(const AppendParams& p, cudaStream_t stream);

// Where the chunk kernel's runs cut a block of rows: the block, and the first of the runs that
// share it (-1: nothing to merge).
struct Cut {
  int b, h, rb, first;
};

struct AttendParams {
  const void* q;                  // [B, Hq, T, D], 16-bit
  int64_t q_sb, q_sh, q_ss;
  void* o;
  int64_t o_sb, o_sh, o_ss;
  float* lse;                     // optional [B, Hq, T] contiguous
  const uint8_t* pages[2];
  const float* scale[2];
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;         // [B] tokens in the cache
  const int32_t* counts;          // [B] or null (all T rows are real)
  unsigned int* status;
  float* part_o;                  // partial outputs, maxima and sums (see sdpa_kv8.cu)
  float* part_ml;
  int2* spans;                    // first and last run of a block of rows; (1, 0): none has keys of it
  Cut* cuts;
  int B, Hq, Hkv, T, D, page, page_shift, width, num_pages, bf16, causal;
  int group;                      // Hq / Hkv, at most kMaxGroup
  uint32_t group_recip;           // for group_of
  int row_blocks;                 // blocks of rows (token, head of the group) per kv head
  float scale_log2;               // softmax scale * log2(e)
};

// n / group for 0 <= n < 2^24 by a multiplication (a division costs some thirty instructions in
// each of its many places): recip = ceil(2^32 / group), exact for group <= kMaxGroup = 2^8.
constexpr int kMaxGroup = 256;
__host__ __device__ __forceinline__ uint32_t group_reciprocal(int group) {
  return group == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + group - 1) / group);
}
__host__ __device__ __forceinline__ int divide_by_group(int n, uint32_t recip) {
  return recip == 0 ? n
                    : static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * recip) >> 32);
}
__host__ __device__ __forceinline__ int group_of(const AttendParams& p, int n) {
  return divide_by_group(n, p.group_recip);
}

// Keys of a sequence that its row of token t may see: [0, limit).
__host__ __device__ __forceinline__ int row_limit(int length, int count, int t, int causal) {
  if (t >= count) return 0;
  const int lim = causal ? length - count + t + 1 : length;
  return lim > 0 ? lim : 0;
}

// Length and count of one sequence with every out-of-range value held in range.
struct SeqExtent {
  int length, count;
  bool bad;
};
__host__ __device__ __forceinline__ SeqExtent checked_extent(int length, int count, int T,
                                                             int64_t capacity) {
  SeqExtent e{length, count, false};
  if (e.length < 0) e.length = 0, e.bad = true;
  if (e.length > capacity) e.length = static_cast<int>(capacity), e.bad = true;
  if (e.count < 0) e.count = 0, e.bad = true;
  if (e.count > T) e.count = T, e.bad = true;
  return e;
}

// Tiles of `tile` keys that hold n, for every n >= 0: n + tile - 1 may pass 2^31.
__host__ __device__ __forceinline__ int tiles_for(int n, int tile) {
  return static_cast<int>((static_cast<uint32_t>(n) + static_cast<uint32_t>(tile) - 1u) / static_cast<uint32_t>(tile));
}

// Key tiles of rows [row0, row0 + n) of a sequence's `rows` rows (token, head of the group):
// up to the last key that any of them sees.
__host__ __device__ __forceinline__ int block_tiles(const SeqExtent& e, int rows, uint32_t recip, int row0,
                                                    int n, int causal, int tile) {
  const int end = row0 + n < rows ? row0 + n : rows;
  if (row0 >= end) return 0;
  const int first = divide_by_group(row0, recip), last = divide_by_group(end - 1, recip);
  if (first >= e.count) return 0;
  const int lim = row_limit(e.length, e.count, last < e.count ? last : e.count - 1, causal);
  return tiles_for(lim, tile);
}

// Work of the split kernel is a line of `total` tiles (sequence, then head and row block, then
// keys), cut into `parts` equal runs: run i is [i * total / parts, (i + 1) * total / parts).
__host__ __device__ __forceinline__ int64_t run_begin(int64_t i, int64_t total, int64_t parts) {
  // i total / parts without the 64-bit division where 32 bits do (parts < 2^16)
  const int64_t each = total <= 0xffffffffll ? static_cast<uint32_t>(total) / static_cast<uint32_t>(parts)
                                             : total / parts;
  const uint32_t rest = static_cast<uint32_t>(total - each * parts);
  return i * each + static_cast<uint32_t>(i) * rest / static_cast<uint32_t>(parts);
}
// The run that holds tile w.
__host__ __device__ __forceinline__ int64_t run_of(int64_t w, int64_t total, int64_t parts) {
  return ((w + 1) * parts - 1) / total;
}

// Byte offset in shared memory of 16-byte chunk c of a row of codes, as TMA's 64- and 128-byte
// swizzles lay out boxes of COLS bytes a row: 8 consecutive rows at one chunk fall on
// different banks. Chunks beyond COLS bytes are in the next plane, PLANE bytes on.
template <int COLS, int PLANE>
__host__ __device__ __forceinline__ uint32_t chunk_at(int row, int c) {
  if constexpr (COLS == 64) return row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
  return (c >> 3) * PLANE + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}

// Order of 16 keys in the matrix instructions (see sdpa_kv8.cu): the key at position p of the
// second product's depth, and the key of column n of score tile `half`, which is position
// 4 (n / 2) + 2 half + n % 2. Chosen so that the 8 rows of every ldmatrix phase, of K (the columns of
// one half) and of V (positions 0-7 and 8-15), differ modulo 8: no bank conflicts.
__host__ __device__ __forceinline__ int key_at(int p) {
  return 8 * (p >> 3) + 4 * (((p >> 1) & 1) ^ (p >> 3)) + 2 * ((p >> 2) & 1) + (p & 1);
}
__host__ __device__ __forceinline__ int key_of_column(int n, int half) {
  return key_at(4 * (n >> 1) + 2 * half + (n & 1));
}

// Keys a warp of the split kernel takes a step, which is also the rows of a copied box where the
// page has as many.
constexpr int kKeysPerStep = 32;

// Workspace of the split kernel's partial results for a problem.
size_t attend_workspace_bytes(int B, int Hq, int Hkv, int T, int D, int sm_count);
// map_k, map_v: 3-D maps (D, page, P * Hkv) of the pages' bytes, boxes of 64 (D <= 64, 64-byte
// swizzle) or 128 columns (128-byte swizzle) x min(page, kKeysPerStep) rows.
cudaError_t launch_attend(const AttendParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v,
                          int sm_count, cudaStream_t stream);

// The kernel for many rows (sdpa_kv8_chunk.cu) and its workspace.
size_t chunk_workspace_bytes(int D, int sm_count);
cudaError_t launch_chunk(const AttendParams& p, int sm_count, cudaStream_t stream);

// Which kernel serves `rows` query rows per cache head: see capi_serving.cu.
bool uses_chunk(int rows, int D);

}  // namespace kv8
}  // namespace ta
