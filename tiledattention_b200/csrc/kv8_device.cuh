// What the kernels that attend over the 8-bit cache share on the device (sdpa_kv8.cu for few query
// rows, sdpa_kv8_chunk.cu for many): 16-bit values, a batch's line of work.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kv8.h"
#include "overlapped_launch.cuh"
#include "sm100_ptx.cuh"
#include "tiledattention_b200.h"

namespace ta {
namespace kv8 {

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack16(uint32_t w, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
  uint32_t r;
  if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float pow2f(int e) {
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// What takes a row of q whose largest magnitude is amax < 2^(ex + 15) into [2^14, 2^15). A row with an
// infinity becomes NaN: so are all its softmax weights (its scores are infinities and NaN, but all of them may
// be -inf, which alone would look like a row without keys).
__device__ __forceinline__ float row_factor(float amax, int ex) {
  return amax == INFINITY ? __int_as_float(0x7fffffff) : pow2f(-ex);
}

// log2 and reciprocal of a value scale as it is stored, its exponent held in range: exact for powers
// of two, which is what this library writes.
struct ValueScale {
  float e, back;
};
__device__ __forceinline__ ValueScale value_scale(uint32_t scale_bits) {
  const int e = stored_exponent(scale_bits);
  ValueScale r{static_cast<float>(e), pow2f(-e)};
  if (scale_bits & 0x7fffffu) {
    const float m = __uint_as_float(0x3f800000u | (scale_bits & 0x7fffffu));
    r.e += __log2f(m);
    r.back = __fdividef(r.back, m);
  }
  return r;
}

// Natural-log log-sum-exp of a row from its maximum (log2) and sum; -inf without a key.
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : (fmaxf(m, -3.4e38f) + log2f(l)) * 0.69314718055994531f;
}

__device__ __forceinline__ SeqExtent extent_of(const AttendParams& p, int b) {
  return checked_extent(p.lengths[b], p.counts ? p.counts[b] : p.T, p.T,
                        static_cast<int64_t>(p.width) * p.page);
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// An exclusive sum over n items by one block of WARPS warps; `work(i)`: item i's. Every thread gets
// the total and the work before its own share [i0, i1) of the items.
struct Scan {
  int64_t total, mine;
  int i0, i1;
};
template <int WARPS, class F>
__device__ __forceinline__ Scan scan_items(int n, int64_t* s_warp, F work) {
  Scan r;
  const int share = (n + WARPS * 32 - 1) / (WARPS * 32);
  r.i0 = min(n, static_cast<int>(threadIdx.x) * share);
  r.i1 = min(n, r.i0 + share);
  int64_t sum = 0;
  for (int i = r.i0; i < r.i1; ++i) sum += work(i);
  int64_t incl = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, d);
    if ((threadIdx.x & 31) >= d) incl += up;
  }
  if ((threadIdx.x & 31) == 31) s_warp[threadIdx.x >> 5] = incl;
  __syncthreads();
  int64_t before = 0;
  r.total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 5)) before += s_warp[w];
    r.total += s_warp[w];
  }
  r.mine = before + incl - sum;
  return r;
}

// Records a sequence whose length or count is out of range.
__device__ __forceinline__ void report_extent(const AttendParams& p, const SeqExtent& e) {
  if (e.bad && blockIdx.x == 0 && p.status) atomicOr(p.status, TA_DEVSTAT_BAD_LENGTH);
}

}  // namespace kv8
}  // namespace ta
