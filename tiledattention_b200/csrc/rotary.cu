// Rotary positions for q and k: pair i of a head at position n turns by the angle
// n * inv_freq[i], times `magnitude`; the gradient is the same kernel turning the other way.
//
//   (a, b) -> m * (a cos - b sin, b cos + a sin)
//
// Pair i is dims (i, half + i), or (2i, 2i + 1) when interleaved; dims from 2 * half on are
// copied. HBM-bound: every value is read and written once.
//
// The angle is reduced in double: turns = n * inv_freq / (2 pi), minus the nearest whole
// number, which at position 2^20 leaves an error near 2^-33 turns where a float product would
// leave 2^-4 radians. The fraction goes to sincospif in float. That costs about 50
// instructions a pair, so a thread computes its pairs' cos and sin once and applies them to
// several heads (they depend on the position only).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "rotary.h"

namespace ta {
namespace {

constexpr int kThreads = 256;

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
  }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ double position_of(const RotaryParams& p, int b, int s) {
  const int64_t at = b * p.pos_sb + s * p.pos_ss;
  return p.pos64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[at])
                 : static_cast<double>(static_cast<const int32_t*>(p.positions)[at]);
}

// cos and sin of position * inv_freq, times the magnitude; sin negated for the inverse.
__device__ __forceinline__ void turn_of(const RotaryParams& p, double position, int pair,
                                        float& c, float& s) {
  constexpr double kInvTwoPi = 0.15915494309189533577;
  const double turns = position * (p.inv_freq[pair] * kInvTwoPi);
  const float frac = static_cast<float>(turns - rint(turns));  // in [-1/2, 1/2]
  sincospif(2.f * frac, &s, &c);
  c *= p.magnitude;
  s *= p.inverse ? -p.magnitude : p.magnitude;
}

// Head h of the tensors taken together: its tensor and base pointers at (b, s).
struct HeadAt {
  const uint16_t* x;
  uint16_t* y;
};
__device__ __forceinline__ HeadAt head_at(const RotaryParams& p, int h, int b, int s) {
  const bool second = h >= p.t[0].heads;
  const RotaryTensor& t = p.t[second ? 1 : 0];
  const int64_t hh = second ? h - p.t[0].heads : h;
  return {static_cast<const uint16_t*>(t.x) + b * t.x_sb + hh * t.x_sh + s * t.x_ss,
          static_cast<uint16_t*>(t.y) + b * t.y_sb + hh * t.y_sh + s * t.y_ss};
}

// 16-byte path. A token's head has n_slots slots: with the half layout half/8 slots of 8 pairs
// (two vectors each), interleaved half/4 slots of 4 pairs (one vector), then one slot for
// each 8 copied dims. Thread = (token, slot), blockIdx.y = group of heads_per_thread heads;
// consecutive threads cover consecutive bytes of one head's tokens.
template <bool BF16, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads)
    rotary_vector_kernel(const RotaryParams p, int n_slots, int heads_per_thread) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t token = id / n_slots;
  const int slot = static_cast<int>(id - token * n_slots);
  if (token >= static_cast<int64_t>(p.B) * p.S) return;
  const int b = static_cast<int>(token / p.S);
  const int s = static_cast<int>(token - static_cast<int64_t>(b) * p.S);
  const int heads = p.t[0].heads + p.t[1].heads;
  const int h0 = blockIdx.y * heads_per_thread;
  const int h1 = min(heads, h0 + heads_per_thread);
  constexpr int kPairs = INTERLEAVED ? 4 : 8;
  const int turning = p.half / kPairs;
  if (slot >= turning) {
    const int d = 2 * p.half + (slot - turning) * 8;
    for (int h = h0; h < h1; ++h) {
      const HeadAt at = head_at(p, h, b, s);
      *reinterpret_cast<uint4*>(at.y + d) = *reinterpret_cast<const uint4*>(at.x + d);
    }
    return;
  }
  float c[kPairs], sn[kPairs];
  const double position = position_of(p, b, s);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) turn_of(p, position, slot * kPairs + i, c[i], sn[i]);
  const int d = slot * 8;
  if constexpr (INTERLEAVED) {
#pragma unroll 4
    for (int h = h0; h < h1; ++h) {
      const HeadAt at = head_at(p, h, b, s);
      const uint4 v = *reinterpret_cast<const uint4*>(at.x + d);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = unpack2<BF16>(w[i]);
        r[i] = pack2<BF16>(a.x * c[i] - a.y * sn[i], a.y * c[i] + a.x * sn[i]);
      }
      *reinterpret_cast<uint4*>(at.y + d) = make_uint4(r[0], r[1], r[2], r[3]);
    }
  } else {
#pragma unroll 2
    for (int h = h0; h < h1; ++h) {
      const HeadAt at = head_at(p, h, b, s);
      const uint4 va = *reinterpret_cast<const uint4*>(at.x + d);
      const uint4 vb = *reinterpret_cast<const uint4*>(at.x + p.half + d);
      const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
      uint32_t ra[4], rb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = unpack2<BF16>(wa[i]), e = unpack2<BF16>(wb[i]);
        const float c0 = c[2 * i], c1 = c[2 * i + 1], s0 = sn[2 * i], s1 = sn[2 * i + 1];
        ra[i] = pack2<BF16>(a.x * c0 - e.x * s0, a.y * c1 - e.y * s1);
        rb[i] = pack2<BF16>(e.x * c0 + a.x * s0, e.y * c1 + a.y * s1);
      }
      *reinterpret_cast<uint4*>(at.y + d) = make_uint4(ra[0], ra[1], ra[2], ra[3]);
      *reinterpret_cast<uint4*>(at.y + p.half + d) = make_uint4(rb[0], rb[1], rb[2], rb[3]);
    }
  }
}

// Any sizes, strides and alignment: thread = (token, pair or copied dim).
template <bool BF16>
__global__ void __launch_bounds__(kThreads)
    rotary_scalar_kernel(const RotaryParams p, int n_slots, int heads_per_thread) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t token = id / n_slots;
  const int slot = static_cast<int>(id - token * n_slots);
  if (token >= static_cast<int64_t>(p.B) * p.S) return;
  const int b = static_cast<int>(token / p.S);
  const int s = static_cast<int>(token - static_cast<int64_t>(b) * p.S);
  const int h0 = blockIdx.y * heads_per_thread;
  const int h1 = min(p.t[0].heads + p.t[1].heads, h0 + heads_per_thread);
  if (slot >= p.half) {
    const int d = p.half + slot;
    for (int h = h0; h < h1; ++h) {
      const HeadAt at = head_at(p, h, b, s);
      at.y[d] = at.x[d];
    }
    return;
  }
  float c, sn;
  turn_of(p, position_of(p, b, s), slot, c, sn);
  const int da = p.interleaved ? 2 * slot : slot;
  const int db = p.interleaved ? 2 * slot + 1 : p.half + slot;
  for (int h = h0; h < h1; ++h) {
    const HeadAt at = head_at(p, h, b, s);
    const float2 v = unpack2<BF16>(static_cast<uint32_t>(at.x[da]) |
                                   (static_cast<uint32_t>(at.x[db]) << 16));
    const uint32_t r = pack2<BF16>(v.x * c - v.y * sn, v.y * c + v.x * sn);
    at.y[da] = static_cast<uint16_t>(r);
    at.y[db] = static_cast<uint16_t>(r >> 16);
  }
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, bool vector, int sm_count, cudaStream_t stream) {
  const int pairs = vector ? (p.interleaved ? 4 : 8) : 1;
  const int n_slots = p.half / pairs + (p.D - 2 * p.half) / (vector ? 8 : 1);
  const int heads = p.t[0].heads + p.t[1].heads;
  const int64_t blocks =
      (static_cast<int64_t>(p.B) * p.S * n_slots + kThreads - 1) / kThreads;
  if (blocks == 0 || heads == 0) return cudaSuccess;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  // Heads per thread: as many as leave two full waves of resident threads (more heads spread
  // the cost of cos and sin, fewer fill the GPU when tokens are few), 16 at most.
  int hpt = 16;
  const int64_t want = 2ll * sm_count * (2048 / kThreads);
  while (hpt > 1 && blocks * ((heads + hpt - 1) / hpt) < want) hpt /= 2;
  while ((heads + hpt - 1) / hpt > 65535) hpt *= 2;
  const dim3 grid(static_cast<unsigned>(blocks), (heads + hpt - 1) / hpt);
  if (vector) {
    if (p.interleaved) {
      if (p.bf16) rotary_vector_kernel<true, true><<<grid, kThreads, 0, stream>>>(p, n_slots, hpt);
      else rotary_vector_kernel<false, true><<<grid, kThreads, 0, stream>>>(p, n_slots, hpt);
    } else {
      if (p.bf16) rotary_vector_kernel<true, false><<<grid, kThreads, 0, stream>>>(p, n_slots, hpt);
      else rotary_vector_kernel<false, false><<<grid, kThreads, 0, stream>>>(p, n_slots, hpt);
    }
  } else {
    if (p.bf16) rotary_scalar_kernel<true><<<grid, kThreads, 0, stream>>>(p, n_slots, hpt);
    else rotary_scalar_kernel<false><<<grid, kThreads, 0, stream>>>(p, n_slots, hpt);
  }
  return cudaGetLastError();
}

}  // namespace ta
