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
// several heads (they depend on the position only). Measured: 8 x 4096 tokens, 32 + 32 heads of 128:
// 161 us, 6.66 TB/s, a copy's rate; 32 single tokens, 32 + 8 heads: 2.3 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "overlapped_launch.cuh"
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

// Token and slot of a thread: a block covers the whole tokens that fit its threads.
struct Place {
  int b, s, slot;
  bool ok;
};
__device__ __forceinline__ Place place_of(const RotaryParams& p, int n_slots) {
  const int per_block = max(1, kThreads / n_slots);
  const int slots_here = min(n_slots, kThreads);  // n_slots > kThreads: only value by value
  const int local = threadIdx.x / slots_here;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * per_block + local;
  const int64_t tokens = static_cast<int64_t>(p.B) * p.S;
  Place at;
  at.slot = threadIdx.x - local * slots_here;
  at.ok = local < per_block && token < tokens;
  if (tokens <= 0xffffffffll) {  // a 64-bit division costs as much as the rotation
    at.b = static_cast<uint32_t>(token) / static_cast<uint32_t>(p.S);
    at.s = static_cast<int>(static_cast<uint32_t>(token) - static_cast<uint32_t>(at.b) * p.S);
  } else {
    at.b = static_cast<int>(token / p.S);
    at.s = static_cast<int>(token - static_cast<int64_t>(at.b) * p.S);
  }
  return at;
}

template <bool BF16>
__device__ __forceinline__ uint32_t turned(uint32_t a, uint32_t b, float c0, float c1, float s0,
                                           float s1) {  // a cos + b sin of two lanes
  const float2 x = unpack2<BF16>(a), y = unpack2<BF16>(b);
  return pack2<BF16>(fmaf(x.x, c0, y.x * s0), fmaf(x.y, c1, y.y * s1));
}

// W values an access. A token's head has n_slots slots, at most kThreads: with the half layout half/W
// slots of W pairs (two vectors each), interleaved 2 half/W slots of W/2 pairs (one vector), then
// one slot for each W copied dims. Thread = (token, slot), blockIdx.y = group of heads_per_thread
// heads; consecutive threads cover consecutive bytes of one head's tokens. The loads of kAhead
// heads are issued before their stores (which may be to the same memory, so the compiler cannot).
template <int W>
struct alignas(2 * W) Vec {
  uint32_t w[W / 2];
};
template <bool BF16, bool INTERLEAVED, int W>
__global__ void __launch_bounds__(kThreads)
    rotary_vector_kernel(const RotaryParams p, int n_slots, int heads_per_thread) {
  constexpr int kAhead = 4;
  using V = Vec<W>;
  wait_for_stream();
  const Place at = place_of(p, n_slots);
  if (!at.ok) return;
  const int heads = p.t[0].heads + p.t[1].heads;
  const int h0 = blockIdx.y * heads_per_thread;
  const int h1 = min(heads, h0 + heads_per_thread);
  constexpr int kPairs = INTERLEAVED ? W / 2 : W;
  const int turning = p.half / kPairs;
  const bool turns = at.slot < turning;
  const int d = turns ? at.slot * W : 2 * p.half + (at.slot - turning) * W;
  V va[kAhead], vb[kAhead];
  uint16_t* y[kAhead];
  auto load = [&](int h) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (h + k >= h1) break;
      const HeadAt x = head_at(p, h + k, at.b, at.s);
      y[k] = x.y + d;
      va[k] = *reinterpret_cast<const V*>(x.x + d);
      if (!INTERLEAVED && turns) vb[k] = *reinterpret_cast<const V*>(x.x + p.half + d);
    }
  };
  load(h0);  // on their way while the angles are computed
  float c[kPairs], sn[kPairs];
  if (turns) {
    const double position = position_of(p, at.b, at.s);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) turn_of(p, position, at.slot * kPairs + i, c[i], sn[i]);
  }
  for (int h = h0; h < h1; h += kAhead) {
    if (h > h0) load(h);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (h + k >= h1) break;
      if (!turns) {
        *reinterpret_cast<V*>(y[k]) = va[k];
        continue;
      }
      V r;
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          const float2 v = unpack2<BF16>(va[k].w[i]);
          r.w[i] = pack2<BF16>(fmaf(v.x, c[i], -v.y * sn[i]), fmaf(v.y, c[i], v.x * sn[i]));
        }
      } else {
        V q;
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          const uint32_t a = va[k].w[i], b = vb[k].w[i];
          r.w[i] = turned<BF16>(a, b, c[2 * i], c[2 * i + 1], -sn[2 * i], -sn[2 * i + 1]);
          q.w[i] = turned<BF16>(b, a, c[2 * i], c[2 * i + 1], sn[2 * i], sn[2 * i + 1]);
        }
        *reinterpret_cast<V*>(y[k] + p.half) = q;
      }
      *reinterpret_cast<V*>(y[k]) = r;
    }
  }
}

// Any sizes, strides and alignment: thread = (token, pair or copied dim).
template <bool BF16>
__global__ void __launch_bounds__(kThreads)
    rotary_scalar_kernel(const RotaryParams p, int n_slots, int heads_per_thread) {
  wait_for_stream();
  const Place at = place_of(p, n_slots);
  if (!at.ok) return;
  const int b = at.b, s = at.s;
  const int h0 = blockIdx.y * heads_per_thread;
  const int h1 = min(p.t[0].heads + p.t[1].heads, h0 + heads_per_thread);
  for (int slot = at.slot; slot < n_slots; slot += kThreads) {
    if (slot >= p.half) {
      const int d = p.half + slot;
      for (int h = h0; h < h1; ++h) {
        const HeadAt x = head_at(p, h, b, s);
        x.y[d] = x.x[d];
      }
      continue;
    }
    float c, sn;
    turn_of(p, position_of(p, b, s), slot, c, sn);
    const int da = p.interleaved ? 2 * slot : slot;
    const int db = p.interleaved ? 2 * slot + 1 : p.half + slot;
    for (int h = h0; h < h1; ++h) {
      const HeadAt x = head_at(p, h, b, s);
      const float2 v = unpack2<BF16>(static_cast<uint32_t>(x.x[da]) |
                                     (static_cast<uint32_t>(x.x[db]) << 16));
      const uint32_t r = pack2<BF16>(fmaf(v.x, c, -v.y * sn), fmaf(v.y, c, v.x * sn));
      x.y[da] = static_cast<uint16_t>(r);
      x.y[db] = static_cast<uint16_t>(r >> 16);
    }
  }
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, int alignment, int sm_count, cudaStream_t stream) {
  // The widest access that alignment and sizes allow, while a block's threads hold a token's slots.
  // Measured, 9 x 2238 tokens of 9 heads, D 80, 40 dims rotated by halves of 20: one value an access
  // 63.8 us, 2 25.0, 4 16.7 (a floor of 8.8).
  int width = 8, n_slots = 0;
  for (; width > 1; width /= 2) {
    const int turning = p.interleaved ? 2 * p.half : p.half;
    n_slots = turning / width + (p.D - 2 * p.half) / width;
    if (alignment % (2 * width) == 0 && turning % width == 0 && p.D % width == 0 && n_slots <= kThreads) break;
  }
  if (width == 1) n_slots = p.D - p.half;
  const int heads = p.t[0].heads + p.t[1].heads;
  const int per_block = kThreads / n_slots > 1 ? kThreads / n_slots : 1;
  const int64_t blocks = (static_cast<int64_t>(p.B) * p.S + per_block - 1) / per_block;
  if (blocks == 0 || heads == 0) return cudaSuccess;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  // Heads per thread: as many as leave a full wave of resident threads (more heads spread the
  // cost of cos and sin, fewer fill the GPU when tokens are few), 16 at most.
  int hpt = 16;
  const int64_t want = static_cast<int64_t>(sm_count) * (2048 / kThreads);
  while (hpt > 1 && blocks * ((heads + hpt - 1) / hpt) < want) hpt /= 2;
  while ((heads + hpt - 1) / hpt > 65535) hpt *= 2;
  const dim3 grid(static_cast<unsigned>(blocks), (heads + hpt - 1) / hpt);
  const auto launch = [&](auto kernel) {
    return launch_overlapped(kernel, grid, kThreads, 0, stream, p, n_slots, hpt);
  };
  const auto launch_vector = [&](auto w) {
    constexpr int W = decltype(w)::value;
    if (p.interleaved)
      return p.bf16 ? launch(rotary_vector_kernel<true, true, W>) : launch(rotary_vector_kernel<false, true, W>);
    return p.bf16 ? launch(rotary_vector_kernel<true, false, W>) : launch(rotary_vector_kernel<false, false, W>);
  };
  if (width == 8) return launch_vector(std::integral_constant<int, 8>());
  if (width == 4) return launch_vector(std::integral_constant<int, 4>());
  if (width == 2) return launch_vector(std::integral_constant<int, 2>());
  return p.bf16 ? launch(rotary_scalar_kernel<true>) : launch(rotary_scalar_kernel<false>);
}

}  // namespace ta
