// Internal interface of the rotary position kernel (rotary.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ta {

// One of the (up to two) tensors [B, H, S, D] turned by the same angles.
struct RotaryTensor {
  const void* x;
  void* y;
  int64_t x_sb, x_sh, x_ss;  // element strides (dim stride 1)
  int64_t y_sb, y_sh, y_ss;
  int heads;
};

struct RotaryParams {
  RotaryTensor t[2];        // t[1].heads == 0: one tensor only
  const void* positions;    // int32 or int64, element strides below
  int64_t pos_sb, pos_ss;
  const double* inv_freq;   // radians per position of pair i, [half]
  int B, S, D;
  int half;                 // pairs; the first 2 * half dims turn, the others are copied
  int pos64, interleaved, inverse, bf16;
  float magnitude;
};

// alignment: bytes (a power of two up to 16) that divide all bases and outer strides.
cudaError_t launch_rotary(const RotaryParams& p, int alignment, int sm_count, cudaStream_t stream);

}  // namespace ta
