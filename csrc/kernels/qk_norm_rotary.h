// Norm of every query and key head and rotation by position, one pass.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "launchers.h"

namespace bitscom_b200 {

// [B, S, H, D] with D contiguous; strides in elements.
struct RotaryTensor {
  void* ptr;
  int64_t sb, ss, sh;
  int h;
};

struct RotaryParams {
  RotaryTensor q, k;        // inputs
  RotaryTensor oq, ok;      // outputs (forward) or dx (backward)
  RotaryTensor gq, gk;      // output gradients (backward)
  const float* wq;          // [D] gains, null for ones
  const float* wk;
  const double* freq;       // [rotated / 2]
  const void* positions;    // int32 or int64, null: 0, 1, ...
  int pos_bytes;
  int64_t pos_sb, pos_ss;
  float* partial;           // [blocks][2][D] sums of the gains' gradients (backward), null: not wanted
  int64_t tokens;           // B * S, below 2^31
  unsigned s;
  int d, rotated, interleaved;
  float eps;
  DType dt;
};

namespace launch {

constexpr int kRotaryMaxDim = 256;

// Blocks of a backward launch, and so rows of `partial`.
int qk_norm_rotary_blocks(const RotaryParams& p, int sms);
void qk_norm_rotary_forward(const RotaryParams& p, int sms, cudaStream_t s);
// dw: [2][D] sums of `partial` over the blocks.
void qk_norm_rotary_backward(const RotaryParams& p, int sms, float* dw, cudaStream_t s);

}  // namespace launch
}  // namespace bitscom_b200
