// Shared parts of the tensor-core attention kernels (forward and backward).
#pragma once

#include "attention_common.cuh"
#include "tcgen05.cuh"

namespace bitscom_b200 {

// fp16 products take the probabilities times 2^10, so that those below 2^-14 of
// the largest keep their 11 bits; bf16 has the range of fp32.
template <typename T>
constexpr float prob_shift() { return std::is_same<T, __half>::value ? 10.f : 0.f; }

// tanh(x) = 1 - 2 / (1 + e^2x): two MUFU operations, absolute error about 2^-23,
// and right at both ends (e^2x = inf, 0).
__device__ __forceinline__ float tanh_ex2(float x2log2e) { return fmaf(-2.f, rcp(1.f + ex2(x2log2e)), 1.f); }

// Score constants of a launch and head.
struct ScoreScale {
  float c;       // plain: scale * log2 e
  float cap_in;  // capped: 2 log2 e * scale / cap
  float cap_out; // capped: cap * log2 e
  float slope;   // distance: slope * log2 e
  __device__ static ScoreScale of(const AttnParams& p, int h) {
    ScoreScale s;
    s.c = p.scale * kLog2e;
    s.cap_in = p.cap > 0.f ? 2.f * kLog2e * p.scale / p.cap : 0.f;
    s.cap_out = p.cap * kLog2e;
    s.slope = p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.f;
    return s;
  }
};

// One 128 x 128 (or narrower) operand tile: sub-tiles of 64 columns.
__device__ __forceinline__ void zero_dead_rows(char* tile, int subtiles, const uint4& dead, int lane) {
  const uint32_t w[4] = {dead.x, dead.y, dead.z, dead.w};
  for (int r = 0; r < kAttnTile; ++r) {
    if (!((w[r >> 5] >> (r & 31)) & 1u)) continue;
    for (int i = lane; i < subtiles * 8; i += 32)
      *reinterpret_cast<uint4*>(tile + (i >> 3) * (kAttnTile * 128) + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
}

__device__ __forceinline__ bool any_bit(const uint4& v) { return (v.x | v.y | v.z | v.w) != 0u; }

}  // namespace bitscom_b200
