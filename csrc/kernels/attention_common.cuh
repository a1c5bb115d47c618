// Device helpers shared by the attention kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention.h"

namespace bitscom_b200 {

constexpr float kLog2e = 1.4426950408889634f;

// The keys that row i of batch entry b sees.
__device__ __forceinline__ int2 attn_row_range(const AttnParams& p, int b, int i) {
  if (p.plan.range != nullptr) return p.plan.range[static_cast<int64_t>(b) * ((p.sq + kAttnTile - 1) / kAttnTile * kAttnTile) + i];
  if (!p.causal) return make_int2(0, p.sk);
  return make_int2(0, max(0, i + p.sk - p.sq + 1));
}

// Bounds over row tile t: x = min lo, y = max hi, z = max lo, w = min hi (see PlanView).
__device__ __forceinline__ int4 attn_tile_range(const AttnParams& p, int b, int t) {
  if (p.plan.tile != nullptr) {
    const int nq = (p.sq + kAttnTile - 1) / kAttnTile;
    return p.plan.tile[static_cast<int64_t>(b) * nq + t];
  }
  if (!p.causal) return make_int4(0, p.sk, 0, p.sk);
  const int first = t * kAttnTile, last = min(first + kAttnTile, p.sq) - 1;
  return make_int4(0, max(0, last + p.sk - p.sq + 1), 0, max(0, first + p.sk - p.sq + 1));
}

// Bit r: row r of row tile t sees no key.
__device__ __forceinline__ uint4 attn_tile_qdead(const AttnParams& p, int b, int t) {
  if (p.plan.qdead != nullptr) return p.plan.qdead[static_cast<int64_t>(b) * ((p.sq + kAttnTile - 1) / kAttnTile) + t];
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  const int none = p.causal ? p.sq - p.sk - t * kAttnTile : 0;  // rows before the first key
  if (none > 0)
    for (int i = 0; i < 4; ++i) w[i] = none >= 32 * (i + 1) ? 0xffffffffu : (none > 32 * i ? (1u << (none - 32 * i)) - 1u : 0u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Whether row i sees no key, and whether key j is padding that no row sees.
__device__ __forceinline__ bool attn_row_dead(const AttnParams& p, int b, int i) {
  const int2 r = attn_row_range(p, b, i);
  return r.y <= r.x;
}

__device__ __forceinline__ bool attn_key_dead(const AttnParams& p, int b, int j) {
  if (p.plan.kdead == nullptr) return false;
  const int nk = (p.sk + kAttnTile - 1) / kAttnTile;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&p.plan.kdead[static_cast<int64_t>(b) * nk + j / kAttnTile]);
  return (w[j % kAttnTile / 32] >> (j % 32)) & 1u;
}

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

}  // namespace bitscom_b200
