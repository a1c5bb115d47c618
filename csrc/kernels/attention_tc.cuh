// Shared parts of the tensor-core attention kernels (forward and backward).
#pragma once

#include <algorithm>
#include <cmath>

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

// Near zero tanh(x) = x P(x^2), coefficients fitted (least squares, reweighted towards the
// largest error): three on |x| <= 0.3 to an absolute error of 1.7e-7, five on |x| <= 0.6 to 3e-8.
constexpr float kTanhNear = 0.3f, kTanhMid = 0.6f;
constexpr float kTanhPoly3[3] = {0.99999601f, -0.33297479f, 0.1252259f};
constexpr float kTanhPoly5[5] = {0.99999964f, -0.33331209f, 0.13299210f, -0.05169674f, 0.014976959f};

// Score constants of a launch, computed on the host: operands from the constant bank.
struct ScoreScale {
  float c;        // plain: scale * log2 e
  float cap_in;   // capped: 2 log2 e * scale / cap
  float cap_out;  // capped: cap * log2 e
  float cap_inv;  // capped: 1 / cap_out
  // A masked score of the backward pass.  Under a cap it is finite, and so is the square of masked * cap_inv in the
  // factor 1 - tanh^2, which a weight of zero then makes zero; the weight is zero for every accepted cap (from 1e-12 on).
  float masked;
  float near, mid;          // capped: largest raw scores of the polynomials, -1: not used
  float poly3[3], poly5[5];  // capped: the polynomials for raw scores, times cap_out
  // In double, as powers of scale / cap leave the range of fp32 for caps that are accepted.
  static ScoreScale of(const AttnParams& p) {
    constexpr double most = 3.4028234663852886e38;  // of fp32
    constexpr double square = 1e18;                 // what the polynomials can square
    ScoreScale s{};
    s.c = p.scale * kLog2e;
    s.masked = -INFINITY;
    if (p.cap > 0.f) {
      const double k = static_cast<double>(p.scale) / p.cap, out = static_cast<double>(p.cap) * kLog2e;
      s.cap_out = static_cast<float>(out);
      s.cap_in = static_cast<float>(std::min(2. * kLog2e * k, most));
      s.cap_inv = static_cast<float>(1. / out);
      s.masked = static_cast<float>(-std::min(1e15, 1e18 * out));
      s.near = static_cast<float>(std::min(kTanhNear / k, square));
      s.mid = static_cast<float>(std::min(kTanhMid / k, square));
      double f = k * out;
      for (int i = 0; i < 5; ++i, f *= k * k) {
        if (i < 3) s.poly3[i] = static_cast<float>(std::min(std::max(kTanhPoly3[i] * f, -most), most));
        s.poly5[i] = static_cast<float>(std::min(std::max(kTanhPoly5[i] * f, -most), most));
        if (f > 1e38 && i < 3) s.near = -1.f;
        if (f > 1e38) s.mid = -1.f;
      }
    }
    return s;
  }
};

// What a launch does to its scores; kCapped covers capped scores with and without a bias.
enum Scores : int { kPlain = 0, kBiased = 1, kCapped = 2 };

inline Scores scores_of(const AttnParams& p) { return p.cap > 0.f ? kCapped : (p.slopes != nullptr ? kBiased : kPlain); }

// Capped base-2 scores of N raw ones in place.
template <int N>
__device__ __forceinline__ void cap_scores(float (&s)[N], const ScoreScale& sc) {
  float far = 0.f;
#pragma unroll
  for (int c = 0; c < N; c += 2) far = fmaxf(far, fmaxf(fabsf(s[c]), fabsf(s[c + 1])));
  // Scores well below the cap, the common case: four or six FMA-pipe operations, two scores at
  // a time, in place of two MUFU ones, of which an SM has 16 a clock.
  if (__all_sync(0xffffffffu, far <= sc.near)) {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const Pair x(s[c], s[c + 1]), u = mul2(x, x);
      Pair y = fma2(u, Pair(sc.poly3[2], sc.poly3[2]), Pair(sc.poly3[1], sc.poly3[1]));
      y = fma2(u, y, Pair(sc.poly3[0], sc.poly3[0]));
      mul2(x, y).split(s[c], s[c + 1]);
    }
  } else if (__all_sync(0xffffffffu, far <= sc.mid)) {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const Pair x(s[c], s[c + 1]), u = mul2(x, x);
      Pair y = fma2(u, Pair(sc.poly5[4], sc.poly5[4]), Pair(sc.poly5[3], sc.poly5[3]));
      y = fma2(u, y, Pair(sc.poly5[2], sc.poly5[2]));
      y = fma2(u, y, Pair(sc.poly5[1], sc.poly5[1]));
      y = fma2(u, y, Pair(sc.poly5[0], sc.poly5[0]));
      mul2(x, y).split(s[c], s[c + 1]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) s[c] = tanh_ex2(s[c] * sc.cap_in) * sc.cap_out;
  }
}

// s = s * factor - slope |d0 + c| for N scores whose distances are d0, d0 + 1, ...  `slope`: of the
// bias times log2 e; `behind`: no distance is positive.
template <int N>
__device__ __forceinline__ void bias_scores(float (&s)[N], float factor, float slope, float d0, bool behind) {
  if (behind) {
    const float base = slope * d0;  // the column is an immediate operand
#pragma unroll
    for (int c = 0; c < N; ++c) s[c] = fmaf(s[c], factor, fmaf(slope, static_cast<float>(c), base));
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) s[c] = fmaf(s[c], factor, -slope * fabsf(d0 + c));
  }
}

// Clears the rows of an operand tile that `dead` names: sub-tiles of 64 columns and ROWS rows.
template <int ROWS>
__device__ __forceinline__ void zero_dead_rows(char* tile, int subtiles, const uint32_t (&dead)[ROWS / 32], int lane) {
#pragma unroll 1
  for (int r = 0; r < ROWS; ++r) {
    if (!((dead[r >> 5] >> (r & 31)) & 1u)) continue;
    for (int i = lane; i < subtiles * 8; i += 32)
      *reinterpret_cast<uint4*>(tile + (i >> 3) * (ROWS * 128) + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
}
// Where 16-byte piece `piece` of row `row` lies in a 64-column tile (128-byte swizzle).
__device__ __forceinline__ char* swizzled(char* tile, int row, int piece) {
  return tile + row * 128 + ((piece ^ (row & 7)) << 4);
}

// 32 fp32 values as four 16-byte pieces of T, from piece `first` on, into a staged row; with
// LOW also what the rounding took, into the same place of a second tile.
template <typename T, bool LOW>
__device__ __forceinline__ void stage_row(char* tile, char* low, int row, int first, const float (&o)[32]) {
#pragma unroll
  for (int e = 0; e < 32; e += 8) {
    uint4 w;
    uint32_t* wp = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
    for (int k = 0; k < 4; ++k) wp[k] = pack2<T>(o[e + 2 * k], o[e + 2 * k + 1]);
    *reinterpret_cast<uint4*>(swizzled(tile, row, first + e / 8)) = w;
    if (LOW) {
      const T* hi = reinterpret_cast<const T*>(&w);
      uint4 v;
      uint32_t* vp = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        vp[k] = pack2<T>(o[e + 2 * k] - to_f32<T>(hi[2 * k]), o[e + 2 * k + 1] - to_f32<T>(hi[2 * k + 1]));
      *reinterpret_cast<uint4*>(swizzled(low, row, first + e / 8)) = v;
    }
  }
}

__device__ __forceinline__ bool any_bit(const uint4& v) { return (v.x | v.y | v.z | v.w) != 0u; }

}  // namespace bitscom_b200
