// Norm of queries and keys for each head, with the position rotation in the
// same pass; forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps);  n = x r;  y = n w
//   (y1, y2) -> (y1 cos a - y2 sin a, y2 cos a + y1 sin a),  a = position * freq
//   backward: g = dy turned by -a;  dw = sum g n;  dx = r (g w - n mean(g w n))
//
// Bound by memory: each head is read once and written once (backward: x and
// dy read, dx written).  A head's D values lie in 16-byte pieces across a group
// of 8, 16 or 32 lanes, so the norm is a few shuffles; the partner of a pair
// (i, i + rotated / 2) sits in another lane at the same place of its piece, one
// shuffle more.  When a half is not a whole number of pieces, the partners are
// exchanged through shared memory.  Norms, rotations and sums are in fp32, with
// one rounding at the end; the angle is formed and reduced to one turn in fp64
// (a position of 10^6 times a frequency leaves fp32 five digits short), once
// for each token and frequency and then shared by all heads of the token.
//
// The gains' gradients are summed in registers over a block's heads, then over
// the block's groups and over the blocks in a fixed order: no atomics, the same
// bits every time.
#include <cuda_runtime.h>

#include "attention_common.cuh"
#include "qk_norm_rotary.h"

namespace bitscom_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kV = 8;  // values of a lane

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int count, float (&o)[kV]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < kV; ++i) o[i] = to_f32<T>(t[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) o[i] = i < count ? to_f32<T>(p[i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, int count, const float (&v)[kV]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 u;
      T* t = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int i = 0; i < kV; ++i) t[i] = from_f32<T>(v[i]);
      *reinterpret_cast<uint4*>(p) = u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i)
      if (i < count) p[i] = from_f32<T>(v[i]);
  }
}

// One head as a lane group holds it.
struct Head {
  unsigned b, i;  // batch entry and place in the row
  int h;
  bool key;
};

template <typename T>
__device__ __forceinline__ T* at(const RotaryTensor& x, const Head& r, int col) {
  return static_cast<T*>(x.ptr) + r.b * x.sb + r.i * x.ss + r.h * x.sh + col;
}

// Rotates the lane's 8 values of a head.  `angles`: this token's (cos, sin).
// SHUFFLE: the partner of every value lies at the same place of another lane.
template <int LANES, bool SHUFFLE>
__device__ __forceinline__ void rotate(float (&y)[kV], const RotaryParams& p, const float2* angles, float sign, int lane,
                                       float* exchange) {
  const int r = p.rotated, half = r / 2, col = lane * kV;
  if (p.interleaved) {  // neighbours: both in this lane
#pragma unroll
    for (int i = 0; i < kV; i += 2) {
      if (col + i < r) {
        const float2 a = angles[(col + i) / 2];
        const float u = y[i], v = y[i + 1], sn = sign * a.y;
        y[i] = u * a.x - v * sn;
        y[i + 1] = v * a.x + u * sn;
      }
    }
    return;
  }
  float o[kV];
  if (SHUFFLE) {
    const int step = half / kV;
    const int from = lane < step ? lane + step : (lane < 2 * step ? lane - step : lane);
#pragma unroll
    for (int i = 0; i < kV; ++i) o[i] = __shfl_sync(0xffffffffu, y[i], from, LANES);
  } else {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kV; ++i) exchange[col + i] = y[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int c = col + i;
      o[i] = c < half ? exchange[c + half] : (c < r ? exchange[c - half] : 0.f);
    }
  }
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    const int c = col + i;
    if (c < r) {
      const bool low = c < half;
      const float2 a = angles[low ? c : c - half];
      y[i] = y[i] * a.x + (low ? -sign : sign) * a.y * o[i];
    }
  }
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// GRAD: dx and the gains' gradients.  A block takes `chunk` tokens at a time.
template <typename T, int LANES, bool SHUFFLE, bool GRAD>
__global__ void __launch_bounds__(kThreads) qk_kernel(const RotaryParams p, int chunk, bool vec) {
  extern __shared__ float2 angles[];  // [chunk][rotated / 2]
  __shared__ float exchange[SHUFFLE ? 1 : kThreads * kV];
  __shared__ float gains[2][launch::kRotaryMaxDim];
  constexpr int kGroups = kThreads / LANES;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int col = lane * kV, count = min(kV, p.d - col), half = p.rotated / 2;
  const bool holds = col < p.d;
  const float inv_d = 1.f / p.d;
  const int heads = p.q.h + p.k.h;
  for (int i = threadIdx.x; i < 2 * p.d; i += kThreads) {
    const float* w = i < p.d ? p.wq : p.wk;
    gains[i / p.d][i % p.d] = w != nullptr ? w[i % p.d] : 1.f;
  }
  float dw[2][kV];
#pragma unroll
  for (int i = 0; i < kV; ++i) dw[0][i] = dw[1][i] = 0.f;

  // Token counts stay below 2^31 (checked by the caller): 32-bit divisions.
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * chunk; t0 < p.tokens; t0 += static_cast<int64_t>(gridDim.x) * chunk) {
    const int n = static_cast<int>(min(static_cast<int64_t>(chunk), p.tokens - t0));
    __syncthreads();
    for (int i = threadIdx.x; i < n * half; i += kThreads) {
      const unsigned t = static_cast<unsigned>(t0) + i / half;
      int64_t pos = t % p.s;
      if (p.positions != nullptr) {
        const int64_t e = t / p.s * p.pos_sb + pos * p.pos_ss;
        pos = p.pos_bytes == 8 ? static_cast<const long long*>(p.positions)[e] : static_cast<const int*>(p.positions)[e];
      }
      const double a = static_cast<double>(pos) * p.freq[i % half];
      const double turns = rint(a * 0.15915494309189535);  // 1 / (2 pi)
      const float x = static_cast<float>(fma(turns, -6.283185307179586, a) - turns * 2.4492935982947064e-16);
      float sn, cs;
      sincosf(x, &sn, &cs);
      angles[i] = make_float2(cs, sn);
    }
    __syncthreads();
    const int total = n * heads;
    for (int r0 = 0; r0 < total; r0 += kGroups) {
      const int row = r0 + group;
      const bool live = row < total && holds;
      Head hd;
      const int in_chunk = min(row, total - 1) / heads;
      hd.b = static_cast<unsigned>(t0 + in_chunk) / p.s;
      hd.i = static_cast<unsigned>(t0 + in_chunk) % p.s;
      hd.h = min(row, total - 1) % heads;
      hd.key = hd.h >= p.q.h;
      if (hd.key) hd.h -= p.q.h;
      float x[kV], w[kV];
#pragma unroll
      for (int i = 0; i < kV; ++i) x[i] = w[i] = 0.f;
      float g[kV];
      if (live) {
        load8<T>(at<T>(hd.key ? p.k : p.q, hd, col), vec, count, x);
        if (GRAD) load8<T>(at<T>(hd.key ? p.gk : p.gq, hd, col), vec, count, g);
#pragma unroll
        for (int i = 0; i < kV; ++i) w[i] = i < count ? gains[hd.key][col + i] : 0.f;
      } else if (GRAD) {
#pragma unroll
        for (int i = 0; i < kV; ++i) g[i] = 0.f;
      }
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kV; ++i) sum += x[i] * x[i];
      const float rs = rsqrtf(group_sum<LANES>(sum) * inv_d + p.eps);
      const float2* an = angles + in_chunk * half;
      float* ex = SHUFFLE ? nullptr : exchange + group * LANES * kV;
      if (!GRAD) {
#pragma unroll
        for (int i = 0; i < kV; ++i) x[i] *= rs * w[i];
        rotate<LANES, SHUFFLE>(x, p, an, 1.f, lane, ex);
        if (live) store8<T>(at<T>(hd.key ? p.ok : p.oq, hd, col), vec, count, x);
      } else {
        rotate<LANES, SHUFFLE>(g, p, an, -1.f, lane, ex);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          x[i] *= rs;  // n
          const float gn = live ? g[i] * x[i] : 0.f;
          if (hd.key)
            dw[1][i] += gn;
          else
            dw[0][i] += gn;
          dot += gn * w[i];
          g[i] *= w[i];
        }
        dot = group_sum<LANES>(dot) * inv_d;
#pragma unroll
        for (int i = 0; i < kV; ++i) x[i] = rs * (g[i] - x[i] * dot);
        if (live) store8<T>(at<T>(hd.key ? p.ok : p.oq, hd, col), vec, count, x);
      }
    }
  }
  if (GRAD && p.partial != nullptr) {
    __shared__ float sums[kThreads * kV];
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kV; ++i) sums[group * LANES * kV + col + i] = which ? dw[1][i] : dw[0][i];
      __syncthreads();
      for (int c = threadIdx.x; c < p.d; c += kThreads) {
        float v = 0.f;
        for (int g = 0; g < kGroups; ++g) v += sums[g * LANES * kV + c];
        p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * p.d + c] = v;
      }
    }
  }
}

// dw[c] = sum over blocks of partial[block][c]; one block of 8 warps for 32 columns.
__global__ void __launch_bounds__(256) gains_kernel(const float* partial, int blocks, int cols, float* dw) {
  __shared__ float sums[8][33];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, part = threadIdx.x / 32;
  float v = 0.f;
  if (c < cols)
    for (int b = part; b < blocks; b += 8) v += partial[static_cast<int64_t>(b) * cols + c];
  sums[part][threadIdx.x % 32] = v;
  __syncthreads();
  if (part == 0 && c < cols) {
    for (int i = 1; i < 8; ++i) v += sums[i][threadIdx.x];
    dw[c] = v;
  }
}

bool aligned(const RotaryTensor& x, int size) {
  if (x.ptr == nullptr) return true;
  const int64_t m = 16 / size;
  return reinterpret_cast<uintptr_t>(x.ptr) % 16 == 0 && x.sb % m == 0 && x.ss % m == 0 && x.sh % m == 0;
}

// Tokens of a chunk: enough heads for every lane group to take four, while
// there are blocks for all SMs.
int chunk_tokens(const RotaryParams& p, int sms) {
  const int lanes = p.d <= 64 ? 8 : (p.d <= 128 ? 16 : 32);
  const int heads = p.q.h + p.k.h, groups = kThreads / lanes;
  int64_t n = (4 * groups + heads - 1) / heads;
  const int64_t most = (p.tokens + 2 * sms - 1) / (2 * sms);
  if (n > most) n = most;
  if (n > 32) n = 32;
  return static_cast<int>(n < 1 ? 1 : n);
}

template <typename T, int LANES, bool SHUFFLE, bool GRAD>
void run(const RotaryParams& p, int sms, cudaStream_t s) {
  const int size = sizeof(T);
  const bool vec = p.d % kV == 0 && aligned(p.q, size) && aligned(p.k, size) && aligned(p.oq, size) &&
                   aligned(p.ok, size) && aligned(p.gq, size) && aligned(p.gk, size);
  const int chunk = chunk_tokens(p, sms);
  int64_t blocks = (p.tokens + chunk - 1) / chunk;
  if (GRAD) blocks = launch::qk_norm_rotary_blocks(p, sms);
  const size_t bytes = sizeof(float2) * chunk * (p.rotated / 2);
  qk_kernel<T, LANES, SHUFFLE, GRAD><<<static_cast<unsigned>(blocks), kThreads, bytes, s>>>(p, chunk, vec);
}

template <typename T, bool GRAD>
void by_size(const RotaryParams& p, int sms, cudaStream_t s) {
  const bool shuffle = p.interleaved || p.rotated % (2 * kV) == 0;
  if (p.d <= 64)
    shuffle ? run<T, 8, true, GRAD>(p, sms, s) : run<T, 8, false, GRAD>(p, sms, s);
  else if (p.d <= 128)
    shuffle ? run<T, 16, true, GRAD>(p, sms, s) : run<T, 16, false, GRAD>(p, sms, s);
  else
    shuffle ? run<T, 32, true, GRAD>(p, sms, s) : run<T, 32, false, GRAD>(p, sms, s);
}

template <bool GRAD>
void by_type(const RotaryParams& p, int sms, cudaStream_t s) {
  if (p.tokens == 0 || p.d == 0) return;
  switch (p.dt) {
    case kF32: return by_size<float, GRAD>(p, sms, s);
    case kBF16: return by_size<__nv_bfloat16, GRAD>(p, sms, s);
    case kF16: return by_size<__half, GRAD>(p, sms, s);
  }
}

}  // namespace

namespace launch {

int qk_norm_rotary_blocks(const RotaryParams& p, int sms) {
  const int chunk = chunk_tokens(p, sms);
  const int64_t all = (p.tokens + chunk - 1) / chunk;
  return static_cast<int>(all < 4 * sms ? all : 4 * sms);  // four resident blocks an SM, then further chunks each
}

void qk_norm_rotary_forward(const RotaryParams& p, int sms, cudaStream_t s) { by_type<false>(p, sms, s); }

void qk_norm_rotary_backward(const RotaryParams& p, int sms, float* dw, cudaStream_t s) {
  by_type<true>(p, sms, s);
  if (p.partial != nullptr)
    gains_kernel<<<(2 * p.d + 31) / 32, 256, 0, s>>>(p.partial, qk_norm_rotary_blocks(p, sms), 2 * p.d, dw);
}

}  // namespace launch
}  // namespace bitscom_b200
