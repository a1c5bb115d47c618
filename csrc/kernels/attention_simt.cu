// Masked attention in fp32 arithmetic on the CUDA cores: forward, dq, and dk/dv.
//
// The form for what the tensor-core kernels do not take: fp32 tensors (whose
// products would lose 13 bits on the tensor cores) and head sizes over 128 or
// not a multiple of 8.  One pass over the keys with the running maximum and sum
// of the softmax; the backward pass recomputes the probabilities from the saved
// log-sum.  Sums stay in fp32 registers, each gradient element is summed by one
// thread in a fixed order (no atomics), the heads that share a key head too.
//
// 256 threads hold a tile of 64 x 32 scores, 2 x 4 each: thread (ty, tx) has rows
// 2 ty + {0, 1}, columns tx + 8 j.  Rows are padded by 16 bytes in shared
// memory, so the 8 columns of a quarter warp fall into different banks.
// Bound by the FMA pipe and shared-memory reads (6 16-byte reads for 32 FMAs).
#include <cuda_runtime.h>

#include <algorithm>

#include "attention_common.cuh"

namespace bitscom_b200 {
namespace {

constexpr int kThreads = 256, kRows = 64, kCols = 32;

// Rows that no pair of theirs is visible in (padding) are taken as zeros: their
// weight is zero, and zero times what may stand there need not be.
template <typename T, int DP, bool KEYS>
__device__ __forceinline__ void load_tile(float* s, const AttnParams& p, const AttnTensor& x, int b, int h, int first,
                                          int count) {
  const T* base = static_cast<const T*>(x.ptr) + b * x.sb + h * x.sh;
  const int limit = KEYS ? p.sk : p.sq;
  for (int i = threadIdx.x; i < count * DP; i += kThreads) {
    const int r = first + i / DP, c = i % DP;
    const bool live = r < limit && c < p.d && !(KEYS ? attn_key_dead(p, b, r) : attn_row_dead(p, b, r));
    s[i / DP * (DP + 4) + c] = live ? to_f32<T>(base[r * x.ss + c]) : 0.f;
  }
}

// Scores of 2 x 4 pairs.
template <int DP>
__device__ __forceinline__ void dots(const float* a, const float* b, int ty, int tx, float (&o)[2][4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
#pragma unroll 4
  for (int c = 0; c < DP; c += 4) {
    float4 x[2], y[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = *reinterpret_cast<const float4*>(a + (2 * ty + i) * (DP + 4) + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 8 * j) * (DP + 4) + c);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[i][j] += x[i].x * y[j].x + x[i].y * y[j].y + x[i].z * y[j].z + x[i].w * y[j].w;
  }
}

// acc[i][c] += sum_j w[2 ty + i][j] * b[j][4 (tx + 8 c) ..]
template <int DP>
__device__ __forceinline__ void accumulate(const float* w, const float* b, int ty, int tx, float4 (&acc)[2][DP / 32]) {
  for (int j = 0; j < kCols; ++j) {
    const float w0 = w[(2 * ty) * (kCols + 1) + j], w1 = w[(2 * ty + 1) * (kCols + 1) + j];
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
      const float4 y = *reinterpret_cast<const float4*>(b + j * (DP + 4) + 4 * (tx + 8 * c));
      acc[0][c].x += w0 * y.x; acc[0][c].y += w0 * y.y; acc[0][c].z += w0 * y.z; acc[0][c].w += w0 * y.w;
      acc[1][c].x += w1 * y.x; acc[1][c].y += w1 * y.y; acc[1][c].z += w1 * y.z; acc[1][c].w += w1 * y.w;
    }
  }
}

template <typename T, int DP>
__device__ __forceinline__ void store_rows(const AttnTensor& x, int b, int h, int row, int limit, int d, int tx,
                                           const float4 (&acc)[DP / 32], float f) {
  if (row >= limit) return;
  T* o = static_cast<T*>(x.ptr) + b * x.sb + h * x.sh + row * x.ss;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c) {
    const float v[4] = {acc[c].x, acc[c].y, acc[c].z, acc[c].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int col = 4 * (tx + 8 * c) + e;
      if (col < d) o[col] = from_f32<T>(v[e] * f);
    }
  }
}

// Base-2 score of a pair and, for the backward pass, the factor that the cap puts on its gradient.
__device__ __forceinline__ float score(const AttnParams& p, float dot, float slope, int pos, int key, float* slope_out) {
  float s = dot * p.scale;
  float f = 1.f;
  if (p.cap > 0.f) {
    const float t = tanhf(s / p.cap);
    s = t * p.cap;
    f = 1.f - t * t;
  }
  if (slope != 0.f) s -= slope * fabsf(static_cast<float>(pos - key));
  *slope_out = f;
  return s * kLog2e;
}

// GRAD: dq instead of the output.
template <typename T, int DP, bool GRAD>
__global__ void __launch_bounds__(kThreads) rows_kernel(const AttnParams p) {
  extern __shared__ float4 smem4[];
  float* sq = reinterpret_cast<float*>(smem4);
  float* sdo = sq + kRows * (DP + 4);
  float* sk = sdo + (GRAD ? kRows * (DP + 4) : 0);
  float* sv = sk + kCols * (DP + 4);
  float* sw = sv + kCols * (DP + 4);
  __shared__ int lo_all, hi_all;
  const int tid = threadIdx.x, ty = tid / 8, tx = tid % 8;
  const int b = blockIdx.z, h = blockIdx.y, hk = h / (p.hq / p.hk), row0 = blockIdx.x * kRows;
  if (tid == 0) {
    lo_all = 0x7fffffff;
    hi_all = 0;
  }
  load_tile<T, DP, false>(sq, p, p.q, b, h, row0, kRows);
  if (GRAD) load_tile<T, DP, false>(sdo, p, p.dout, b, h, row0, kRows);
  __syncthreads();
  int2 range[2];
  float m[2], l[2], lse[2], delta[2];
  float4 acc[2][DP / 32];
  const float slope = p.slopes != nullptr ? p.slopes[h] : 0.f;
  const int64_t stat = (static_cast<int64_t>(b) * p.hq + h) * p.sq;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = row0 + 2 * ty + i;
    range[i] = row < p.sq ? attn_row_range(p, b, row) : make_int2(0, 0);
    m[i] = -INFINITY;
    l[i] = lse[i] = delta[i] = 0.f;
    if (GRAD && row < p.sq) {
      lse[i] = p.lse[stat + row];
      delta[i] = p.delta[stat + row];
    }
    if (tx == 0 && range[i].y > range[i].x) {
      atomicMin(&lo_all, range[i].x);
      atomicMax(&hi_all, range[i].y);
    }
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __syncthreads();
  for (int key0 = (lo_all < hi_all ? lo_all / kCols * kCols : hi_all); key0 < hi_all; key0 += kCols) {
    __syncthreads();
    load_tile<T, DP, true>(sk, p, p.k, b, hk, key0, kCols);
    load_tile<T, DP, true>(sv, p, p.v, b, hk, key0, kCols);
    __syncthreads();
    float s[2][4], dp[2][4];
    dots<DP>(sq, sk, ty, tx, s);
    if (GRAD) dots<DP>(sdo, sv, ty, tx, dp);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int pos = row0 + 2 * ty + i + p.sk - p.sq;
      float f[4], best = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = key0 + tx + 8 * j;
        const bool seen = key >= range[i].x && key < range[i].y;
        s[i][j] = seen ? score(p, s[i][j], slope, pos, key, &f[j]) : -INFINITY;
        best = fmaxf(best, s[i][j]);
      }
      if (GRAD) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + tx + 8 * j;
          const bool seen = key >= range[i].x && key < range[i].y;
          sw[(2 * ty + i) * (kCols + 1) + tx + 8 * j] =
              seen ? exp2f(s[i][j] - lse[i]) * (dp[i][j] - delta[i]) * f[j] : 0.f;
        }
      } else {
        for (int o = 1; o < 8; o <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
        const float mn = fmaxf(m[i], best);
        const float base = mn == -INFINITY ? 0.f : mn;
        const float shrink = exp2f(m[i] - base);
        m[i] = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = exp2f(s[i][j] - base);
          sum += e;
          sw[(2 * ty + i) * (kCols + 1) + tx + 8 * j] = e;
        }
        l[i] = l[i] * shrink + sum;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          acc[i][c].x *= shrink; acc[i][c].y *= shrink; acc[i][c].z *= shrink; acc[i][c].w *= shrink;
        }
      }
    }
    __syncthreads();
    accumulate<DP>(sw, GRAD ? sk : sv, ty, tx, acc);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = row0 + 2 * ty + i;
    if (GRAD) {
      store_rows<T, DP>(p.dq, b, h, row, p.sq, p.d, tx, acc[i], p.scale);
    } else {
      float sum = l[i];
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const bool none = range[i].y <= range[i].x;
      store_rows<T, DP>(p.o, b, h, row, p.sq, p.d, tx, acc[i], none ? 0.f : 1.f / sum);
      if (tx == 0 && row < p.sq && p.lse != nullptr) p.lse[stat + row] = none ? INFINITY : m[i] + log2f(sum);
    }
  }
}

// dk and dv of 64 keys of one key head, over all rows of the query heads that share it.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) keys_kernel(const AttnParams p) {
  extern __shared__ float4 smem4[];
  float* sk = reinterpret_cast<float*>(smem4);
  float* sv = sk + kRows * (DP + 4);
  float* sq = sv + kRows * (DP + 4);
  float* sdo = sq + kCols * (DP + 4);
  float* sw = sdo + kCols * (DP + 4);
  __shared__ int2 range[kCols];
  __shared__ float lse[kCols], delta[kCols];
  const int tid = threadIdx.x, ty = tid / 8, tx = tid % 8;
  const int b = blockIdx.z, hk = blockIdx.y, group = p.hq / p.hk, key0 = blockIdx.x * kRows;
  load_tile<T, DP, true>(sk, p, p.k, b, hk, key0, kRows);
  load_tile<T, DP, true>(sv, p, p.v, b, hk, key0, kRows);
  float4 dk[2][DP / 32], dv[2][DP / 32];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) dk[i][c] = dv[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int g = 0; g < group; ++g) {
    const int h = hk * group + g;
    const float slope = p.slopes != nullptr ? p.slopes[h] : 0.f;
    const int64_t stat = (static_cast<int64_t>(b) * p.hq + h) * p.sq;
    for (int row0 = 0; row0 < p.sq; row0 += kCols) {
      __syncthreads();
      bool some = false;
      if (tid < kCols) {
        const int row = row0 + tid;
        const int2 r = row < p.sq ? attn_row_range(p, b, row) : make_int2(0, 0);
        range[tid] = r;
        lse[tid] = row < p.sq ? p.lse[stat + row] : INFINITY;
        delta[tid] = row < p.sq ? p.delta[stat + row] : 0.f;
        some = r.x < r.y && r.x < key0 + kRows && r.y > key0;
      }
      if (!__syncthreads_or(some)) continue;
      load_tile<T, DP, false>(sq, p, p.q, b, h, row0, kCols);
      load_tile<T, DP, false>(sdo, p, p.dout, b, h, row0, kCols);
      __syncthreads();
      float s[2][4], dp[2][4];
      dots<DP>(sk, sq, ty, tx, s);
      dots<DP>(sv, sdo, ty, tx, dp);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = key0 + 2 * ty + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = tx + 8 * j;
          float f = 1.f, e = 0.f;
          if (key >= range[c].x && key < range[c].y)
            e = exp2f(score(p, s[i][j], slope, row0 + c + p.sk - p.sq, key, &f) - lse[c]);
          s[i][j] = e;
          dp[i][j] = e == 0.f ? 0.f : e * (dp[i][j] - delta[c]) * f;
          sw[(2 * ty + i) * (kCols + 1) + c] = e;
        }
      }
      __syncthreads();
      accumulate<DP>(sw, sdo, ty, tx, dv);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sw[(2 * ty + i) * (kCols + 1) + tx + 8 * j] = dp[i][j];
      __syncthreads();
      accumulate<DP>(sw, sq, ty, tx, dk);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    store_rows<T, DP>(p.dk, b, hk, key0 + 2 * ty + i, p.sk, p.d, tx, dk[i], p.scale);
    store_rows<T, DP>(p.dv, b, hk, key0 + 2 * ty + i, p.sk, p.d, tx, dv[i], 1.f);
  }
}

// delta = sum over d of dout * o, one warp a row.  In 16 bits o is the rounded result: delta is off by up to half a
// step of sum |dout| |o|, beside the half step that every gradient is rounded by.
template <typename T>
__global__ void __launch_bounds__(kThreads) delta_kernel(const AttnParams p) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32;
  if (row >= static_cast<int64_t>(p.b) * p.hq * p.sq) return;
  const int i = row % p.sq, h = row / p.sq % p.hq, b = row / (static_cast<int64_t>(p.sq) * p.hq);
  const T* o = static_cast<const T*>(p.o.ptr) + b * p.o.sb + h * p.o.sh + i * p.o.ss;
  const T* g = static_cast<const T*>(p.dout.ptr) + b * p.dout.sb + h * p.dout.sh + i * p.dout.ss;
  float sum = 0.f;
  for (int c = threadIdx.x & 31; c < p.d; c += 32)
    sum += to_f32<T>(o[c]) * to_f32<T>(g[c]);
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  if ((threadIdx.x & 31) == 0) p.delta[row] = sum;
}

template <typename T, int DP>
void run_forward(const AttnParams& p, cudaStream_t s) {
  const int bytes = ((kRows + 2 * kCols) * (DP + 4) + kRows * (kCols + 1)) * 4;
  cudaFuncSetAttribute(rows_kernel<T, DP, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  rows_kernel<T, DP, false><<<dim3((p.sq + kRows - 1) / kRows, p.hq, p.b), kThreads, bytes, s>>>(p);
}

template <typename T, int DP>
void run_backward(const AttnParams& p, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.b) * p.hq * p.sq;
  const int warps = kThreads / 32;
  delta_kernel<T><<<static_cast<unsigned>((rows + warps - 1) / warps), kThreads, 0, s>>>(p);
  const int bytes = (2 * (kRows + kCols) * (DP + 4) + kRows * (kCols + 1)) * 4;
  cudaFuncSetAttribute(rows_kernel<T, DP, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  cudaFuncSetAttribute(keys_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  rows_kernel<T, DP, true><<<dim3((p.sq + kRows - 1) / kRows, p.hq, p.b), kThreads, bytes, s>>>(p);
  keys_kernel<T, DP><<<dim3((p.sk + kRows - 1) / kRows, p.hk, p.b), kThreads, bytes, s>>>(p);
}

template <typename T>
void by_size(const AttnParams& p, bool grad, cudaStream_t s) {
  if (p.d <= 64)
    grad ? run_backward<T, 64>(p, s) : run_forward<T, 64>(p, s);
  else if (p.d <= 128)
    grad ? run_backward<T, 128>(p, s) : run_forward<T, 128>(p, s);
  else
    grad ? run_backward<T, 256>(p, s) : run_forward<T, 256>(p, s);
}

void by_type(const AttnParams& p, bool grad, cudaStream_t s) {
  switch (p.dt) {
    case kF32: return by_size<float>(p, grad, s);
    case kBF16: return by_size<__nv_bfloat16>(p, grad, s);
    case kF16: return by_size<__half>(p, grad, s);
  }
}

}  // namespace

namespace launch {

void attention_simt_forward(const AttnParams& p, cudaStream_t s) { by_type(p, false, s); }
void attention_simt_backward(const AttnParams& p, cudaStream_t s) { by_type(p, true, s); }

}  // namespace launch
}  // namespace bitscom_b200
