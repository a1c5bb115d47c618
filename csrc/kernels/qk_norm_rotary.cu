// Norm of queries and keys for each head, with the position rotation in the
// same pass; forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps);  n = x r;  y = n w
//   (y1, y2) -> (y1 cos a - y2 sin a, y2 cos a + y1 sin a),  a = position * freq
//   backward: g = dy turned by -a;  dw = sum g n;  dx = r (g w - n mean(g w n))
//
// Each head is read once and written once (backward: x and dy read, dx written).  Long
// rows are bound by memory with too few loads in flight; what fits in L2 (8 x 1024 tokens x 32
// heads x 64) by the instructions of a token's angles and heads, issuing on half of all clocks.  A head's D values lie in 16-byte pieces across a group
// of 8, 16 or 32 lanes, so the norm is a few shuffles; the partner of a pair
// (i, i + rotated / 2) sits in another lane at the same place of its piece, one
// shuffle more.  When a half is not a whole number of pieces, the partners are
// exchanged through shared memory.  Norms, rotations and sums are in fp32, with
// one rounding at the end; the angle is formed and reduced to one turn in fp64
// (a position of 10^6 times a frequency leaves fp32 five digits short).
//
// A lane group takes a token, forms the angles of its own values once (4 % of the
// time at 20 heads) and goes through the heads with them in registers, the next
// heads' loads under way.  No lane group waits for another: with angles
// formed by the block in shared memory and a head to a lane group, the barriers and the
// divisions for each head held 131072 tokens x 20 heads x 128 (fp16) at 629 us; this
// form takes 336 us (4.0 TB/s, 61 % of a copy).  Two blocks of 128
// registers a thread an SM: three of 80 spill (452 us).
//
// The gains' gradients are summed in registers over a lane group's heads, then
// over the block's groups and over the blocks in a fixed order: no atomics, the
// same bits every time.
#include <cuda_runtime.h>

#include "attention_common.cuh"
#include "qk_norm_rotary.h"

namespace bitscom_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kV = 8;  // values of a lane
constexpr int kBlocks = 2;  // resident on an SM

// A lane's 8 values as they lie in memory.
template <typename T>
struct Raw {
  uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int count, Raw<T>& o) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) o.w[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T* t = reinterpret_cast<T*>(o.w);
#pragma unroll
    for (int i = 0; i < kV; ++i) t[i] = i < count ? p[i] : from_f32<T>(0.f);
  }
}

template <typename T>
__device__ __forceinline__ void values(const Raw<T>& r, bool live, float (&o)[kV]) {
  const T* t = reinterpret_cast<const T*>(r.w);
#pragma unroll
  for (int i = 0; i < kV; ++i) o[i] = live ? to_f32<T>(t[i]) : 0.f;
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

template <int LANES, int U>
__device__ __forceinline__ void group_sums(float (&v)[U]) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(0xffffffffu, v[u], o);
}

// Rotates the lane's 8 values of a head.  `cs`, `sn`: cosine and signed sine of each value's pair (1, 0 where
// nothing is rotated): y cs + partner sn.
template <int LANES, bool SHUFFLE>
__device__ __forceinline__ void rotate(float (&y)[kV], const RotaryParams& p, const float (&cs)[kV], const float (&sn)[kV],
                                       int from, int lane, float* exchange) {
  float o[kV];
  if (p.interleaved) {  // neighbours: both in this lane
#pragma unroll
    for (int i = 0; i < kV; ++i) o[i] = y[i ^ 1];
  } else if (SHUFFLE) {
#pragma unroll
    for (int i = 0; i < kV; ++i) o[i] = __shfl_sync(0xffffffffu, y[i], from, LANES);
  } else {
    const int half = p.rotated / 2, col = lane * kV;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kV; ++i) exchange[col + i] = y[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int c = col + i;
      o[i] = c < half ? exchange[c + half] : (c < p.rotated ? exchange[c - half] : 0.f);
    }
  }
#pragma unroll
  for (int i = 0; i < kV; ++i) y[i] = y[i] * cs[i] + sn[i] * o[i];
}

// What a lane keeps while it goes through the heads of one token.
template <typename T>
struct Lane {
  int col, count, from, lane;
  bool holds, vec;
  float inv_d;
  float cs[kV], sn[kV];
  float* exchange;
};

// `n` heads of one tensor; AHEAD of them are on their way while one is worked on, which is what
// keeps enough bytes in flight.  `rounds` is the most heads that any lane group of the warp has.
template <typename T, int LANES, bool SHUFFLE, bool GRAD>
__device__ __forceinline__ void heads(const RotaryParams& p, const Lane<T>& ln, const T* in, int64_t in_sh, const T* grad,
                                      int64_t grad_sh, T* out, int64_t out_sh, int n, int rounds, const float (&w)[kV],
                                      float (&dw)[kV]) {
  constexpr int AHEAD = sizeof(T) == 4 || GRAD ? 2 : 4, U = GRAD ? 1 : 2;
  Raw<T> xr[AHEAD], gr[GRAD ? AHEAD : 1];
  if (!ln.holds) n = 0;
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {
    if (u < n) {
      load8<T>(in + u * in_sh, ln.vec, ln.count, xr[u]);
      if (GRAD) load8<T>(grad + u * grad_sh, ln.vec, ln.count, gr[u]);
    }
  }
  for (int h0 = 0; h0 < rounds; h0 += AHEAD) {
#pragma unroll
    for (int a = 0; a < AHEAD; a += U) {  // U heads side by side: their chains of shuffles overlap
      const int h = h0 + a;
      float x[U][kV], g[U][kV], sum[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        values<T>(xr[a + u], h + u < n, x[u]);
        if (GRAD) values<T>(gr[GRAD ? a + u : 0], h + u < n, g[u]);
        if (h + u + AHEAD < n) {
          load8<T>(in + (h + u + AHEAD) * in_sh, ln.vec, ln.count, xr[a + u]);
          if (GRAD) load8<T>(grad + (h + u + AHEAD) * grad_sh, ln.vec, ln.count, gr[GRAD ? a + u : 0]);
        }
        sum[u] = 0.f;
#pragma unroll
        for (int i = 0; i < kV; ++i) sum[u] += x[u][i] * x[u][i];
      }
      group_sums<LANES, U>(sum);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float rs = rsqrtf(sum[u] * ln.inv_d + p.eps);
        sum[u] = rs;
#pragma unroll
        for (int i = 0; i < kV; ++i) x[u][i] *= GRAD ? rs : rs * w[i];
      }
      if (!GRAD) {
#pragma unroll
        for (int u = 0; u < U; ++u) rotate<LANES, SHUFFLE>(x[u], p, ln.cs, ln.sn, ln.from, ln.lane, ln.exchange);
      } else {
        float dot[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          rotate<LANES, SHUFFLE>(g[u], p, ln.cs, ln.sn, ln.from, ln.lane, ln.exchange);
          dot[u] = 0.f;
#pragma unroll
          for (int i = 0; i < kV; ++i) {
            dw[i] += g[u][i] * x[u][i];
            g[u][i] *= w[i];
            dot[u] += g[u][i] * x[u][i];
          }
        }
        group_sums<LANES, U>(dot);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < kV; ++i) x[u][i] = sum[u] * (g[u][i] - x[u][i] * (dot[u] * ln.inv_d));
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (h + u < n) store8<T>(out + (h + u) * out_sh, ln.vec, ln.count, x[u]);
    }
  }
}

// Cosine and sine of position * frequency.
__device__ __forceinline__ void turn(int64_t pos, double freq, float* cs, float* sn) {
  const double a = static_cast<double>(pos) * freq;
  const double turns = rint(a * 0.15915494309189535);  // 1 / (2 pi)
  sincosf(static_cast<float>(fma(turns, -6.283185307179586, a) - turns * 2.4492935982947064e-16), sn, cs);
}

// GRAD: dx and the gains' gradients.  A lane group takes a token (or one of `split` parts of its heads), forms the
// angles of its values and goes through the heads with them in registers; nothing is shared between groups.
template <typename T, int LANES, bool SHUFFLE, bool GRAD>
__global__ void __launch_bounds__(kThreads, kBlocks) qk_kernel(const RotaryParams p, int split, bool vec) {
  constexpr int kGroups = kThreads / LANES;
  __shared__ float exchange[SHUFFLE ? 1 : kThreads * kV];
  const int group = threadIdx.x / LANES;
  const int half = p.rotated / 2, all = p.q.h + p.k.h;
  const int per = (all + split - 1) / split;
  Lane<T> ln;
  ln.lane = threadIdx.x % LANES;
  ln.col = ln.lane * kV;
  ln.count = min(kV, p.d - ln.col);
  ln.holds = ln.col < p.d;
  ln.vec = vec;
  ln.inv_d = 1.f / p.d;
  ln.exchange = SHUFFLE ? nullptr : exchange + group * LANES * kV;
  const int step = half / kV;
  ln.from = ln.lane < step ? ln.lane + step : (ln.lane < 2 * step ? ln.lane - step : ln.lane);
  float wq[kV], wk[kV], dwq[kV], dwk[kV];
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    wq[i] = wk[i] = i < ln.count ? 1.f : 0.f;
    if (i < ln.count && p.wq != nullptr) wq[i] = p.wq[ln.col + i];
    if (i < ln.count && p.wk != nullptr) wk[i] = p.wk[ln.col + i];
    dwq[i] = dwk[i] = 0.f;
  }

  // All lanes of a warp make the same number of steps (the shuffles want them); token
  // counts stay below 2^31 (checked by the caller): 32-bit divisions.
  const int64_t items = p.tokens * split, stride = static_cast<int64_t>(gridDim.x) * kGroups;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups + group / (32 / LANES) * (32 / LANES); first < items; first += stride) {
    const int64_t item = first + group % (32 / LANES);
    const bool has = item < items;
    const unsigned t = has ? static_cast<unsigned>(split == 1 ? item : item / split) : 0u;
    const int part = split == 1 ? 0 : static_cast<int>(item % split);
    const unsigned b = t / p.s, i0 = t % p.s;
    int64_t pos = i0;
    if (p.positions != nullptr) {
      const int64_t e = b * p.pos_sb + i0 * p.pos_ss;
      pos = p.pos_bytes == 8 ? static_cast<const long long*>(p.positions)[e] : static_cast<const int*>(p.positions)[e];
    }
    if (p.interleaved) {
#pragma unroll
      for (int i = 0; i < kV; i += 2) {
        ln.cs[i] = ln.cs[i + 1] = 1.f;
        ln.sn[i] = ln.sn[i + 1] = 0.f;
        if (ln.col + i < p.rotated) {
          turn(pos, p.freq[(ln.col + i) / 2], &ln.cs[i], &ln.sn[i + 1]);
          ln.cs[i + 1] = ln.cs[i];
          ln.sn[i] = -ln.sn[i + 1];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int c = ln.col + i;
        ln.cs[i] = 1.f;
        ln.sn[i] = 0.f;
        if (c < p.rotated) {
          turn(pos, p.freq[c < half ? c : c - half], &ln.cs[i], &ln.sn[i]);
          if (c < half) ln.sn[i] = -ln.sn[i];
        }
      }
    }
    if (GRAD) {
#pragma unroll
      for (int i = 0; i < kV; ++i) ln.sn[i] = -ln.sn[i];
    }
    const auto at = [&](const RotaryTensor& x, int h) {
      return static_cast<T*>(x.ptr) + b * x.sb + i0 * x.ss + h * x.sh + ln.col;
    };
    // Heads [h0, h1) of the list q heads, k heads.
    const int h0 = min(all, part * per), h1 = min(all, h0 + per);
    const int q0 = min(h0, p.q.h), q1 = min(h1, p.q.h), k0 = max(h0, p.q.h) - p.q.h, k1 = max(h1, p.q.h) - p.q.h;
    const int nq = has ? q1 - q0 : 0, nk = has ? k1 - k0 : 0;
    const int rounds_q = __reduce_max_sync(0xffffffffu, nq), rounds_k = __reduce_max_sync(0xffffffffu, nk);
    heads<T, LANES, SHUFFLE, GRAD>(p, ln, at(p.q, q0), p.q.sh, GRAD ? at(p.gq, q0) : nullptr, p.gq.sh, at(p.oq, q0),
                                      p.oq.sh, nq, rounds_q, wq, dwq);
    heads<T, LANES, SHUFFLE, GRAD>(p, ln, at(p.k, k0), p.k.sh, GRAD ? at(p.gk, k0) : nullptr, p.gk.sh, at(p.ok, k0),
                                      p.ok.sh, nk, rounds_k, wk, dwk);
  }
  if (GRAD && p.partial != nullptr) {
    __shared__ float sums[kThreads * kV];
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kV; ++i) sums[group * LANES * kV + ln.col + i] = which ? dwk[i] : dwq[i];
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

// Parts of a token's heads: one, so that angles are formed once for all heads, unless the
// tokens are too few to fill every SM's blocks twice.
int head_split(const RotaryParams& p, int sms) {
  const int lanes = p.d <= 64 ? 8 : (p.d <= 128 ? 16 : 32);
  const int groups = kThreads / lanes, all = p.q.h + p.k.h;
  int split = 1;
  while (split < groups && 4 * split <= 2 * all && p.tokens * split < int64_t(2) * kBlocks * sms * groups) split *= 2;
  return split;
}

template <typename T, int LANES, bool SHUFFLE, bool GRAD>
void run(const RotaryParams& p, int sms, cudaStream_t s) {
  const int size = sizeof(T);
  const bool vec = p.d % kV == 0 && aligned(p.q, size) && aligned(p.k, size) && aligned(p.oq, size) &&
                   aligned(p.ok, size) && aligned(p.gq, size) && aligned(p.gk, size);
  const int split = head_split(p, sms), groups = kThreads / LANES;
  const int64_t blocks = GRAD ? launch::qk_norm_rotary_blocks(p, sms) : (p.tokens * split + groups - 1) / groups;
  qk_kernel<T, LANES, SHUFFLE, GRAD><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(p, split, vec);
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
  const int groups = kThreads / (p.d <= 64 ? 8 : (p.d <= 128 ? 16 : 32));
  const int64_t all = (p.tokens * head_split(p, sms) + groups - 1) / groups;
  return static_cast<int>(all < kBlocks * sms ? all : kBlocks * sms);  // the resident blocks, further tokens in turn
}

void qk_norm_rotary_forward(const RotaryParams& p, int sms, cudaStream_t s) { by_type<false>(p, sms, s); }

void qk_norm_rotary_backward(const RotaryParams& p, int sms, float* dw, cudaStream_t s) {
  by_type<true>(p, sms, s);
  if (p.partial != nullptr)
    gains_kernel<<<(2 * p.d + 31) / 32, 256, 0, s>>>(p.partial, qk_norm_rotary_blocks(p, sms), 2 * p.d, dw);
}

}  // namespace launch
}  // namespace bitscom_b200
