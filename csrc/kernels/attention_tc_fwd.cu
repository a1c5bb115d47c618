// Masked attention forward on the 5th-generation tensor cores.
//
// One CTA holds a tile of 128 rows of queries and walks over its visible keys,
// 128 at a time: S = Q K^T into TMEM, softmax with the running maximum and sum in
// registers (one thread a row), P as 16-bit values back into TMEM, O += P V with
// P as the TMEM operand.  S, P and O never leave the SM.
//
//   warps 0-3  softmax: row r of the tile is thread r
//   warp 4     copies: Q once, then K and V tiles through tensor maps
//   warp 5     issues the MMAs (and clears padding rows of a tile)
//
// What bounds it: a score costs one exponential, 16 a clock and SM, and 4 D
// operations, 8192 a clock and SM, so up to D = 128 the exponentials are the
// floor (D = 64: twice the MMA time).  Two CTAs share an SM (256 TMEM columns,
// at most 97 KB each), so one's softmax runs beside the other's MMAs, copies,
// start and end; registers are moved from the copy warps to the softmax warps so
// that a row's 128 scores stay in registers between the maximum and the
// exponentials.
//
// The running maximum is only followed when it grows by more than 4 (a factor of
// 16 in P), so most tiles do not touch O; the sum uses the same reference, so the
// result is the same up to rounding.
//
// Few rows: the rows of query heads that share a key head are packed into one
// tile (the cache is read once), and the keys are split over CTAs when there are
// fewer tiles than CTA places; each split writes its normalised fp32 result and log-sum,
// and a second kernel joins them in a fixed order.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>

#include "attention_tc.cuh"
#include "attention_tc_host.h"

namespace bitscom_b200 {

namespace {

__device__ int attn_status = 0;

constexpr int kThreads = 256;
constexpr float kFollow = 4.f;

// Q, then KS tiles of K and VS of V.
template <int D>
struct Shape {
  static constexpr int kTileBytes = kAttnTile * D * 2;
  static constexpr int kStages = D == 64 ? 2 : 1;
  static constexpr int kSmem = kTileBytes * (1 + 2 * kStages) + 1024;
  static constexpr bool kOwnP = D == 64;  // P has columns of its own, else it takes S's
  static constexpr int kColP = kOwnP ? 128 : 0;
  static constexpr int kColO = D == 64 ? 192 : 128;
};

struct FwdParams {
  AttnParams a;
  int packed;  // query heads of one key head in one tile
  int tiles_q;
  int* status;
};

struct Barriers {
  uint64_t q_full, s_full, s_free, p_full, pv_done, drain;
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
};

template <typename T, int D, bool GENERAL>
__global__ void __launch_bounds__(kThreads, 2)
    fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v, const __grid_constant__ FwdParams fp) {
  using S = Shape<D>;
  const AttnParams& p = fp.a;
  extern __shared__ char smem_raw[];
  __shared__ Barriers bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int raised;
  char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* sq = base;
  char* sk = base + S::kTileBytes;
  char* sv = sk + S::kStages * S::kTileBytes;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // Tiles with the most keys first: the last rows of a causal mask.
  const int group = p.hq / p.hk;
  const int heads = fp.packed ? p.hk : p.hq;
  int id = blockIdx.x;
  const int split = id % p.splits;
  id /= p.splits;
  const int h = id % heads;
  id /= heads;
  const int b = id % p.b;
  const int qt = fp.tiles_q - 1 - id / p.b;
  const int kv_head = fp.packed ? h : h / group;

  const int4 tr = [&] {
    if (fp.packed && p.plan.tile == nullptr)  // all rows of the row tile at once
      return p.causal ? make_int4(0, max(0, p.sk), 0, max(0, p.sk - p.sq + 1)) : make_int4(0, p.sk, 0, p.sk);
    return attn_tile_range(p, b, qt);
  }();
  int t0 = tr.x / kAttnTile, t1 = (tr.y + kAttnTile - 1) / kAttnTile;
  if (p.splits > 1) {
    t0 = max(t0, split * p.split_tiles);
    t1 = min(t1, (split + 1) * p.split_tiles);
  }
  const int n = max(0, t1 - t0);

  if (warp == 5) {
    tmem_alloc(&tmem_slot, 256);
  } else if (threadIdx.x == 128) {
    prefetch_tensor_map(&map_q);
    prefetch_tensor_map(&map_k);
    prefetch_tensor_map(&map_v);
    raised = 0;
    mbar_init(&bar.q_full, 1);
    mbar_init(&bar.s_full, 1);
    mbar_init(&bar.s_free, 128);
    mbar_init(&bar.p_full, 128);
    mbar_init(&bar.pv_done, 1);
    mbar_init(&bar.drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.k_full[i], 1);
      mbar_init(&bar.k_empty[i], 1);
      mbar_init(&bar.v_full[i], 1);
      mbar_init(&bar.v_empty[i], 1);
    }
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const Guard guard{&raised, fp.status};

  if (warp >= 4) {
    regs_down<56>();
    if (warp == 4 && n > 0) {
      if (elect_one()) {
        const int rows_q = fp.packed ? group * p.sq : kAttnTile;  // rows of the tensor map's box
        mbar_arrive_expect_tx(&bar.q_full, rows_q * D * 2);
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(sq + c * kAttnTile * 128, &map_q, &bar.q_full, c * 64, fp.packed ? 0 : qt * kAttnTile,
                      fp.packed ? h * group : h, b);
        int j = 0;
        for (; j < n; ++j) {
          const int st = j % S::kStages, ph = (j / S::kStages) & 1;
          if (!guard.wait(&bar.k_empty[st], ph ^ 1)) break;
          mbar_arrive_expect_tx(&bar.k_full[st], S::kTileBytes);
          for (int c = 0; c < D / 64; ++c)
            tma_load_4d(sk + st * S::kTileBytes + c * kAttnTile * 128, &map_k, &bar.k_full[st], c * 64,
                        (t0 + j) * kAttnTile, kv_head, b);
          if (!guard.wait(&bar.v_empty[st], ph ^ 1)) {  // K of this tile is on its way, V is not
            Guard::drain(&bar.k_full[st], ph);
            break;
          }
          mbar_arrive_expect_tx(&bar.v_full[st], S::kTileBytes);
          for (int c = 0; c < D / 64; ++c)
            tma_load_4d(sv + st * S::kTileBytes + c * kAttnTile * 128, &map_v, &bar.v_full[st], c * 64,
                        (t0 + j) * kAttnTile, kv_head, b);
        }
        // No copy may be in flight when the block leaves: the last ones of each stage.
        if (raised) {
          Guard::drain(&bar.q_full, 0);
          for (int i = max(0, j - S::kStages); i < j; ++i) {
            Guard::drain(&bar.k_full[i % S::kStages], (i / S::kStages) & 1);
            Guard::drain(&bar.v_full[i % S::kStages], (i / S::kStages) & 1);
          }
        }
      }
      __syncwarp();
    } else if (warp == 5 && n > 0) {
      constexpr uint32_t kQK = mma_desc<T>(128, 128, false, false);
      constexpr uint32_t kPV = mma_desc<T>(128, D, false, true);
      const uint32_t aq = smem_addr(sq), ak = smem_addr(sk), av = smem_addr(sv);
      const int nk = (p.sk + kAttnTile - 1) / kAttnTile;
      const uint4* dead = p.plan.kdead != nullptr ? p.plan.kdead + static_cast<int64_t>(b) * nk + t0 : nullptr;
      const bool leader = elect_one();
      bool ok = guard.wait_warp(&bar.q_full, 0);
      // S of tile j; padding keys are cleared first, whatever they hold.
      auto scores = [&](int j) {
        const int st = j % S::kStages;
        if (!(ok = ok && guard.wait_warp(&bar.k_full[st], (j / S::kStages) & 1))) return;
        if (dead != nullptr) {
          const uint4 w = dead[j];
          if (any_bit(w)) {
            zero_dead_rows(sk + st * S::kTileBytes, D / 64, w, lane);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        tc_fence_after();
        if (leader) {
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k / 4) * kAttnTile * 128 + (k % 4) * 32;
            mma_ss(tmem, smem_desc(aq + off, 16, 1024), smem_desc(ak + st * S::kTileBytes + off, 16, 1024), kQK, k > 0);
          }
          mma_commit(&bar.k_empty[st]);
          mma_commit(&bar.s_full);
        }
        __syncwarp();
      };
      scores(0);
      for (int j = 0; j < n && ok; ++j) {
        if (S::kOwnP && j + 1 < n) {
          if (!(ok = guard.wait_warp(&bar.s_free, j & 1))) break;
          scores(j + 1);
        }
        const int st = j % S::kStages;
        if (!(ok = ok && guard.wait_warp(&bar.v_full[st], (j / S::kStages) & 1))) break;
        if (dead != nullptr) {
          const uint4 w = dead[j];
          if (any_bit(w)) {
            zero_dead_rows(sv + st * S::kTileBytes, D / 64, w, lane);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        if (!(ok = guard.wait_warp(&bar.p_full, j & 1))) break;
        tc_fence_after();
        if (leader) {
          for (int k = 0; k < kAttnTile / 16; ++k)
            mma_ts(tmem + S::kColO, tmem + S::kColP + k * 8,
                   smem_desc(av + st * S::kTileBytes + k * 2048, kAttnTile * 128, 1024), kPV, j > 0 || k > 0);
          mma_commit(&bar.v_empty[st]);
          mma_commit(&bar.pv_done);
        }
        __syncwarp();
        if (!S::kOwnP && j + 1 < n) {  // the next S overwrites this P
          if (!(ok = guard.wait_warp(&bar.pv_done, j & 1))) break;
          scores(j + 1);
        }
      }
      if (!ok) {  // no MMA may be in flight when TMEM is freed
        if (leader) {
          mma_commit(&bar.drain);
          Guard::drain(&bar.drain, 0);
        }
        __syncwarp();
      }
    }
  } else {
    regs_up<200>();
    const int r = threadIdx.x;
    const int i = fp.packed ? r % p.sq : qt * kAttnTile + r;
    const int head = fp.packed ? h * group + r / p.sq : h;
    const bool valid = fp.packed ? r < group * p.sq : i < p.sq;
    const int2 range = valid ? attn_row_range(p, b, i) : make_int2(0, 0);
    const bool warp_works = __any_sync(0xffffffffu, range.y > range.x);
    const int pos = i + p.sk - p.sq;
    const ScoreScale sc = ScoreScale::of(p, valid ? head : 0);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      if (!(ok = guard.wait_warp(&bar.s_full, j & 1))) break;
      tc_fence_after();
      if (!warp_works) {  // rows of no use: their P is never looked at
        if (S::kOwnP) mbar_arrive(&bar.s_free);
        if (j > 0 && !(ok = guard.wait_warp(&bar.pv_done, (j - 1) & 1))) break;
        mbar_arrive(&bar.p_full);
        continue;
      }
      const int key0 = (t0 + j) * kAttnTile;
      float s[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(lanes + c * 32, reinterpret_cast<uint32_t*>(s) + c * 32);
      tmem_wait_ld();
      if (S::kOwnP) {
        tc_fence_before();
        mbar_arrive(&bar.s_free);
      }
      if (GENERAL) {  // base-2 scores in place
        if (p.cap > 0.f) {
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = tanh_ex2(s[c] * sc.cap_in) * sc.cap_out;
        } else {
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] *= sc.c;
        }
        if (p.slopes != nullptr) {
          const float d0 = static_cast<float>(key0 - pos);
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = fmaf(-sc.slope, fabsf(d0 + c), s[c]);
        }
      }
      if (!(tr.z <= key0 && tr.w >= key0 + kAttnTile)) {
        const unsigned len = static_cast<unsigned>(range.y - range.x), from = static_cast<unsigned>(key0 - range.x);
#pragma unroll
        for (int c = 0; c < 128; ++c) s[c] = from + c < len ? s[c] : -INFINITY;
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c < 128; c += 4)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[c + e]);
      float best = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      if (!GENERAL) best *= sc.c;  // the factor is positive
      // P of the last tile has to be read, and O to be whole, before either is written.
      if (j > 0) {
        if (!(ok = guard.wait_warp(&bar.pv_done, (j - 1) & 1))) break;
        tc_fence_after();
      }
      if (__any_sync(0xffffffffu, best > m + kFollow)) {
        const float mn = fmaxf(m, best);
        const float f = mn == -INFINITY ? 1.f : ex2(m - mn);
        m = mn;
        l *= f;
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(lanes + S::kColO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(lanes + S::kColO + c * 32, o);
          }
        }
      }
      const float ref = (m == -INFINITY ? 0.f : m) - prob_shift<T>();
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int at = c * 32 + e * 2;
          const float x = ex2(GENERAL ? s[at] - ref : fmaf(s[at], sc.c, -ref));
          const float y = ex2(GENERAL ? s[at + 1] - ref : fmaf(s[at + 1], sc.c, -ref));
          sum[e & 3] += x + y;
          w[e] = pack2<T>(x, y);
        }
        tmem_st16(lanes + S::kColP + c * 16, w);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bar.p_full);
    }
    if (ok && n > 0) {
      ok = guard.wait_warp(&bar.pv_done, (n - 1) & 1);
      tc_fence_after();
    }
    // A row that sees nothing is zero; after a wait that ran out, rows are NaN.
    const bool none = l == 0.f && m == -INFINITY;
    const float f = !ok ? __int_as_float(0x7fc00000) : (none ? 0.f : 1.f / l);
    const int64_t row = (static_cast<int64_t>(b) * p.hq + head) * p.sq + i;
    if (warp_works || n == 0 || !ok || __any_sync(0xffffffffu, valid)) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        if (n > 0 && ok) {
          tmem_ld32(lanes + S::kColO + c * 32, reinterpret_cast<uint32_t*>(o));
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = (n > 0 && !none) || !ok ? (ok ? o[e] : 1.f) * f : 0.f;
        if (!valid) continue;
        if (p.splits > 1) {
          float* dst = p.part_o + (split * (static_cast<int64_t>(p.b) * p.hq * p.sq) + row) * p.d + c * 32;
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (c * 32 + e < p.d) *reinterpret_cast<float4*>(dst + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else {
          const int64_t at = b * p.o.sb + head * p.o.sh + i * p.o.ss + c * 32;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (c * 32 + e >= p.d) continue;
            uint4 w;
            uint32_t* wp = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int k = 0; k < 4; ++k) wp[k] = pack2<T>(o[e + 2 * k], o[e + 2 * k + 1]);
            *reinterpret_cast<uint4*>(static_cast<T*>(p.o.ptr) + at + e) = w;
            if (p.lo.ptr != nullptr) {
              const T* hi = reinterpret_cast<const T*>(&w);
              uint4 v;
              uint32_t* vp = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                vp[k] = pack2<T>(o[e + 2 * k] - to_f32<T>(hi[2 * k]), o[e + 2 * k + 1] - to_f32<T>(hi[2 * k + 1]));
              *reinterpret_cast<uint4*>(static_cast<T*>(p.lo.ptr) + at + e) = v;
            }
          }
        }
      }
    }
    if (valid) {
      const float lse = ok ? m + log2f(l) - prob_shift<T>() : __int_as_float(0x7fc00000);
      if (p.splits > 1)
        p.part_lse[split * (static_cast<int64_t>(p.b) * p.hq * p.sq) + row] = none && ok ? -INFINITY : lse;
      else if (p.lse != nullptr)
        p.lse[row] = none && ok ? INFINITY : lse;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_free(tmem, 256);
}

// Joins the splits of a row: sum of 2^(lse_s - max) o_s over their sum.  One warp a row.
template <typename T>
__global__ void __launch_bounds__(128) join_kernel(const FwdParams fp) {
  const AttnParams& p = fp.a;
  const int64_t rows = static_cast<int64_t>(p.b) * p.hq * p.sq;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 32;
  if (row >= rows) return;
  const int lane = threadIdx.x % 32;
  float m = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, p.part_lse[s * rows + row]);
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float total = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  const int col = lane * 4;
  for (int s = 0; s < p.splits; ++s) {
    const float w = ex2(p.part_lse[s * rows + row] - ref);
    total += w;
    if (col < p.d && w != 0.f) {
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * p.d + col);
      o[0] += w * v.x; o[1] += w * v.y; o[2] += w * v.z; o[3] += w * v.w;
    }
  }
  const bool none = m == -INFINITY;
  const float f = none ? 0.f : 1.f / total;
  const int i = row % p.sq, h = row / p.sq % p.hq, b = row / (static_cast<int64_t>(p.sq) * p.hq);
  if (col < p.d) {
    const int64_t at = b * p.o.sb + h * p.o.sh + i * p.o.ss + col;
    for (int e = 0; e < 4; ++e) {
      const float x = o[e] * f;
      const T hi = from_f32<T>(x);
      static_cast<T*>(p.o.ptr)[at + e] = hi;
      if (p.lo.ptr != nullptr) static_cast<T*>(p.lo.ptr)[at + e] = from_f32<T>(x - to_f32<T>(hi));
    }
  }
  if (lane == 0 && p.lse != nullptr) p.lse[row] = none ? INFINITY : m + log2f(total);
}

template <typename T, int D, bool GENERAL>
cudaError_t run(const FwdParams& fp, cudaStream_t s) {
  const AttnParams& p = fp.a;
  CUtensorMap q, k, v;
  const int group = p.hq / p.hk;
  if (!attn_map(&q, p.q, p, p.hq, p.sq, fp.packed ? p.sq : kAttnTile, fp.packed ? group : 1) ||
      !attn_map(&k, p.k, p, p.hk, p.sk, kAttnTile, 1) || !attn_map(&v, p.v, p, p.hk, p.sk, kAttnTile, 1))
    return cudaErrorInvalidValue;
  const auto kernel = fwd_kernel<T, D, GENERAL>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
  if (e != cudaSuccess) return e;
  const int64_t blocks = static_cast<int64_t>(fp.tiles_q) * p.b * (fp.packed ? p.hk : p.hq) * p.splits;
  kernel<<<static_cast<unsigned>(blocks), kThreads, Shape<D>::kSmem, s>>>(q, k, v, fp);
  if (p.splits > 1) {
    const int64_t rows = static_cast<int64_t>(p.b) * p.hq * p.sq;
    join_kernel<T><<<static_cast<unsigned>((rows + 3) / 4), 128, 0, s>>>(fp);
  }
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t by_scores(const FwdParams& fp, cudaStream_t s) {
  return fp.a.cap > 0.f || fp.a.slopes != nullptr ? run<T, D, true>(fp, s) : run<T, D, false>(fp, s);
}

bool packs(const AttnParams& p) { return p.hq > p.hk && p.hq / p.hk * p.sq <= kAttnTile; }

}  // namespace

bool attn_map(CUtensorMap* m, const AttnTensor& t, const AttnParams& p, int heads, int len, int box_rows, int box_heads) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.d), static_cast<cuuint64_t>(len), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(p.b)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(t.ss) * 2, static_cast<cuuint64_t>(t.sh) * 2,
                                 static_cast<cuuint64_t>(t.sb) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(box_heads), 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  return cuTensorMapEncodeTiled(m, p.dt == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                                t.ptr, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int* attn_status_ptr() {
  int* p = nullptr;
  cudaGetSymbolAddress(reinterpret_cast<void**>(&p), attn_status);
  return p;
}

namespace launch {

int attention_status(bool reset) {
  int v = 0;
  const int zero = 0;
  cudaMemcpyFromSymbol(&v, attn_status, sizeof(int));
  if (reset) cudaMemcpyToSymbol(attn_status, &zero, sizeof(int));
  return v;
}

// Key ranges of a forward launch.  Splitting pays when the row tiles leave most
// of the two CTA places an SM empty; a split of fewer than four tiles would
// spend more on its start and the joining than it saves.
void attention_tc_splits(const AttnParams& p, int sms, int* splits, int* split_tiles) {
  const int64_t tiles_q = packs(p) ? 1 : (p.sq + kAttnTile - 1) / kAttnTile;
  const int64_t ctas = tiles_q * p.b * (packs(p) ? p.hk : p.hq);
  const int tiles = (p.sk + kAttnTile - 1) / kAttnTile;
  int64_t n = 2 * sms / std::max<int64_t>(1, ctas);
  n = std::min<int64_t>(n, tiles / 4);
  if (n <= 1) {
    *splits = 1;
    *split_tiles = tiles;
    return;
  }
  *split_tiles = static_cast<int>((tiles + n - 1) / n);
  *splits = (tiles + *split_tiles - 1) / *split_tiles;
}

cudaError_t attention_tc_forward(const AttnParams& p, cudaStream_t s) {
  FwdParams fp{};
  fp.a = p;
  fp.packed = packs(p);
  fp.tiles_q = fp.packed ? 1 : (p.sq + kAttnTile - 1) / kAttnTile;
  fp.status = attn_status_ptr();
  if (p.dt == kBF16) return p.d <= 64 ? by_scores<__nv_bfloat16, 64>(fp, s) : by_scores<__nv_bfloat16, 128>(fp, s);
  return p.d <= 64 ? by_scores<__half, 64>(fp, s) : by_scores<__half, 128>(fp, s);
}

}  // namespace launch
}  // namespace bitscom_b200
