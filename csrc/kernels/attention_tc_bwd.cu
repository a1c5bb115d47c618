// Masked attention backward on the 5th-generation tensor cores.
//
//   dq:     a CTA holds 128 rows of Q and dO, forms delta = dout.(o + what its rounding took) for
//           itself and the next kernel, and walks over the rows' keys:
//             S = Q K^T, dP = dO V^T, dS = P (dP - delta), dQ += dS K
//   dk, dv: a CTA holds 128 keys and values and walks over the rows that see them, through all
//           query heads that share the key head:
//             S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//
// Both recompute P from the saved log-sum.  Every gradient element has one owner
// that adds in a fixed order: no atomics, the same bits every time, shared heads
// summed in fp32.  That costs S and dP twice, seven products in place of five.
//
// All accumulators live in TMEM (512 columns, one CTA an SM).  P and dS go back
// to TMEM as 16-bit values and are the TMEM operand of the second products; Q, dO
// and K lie in shared memory once and are read along their columns by the first
// products and along their rows by the second ones.
//
//   warps 0-15 arithmetic: a thread has one lane of TMEM and a quarter of the 128 columns
//   warp 16    copies, warp 17 MMAs
//
// The MMAs of the next tile's S and dP are issued as soon as the arithmetic has read
// (or, where P and dS share their columns, the second product has read) the present
// ones, so that exponentials and products run side by side.
//
// Measured, 16 heads x 4096 rows, causal, dq and dk/dv: D = 64 80 + 103 us (with 8 warps of
// arithmetic and half the columns a thread 11 % slower), D = 128 148 + 138 us, capped 155 + 191 us.
// The tensor cores are busy 30 % of the time and the exponentials 33 to 44 %: the latency of
// a tile's way through the arithmetic warps bounds it.  When key heads x key tiles are
// fewer than the SMs, dk/dv leaves SMs idle and walks its query heads one after another.
#include <cuda_runtime.h>

#include "attention_tc.cuh"
#include "attention_tc_host.h"

namespace bitscom_b200 {
namespace {

constexpr int kCompute = 512;
constexpr int kThreads = kCompute + 64;
constexpr int kPart = 32;  // of the 128 columns: a thread's share
constexpr int kCopier = kCompute / 32, kIssuer = kCopier + 1;

struct BwdParams {
  AttnParams a;
  ScoreScale sc;
  int nq, nk;
  int* status;
};

template <typename T>
constexpr float prob_unshift() { return std::is_same<T, __half>::value ? 0.0009765625f : 1.f; }

template <int D>
struct Shape {
  static constexpr int kTileBytes = kAttnTile * D * 2;
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kRowBytes = 2048;  // per stage: statistics and intervals of 128 rows
  static constexpr int kSmem = kTileBytes * (2 + 2 * kStages) + kRowBytes * kStages + 1024;
};

struct Barriers {
  uint64_t fixed_full, s_full, s_free, p_full, dp_full, ds_full, first_done, second_done, drain;
  uint64_t full[3], empty[3];
};

__device__ __forceinline__ void init_barriers(Barriers& bar, int64_t wait_limit) {
  mbar_init(&bar.fixed_full, 1);
  mbar_init(&bar.s_full, wait_limit == 0 ? 2 : 1);
  mbar_init(&bar.s_free, kCompute);
  mbar_init(&bar.p_full, kCompute);
  mbar_init(&bar.dp_full, 1);
  mbar_init(&bar.ds_full, kCompute);
  mbar_init(&bar.first_done, 1);
  mbar_init(&bar.second_done, 1);
  mbar_init(&bar.drain, 1);
  for (int i = 0; i < 3; ++i) {
    mbar_init(&bar.full[i], 1);
    mbar_init(&bar.empty[i], 1);
  }
  mbar_init_fence();
}

// Behind the barrier at which the roles meet: whether no wait ran out, in which case all copies and products
// are over.  Else they are waited for here, for the whole block, before their places are used again.
// `fixed`: the fixed tiles were copied; `loads`: stages copied.
template <int STAGES>
__device__ __forceinline__ bool over(Barriers& bar, const volatile int* raised, bool fixed, int loads, int warp) {
  if (!*raised) return true;
  if (warp == kCopier && elect_one()) {
    if (fixed) Guard::drain(&bar.fixed_full, 0);
    for (int j = max(0, loads - STAGES); j < loads; ++j) Guard::drain(&bar.full[j % STAGES], (j / STAGES) & 1);
  }
  if (warp == kIssuer && elect_one()) {
    mma_commit(&bar.drain);
    Guard::drain(&bar.drain, 0);
  }
  __syncthreads();
  return false;
}

// The products, from descriptors of whole tiles (an instruction takes 16 values of the
// contraction; addresses in a descriptor count 16 bytes).  Called by one elected thread of a
// converged warp with values that are the same for the whole warp: descriptors built a thread
// at a time take longer than the instructions.
//
// Along the columns of both: 128 x 128, contraction over D.
template <int D>
__device__ __forceinline__ void mma_scores(uint32_t d, uint64_t a, uint64_t b, uint32_t desc) {
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    const uint32_t off = ((k / 4) * kAttnTile * 128 + (k % 4) * 32) / 16;
    mma_ss(d, a + off, b + off, desc, k > 0);
  }
}
// With a TMEM operand: 128 x D, contraction over the 128 rows of b.  The operand's four parts, written by
// different warps, start PART columns apart.
template <int PART>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add) {
#pragma unroll
  for (int k = 0; k < kAttnTile / 16; ++k) mma_ts(d, a + (k / 2) * PART + (k % 2) * 8, b + k * 128, desc, add || k > 0);
}
// Descriptors of a tile read along its columns and along its rows.
__device__ __forceinline__ uint64_t by_columns(uint32_t addr) { return smem_desc(addr, 16, 1024); }
__device__ __forceinline__ uint64_t by_rows(uint32_t addr) { return smem_desc(addr, kAttnTile * 128, 1024); }

// COLS fp32 columns of TMEM (from `col` on) as T, times f, into a staged tile of 128 rows.
template <typename T, int COLS>
__device__ __forceinline__ void stage_tmem_row(uint32_t addr, char* tile, int row, int col, float f, bool some, bool ok) {
#pragma unroll
  for (int c = 0; c < COLS; c += 32) {
    float o[32];
    if (some && ok) {
      tmem_ld32(addr + c, reinterpret_cast<uint32_t*>(o));
      tmem_wait_ld();
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = !ok ? __int_as_float(0x7fc00000) : (some ? o[e] * f : 0.f);
    stage_row<T, false>(tile + (col + c) / 64 * (kAttnTile * 128), nullptr, row, (col + c) % 64 / 8, o);
  }
}

// A staged tile to global memory, once all compute threads have written their part.
template <int D>
__device__ __forceinline__ void store_tile(const CUtensorMap* m, const char* tile, int row, int h, int b) {
  for (int c = 0; c < D / 64; ++c) tma_store_4d(m, tile + c * kAttnTile * 128, c * 64, row, h, b);
  bulk_commit();
}

// --- dq ---------------------------------------------------------------------------------------------------------

template <typename T, int D, Scores MODE>
__global__ void __launch_bounds__(kThreads, 1)
    dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
              const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
              const __grid_constant__ CUtensorMap map_dq, const __grid_constant__ BwdParams bp) {
  using S = Shape<D>;
  constexpr int kColS = 0, kColDP = 128, kColDQ = 256, kColDS = 384;  // dS: 64 columns of its own
  const AttnParams& p = bp.a;
  extern __shared__ char smem_raw[];
  __shared__ Barriers bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int raised, loads;
  __shared__ float partial[4][kAttnTile];
  char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* sq = base;
  char* sdo = base + S::kTileBytes;
  char* skv = base + 2 * S::kTileBytes;  // stages of K, V

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int id = blockIdx.x;
  const int h = id % p.hq;
  id /= p.hq;
  const int b = id % p.b;
  const int qt = bp.nq - 1 - id / p.b;  // the last rows of a causal mask see the most keys
  const int kv_head = h / (p.hq / p.hk);
  const int4 tr = attn_tile_range(p, b, qt);
  const int t0 = tr.x / kAttnTile, n = max(0, (tr.y + kAttnTile - 1) / kAttnTile - t0);

  auto load = [&](int j) {
    const int st = j % S::kStages;
    char* dst = skv + st * 2 * S::kTileBytes;
    mbar_arrive_expect_tx(&bar.full[st], 2 * S::kTileBytes);
    for (int c = 0; c < D / 64; ++c) {
      tma_load_4d(dst + c * kAttnTile * 128, &map_k, &bar.full[st], c * 64, (t0 + j) * kAttnTile, kv_head, b);
      tma_load_4d(dst + S::kTileBytes + c * kAttnTile * 128, &map_v, &bar.full[st], c * 64, (t0 + j) * kAttnTile, kv_head, b);
    }
  };
  if (warp == kIssuer) {
    tmem_alloc(&tmem_slot, 512);
  } else if (warp == kCopier) {  // the first copies are under way before the block meets
    if (elect_one()) {
      raised = loads = 0;
      init_barriers(bar, p.wait_limit);
      if (n > 0) {
        mbar_arrive_expect_tx(&bar.fixed_full, 2 * S::kTileBytes);
        for (int c = 0; c < D / 64; ++c) {
          tma_load_4d(sq + c * kAttnTile * 128, &map_q, &bar.fixed_full, c * 64, qt * kAttnTile, h, b);
          tma_load_4d(sdo + c * kAttnTile * 128, &map_do, &bar.fixed_full, c * 64, qt * kAttnTile, h, b);
        }
        for (int j = 0; j < min(n, S::kStages); ++j) load(j);
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const Guard guard{&raised, bp.status, p.wait_limit};
  bool ok = true;

  if (warp == kCopier) {
    if (n > 0 && elect_one()) {
      int j = min(n, S::kStages);
      for (; j < n; ++j) {
        if (!guard.wait(&bar.empty[j % S::kStages], ((j / S::kStages) & 1) ^ 1)) break;
        load(j);
      }
      loads = j;
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    if (n > 0) {
      constexpr uint32_t kScores = mma_desc<T>(128, 128, false, false);
      constexpr uint32_t kRows = mma_desc<T>(128, D, false, true);
      const uint64_t dq = by_columns(smem_addr(sq)), ddo = by_columns(smem_addr(sdo));
      const uint64_t dkv = by_columns(smem_addr(skv)), dkv_rows = by_rows(smem_addr(skv));
      const uint4* dead = p.plan.kdead != nullptr ? p.plan.kdead + static_cast<int64_t>(b) * bp.nk + t0 : nullptr;
      ok = guard.wait_warp(&bar.fixed_full, 0);
      auto stage = [&](int j) { return static_cast<uint64_t>((j % S::kStages) * (2 * S::kTileBytes / 16)); };
      auto arrived = [&](int j) {  // K and V of tile j; padding keys cleared
        ok = ok && guard.wait_warp(&bar.full[j % S::kStages], (j / S::kStages) & 1);
        if (!ok) return;
        if (dead != nullptr) {
          const uint4 w = dead[j];
          if (any_bit(w)) {
            zero_dead_rows<kAttnTile>(skv + (j % S::kStages) * 2 * S::kTileBytes, 2 * (D / 64), {w.x, w.y, w.z, w.w}, lane);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
      };
      auto scores = [&](int j) {
        if (elect_one()) {
          mma_scores<D>(tmem + kColS, dq, dkv + stage(j), kScores);
          mma_commit(&bar.s_full);
        }
        __syncwarp();
      };
      auto products = [&](int j) {
        if (elect_one()) {
          mma_scores<D>(tmem + kColDP, ddo, dkv + (stage(j) + S::kTileBytes / 16), kScores);
          mma_commit(&bar.dp_full);
        }
        __syncwarp();
      };
      arrived(0);
      if (ok) {
        scores(0);
        products(0);
      }
      for (int j = 0; j < n && ok; ++j) {
        if (j + 1 < n) {
          if (!(ok = guard.wait_warp(&bar.s_free, j & 1))) break;
          arrived(j + 1);
          if (!ok) break;
          tc_fence_after();
          scores(j + 1);
        }
        if (!(ok = guard.wait_warp(&bar.ds_full, j & 1))) break;
        tc_fence_after();
        if (j + 1 < n) products(j + 1);
        if (elect_one()) {
          mma_rows<16>(tmem + kColDQ, tmem + kColDS, dkv_rows + stage(j), kRows, j > 0);
          mma_commit(&bar.empty[j % S::kStages]);
          mma_commit(&bar.second_done);
        }
        __syncwarp();
      }
    }
  } else {
    const int r = (warp % 4) * 32 + lane, part = warp / 4;
    const int i = qt * kAttnTile + r;
    const bool valid = i < p.sq;
    const int2 range = valid ? attn_row_range(p, b, i) : make_int2(0, 0);
    const int pos = i + p.sk - p.sq;
    const float slope = MODE != kPlain && p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.f;
    // delta = dout . (o + what its rounding took), a quarter of the columns a thread; kept for the other kernel.
    float sum = 0.f, lse = INFINITY;
    if (valid) {
      lse = p.lse[(static_cast<int64_t>(b) * p.hq + h) * p.sq + i];
      const int64_t at = b * p.o.sb + h * p.o.sh + i * p.o.ss, at_g = b * p.dout.sb + h * p.dout.sh + i * p.dout.ss;
#pragma unroll
      for (int c = part * (D / 4); c < (part + 1) * (D / 4); c += 8) {
        if (c >= p.d) continue;
        const uint4 uo = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.o.ptr) + at + c);
        const uint4 ul = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.lo.ptr) + at + c);
        const uint4 ug = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.dout.ptr) + at_g + c);
        const T *o = reinterpret_cast<const T*>(&uo), *l = reinterpret_cast<const T*>(&ul), *g = reinterpret_cast<const T*>(&ug);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += (to_f32<T>(o[e]) + to_f32<T>(l[e])) * to_f32<T>(g[e]);
      }
    }
    partial[part][r] = sum;
    asm volatile("bar.sync 1, 512;" ::: "memory");
    static_assert(kCompute == 512, "threads of the barrier");
    // A row without keys: whatever its gradient holds.
    const float delta = lse == INFINITY ? 0.f : (partial[0][r] + partial[1][r]) + (partial[2][r] + partial[3][r]);
    if (part == 0) {
      float* st = p.stats + ((static_cast<int64_t>(b) * p.hq + h) * bp.nq + qt) * 2 * kAttnTile + r;
      st[0] = -lse;
      st[kAttnTile] = delta;
    }
    const float nlse = prob_shift<T>() - lse;
    const Pair nlse2(nlse, nlse), delta2(-delta, -delta), c2(bp.sc.c, bp.sc.c);
    const Pair inv2(bp.sc.cap_inv, bp.sc.cap_inv), one2(1.f, 1.f), minus2(-1.f, -1.f);
    const Pair unshift2(prob_unshift<T>(), prob_unshift<T>());
    const float masked = MODE == kCapped ? bp.sc.masked : -INFINITY;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
    for (int j = 0; j < n; ++j) {
      const int key0 = (t0 + j) * kAttnTile + part * kPart;
      const bool full = tr.z <= key0 && tr.w >= key0 + kPart;
      if (!(ok = guard.wait_warp(&bar.s_full, j & 1))) break;
      tc_fence_after();
      float pf[kPart];  // scores, then probability times the cap's factor
      tmem_ld32(lanes + kColS + part * kPart, reinterpret_cast<uint32_t*>(pf));
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive(&bar.s_free);
      if (MODE == kCapped) cap_scores(pf, bp.sc);
      if (!full) {
        const unsigned len = static_cast<unsigned>(range.y - range.x), from = static_cast<unsigned>(key0 - range.x);
#pragma unroll
        for (int c = 0; c < kPart; ++c) pf[c] = from + c < len ? pf[c] : masked;
      }
      const float d0 = static_cast<float>(key0 - pos);
      // The distance's sign is known (masked pairs do not count): the bias joins the log-sum.
      const bool behind = MODE != kPlain &&
                          __all_sync(0xffffffffu, key0 + kPart - 1 <= pos || (p.causal && p.plan.range == nullptr));
      if (MODE == kPlain || behind || slope == 0.f) {
        const float base = fmaf(slope, d0, nlse);
#pragma unroll
        for (int c = 0; c < kPart; c += 2) {
          const Pair x(pf[c], pf[c + 1]);
          const Pair add = MODE == kPlain ? nlse2 : Pair(fmaf(slope, static_cast<float>(c), base), fmaf(slope, static_cast<float>(c + 1), base));
          float e0, e1;
          (MODE == kCapped ? add2(x, add) : fma2(x, c2, add)).split(e0, e1);
          Pair e(ex2(e0), ex2(e1));
          if (MODE == kCapped) {  // 1 - tanh^2, from the score without the bias
            const Pair u = mul2(x, inv2);
            e = mul2(e, fma2(mul2(u, minus2), u, one2));
          }
          if (prob_unshift<T>() != 1.f) e = mul2(e, unshift2);
          e.split(pf[c], pf[c + 1]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < kPart; ++c) {
          const float u = pf[c] * bp.sc.cap_inv, f = MODE == kCapped ? fmaf(-u, u, 1.f) : 1.f;
          const float x = fmaf(pf[c], MODE == kCapped ? 1.f : bp.sc.c, fmaf(-slope, fabsf(d0 + c), nlse));
          pf[c] = ex2(x) * (f * prob_unshift<T>());
        }
      }
      if (!(ok = guard.wait_warp(&bar.dp_full, j & 1))) break;
      tc_fence_after();
      uint32_t w[kPart / 2];
#pragma unroll
      for (int c = 0; c < kPart / 32; ++c) {
        float dp[32];
        tmem_ld32(lanes + kColDP + part * kPart + c * 32, reinterpret_cast<uint32_t*>(dp));
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float x, y;
          mul2(Pair(pf[c * 32 + e], pf[c * 32 + e + 1]), add2(Pair(dp[e], dp[e + 1]), delta2)).split(x, y);
          dp[e] = x;
          dp[e + 1] = y;
        }
        if (!full) {  // a masked pair is zero, whatever its product is
#pragma unroll
          for (int e = 0; e < 32; ++e) dp[e] = pf[c * 32 + e] == 0.f ? 0.f : dp[e];
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) w[c * 16 + e / 2] = pack2<T>(dp[e], dp[e + 1]);
      }
      if (j > 0) {  // the last dS has been read
        if (!(ok = guard.wait_warp(&bar.second_done, (j - 1) & 1))) break;
        tc_fence_after();
      }
      tmem_st16(lanes + kColDS + part * 16, w);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bar.ds_full);
    }
    if (ok && n > 0) {
      ok = guard.wait_warp(&bar.second_done, (n - 1) & 1);
      tc_fence_after();
    }
  }
  __syncthreads();
  ok = over<S::kStages>(bar, &raised, n > 0, loads, warp);  // Q's place takes the result
  if (warp < 8) {
    const int half = warp / 4, row = (warp % 4) * 32 + lane;
    stage_tmem_row<T, D / 2>(tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16) + kColDQ + half * (D / 2), sq, row,
                             half * (D / 2), p.scale, n > 0, ok);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0) {
    store_tile<D>(&map_dq, sq, qt * kAttnTile, h, b);
    bulk_wait_read();
  }
  if (warp == kIssuer) tmem_free(tmem, 512);
}

// --- dk, dv -----------------------------------------------------------------------------------------------------

// The (query head, row tile) pairs that see a tile of keys, in order.
struct RowTiles {
  const AttnParams* p;
  int b, key0, first, last, group;
  int g, t;
  bool full;  // every row of the tile sees every key
  __device__ bool take() {
    const int4 r = attn_tile_range(*p, b, t);
    full = r.z <= key0 && r.w >= key0 + kAttnTile;
    return r.y > key0 && r.x < key0 + kAttnTile;
  }
  __device__ bool begin() {
    g = 0;
    t = first;
    if (first > last) return false;
    return take() || next();
  }
  __device__ bool next() {
    for (;;) {
      if (++t > last) {
        t = first;
        if (++g == group) return false;
      }
      if (take()) return true;
    }
  }
};

template <typename T, int D, Scores MODE>
__global__ void __launch_bounds__(kThreads, 1)
    dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
               const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
               const __grid_constant__ CUtensorMap map_dk, const __grid_constant__ CUtensorMap map_dv,
               const __grid_constant__ BwdParams bp) {
  using S = Shape<D>;
  // D = 64 leaves room for P and dS beside S and dP; else each warp writes them over
  // the scores that it alone has read.
  constexpr bool kOwn = D == 64;
  constexpr int kPartCols = kOwn ? 16 : 32;
  constexpr int kColS = 0, kColDP = 128, kColDV = 256, kColDK = 256 + D;
  constexpr int kColP = kOwn ? 384 : kColS, kColDS = kOwn ? 448 : kColDP;
  const AttnParams& p = bp.a;
  extern __shared__ char smem_raw[];
  __shared__ Barriers bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int raised, loads, first_tile, last_tile;
  char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* sk = base;
  char* sv = base + S::kTileBytes;
  char* sqd = base + 2 * S::kTileBytes;  // stages of Q, dO
  char* rows = sqd + S::kStages * 2 * S::kTileBytes;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int id = blockIdx.x;
  const int hk = id % p.hk;
  id /= p.hk;
  const int b = id % p.b;
  const int key0 = id / p.b * kAttnTile;  // the first keys of a causal mask are seen by the most rows
  const int group = p.hq / p.hk;

  if (warp == kIssuer) {
    tmem_alloc(&tmem_slot, 512);
  } else if (warp == kCopier) {  // the first copies are under way before the block meets
    if (elect_one()) {
      raised = loads = 0;
      first_tile = 0x7fffffff;
      last_tile = -1;
      init_barriers(bar, p.wait_limit);
      mbar_arrive_expect_tx(&bar.fixed_full, 2 * S::kTileBytes);
      for (int c = 0; c < D / 64; ++c) {
        tma_load_4d(sk + c * kAttnTile * 128, &map_k, &bar.fixed_full, c * 64, key0, hk, b);
        tma_load_4d(sv + c * kAttnTile * 128, &map_v, &bar.fixed_full, c * 64, key0, hk, b);
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (p.plan.tile != nullptr) {  // the first and last row tile that see a key of this tile
    int a = 0x7fffffff, z = -1;
    for (int t = threadIdx.x; t < bp.nq; t += kThreads) {
      const int4 r = attn_tile_range(p, b, t);
      if (r.y > key0 && r.x < key0 + kAttnTile) {
        a = min(a, t);
        z = t;
      }
    }
    a = __reduce_min_sync(0xffffffffu, a);
    z = __reduce_max_sync(0xffffffffu, z);
    if (lane == 0 && z >= 0) {
      atomicMin(&first_tile, a);
      atomicMax(&last_tile, z);
    }
    __syncthreads();
  }
  const uint32_t tmem = tmem_slot;
  const Guard guard{&raised, bp.status, p.wait_limit};
  bool ok = true;
  RowTiles it{&p, b, key0, first_tile, last_tile, group, 0, 0, false};
  if (p.plan.tile == nullptr) {
    it.first = p.causal ? max(0, key0 - (p.sk - p.sq)) / kAttnTile : 0;
    it.last = bp.nq - 1;
  }
  const bool some = it.begin();

  if (warp == kCopier) {
    if (some && elect_one()) {
      int j = 0;
      bool more = true;
      for (; more; ++j, more = it.next()) {
        const int st = j % S::kStages, ph = (j / S::kStages) & 1;
        if (!guard.wait(&bar.empty[st], ph ^ 1)) break;
        const int h = hk * group + it.g;
        char* dst = sqd + st * 2 * S::kTileBytes;
        char* rd = rows + st * S::kRowBytes;
        mbar_arrive_expect_tx(&bar.full[st], 2 * S::kTileBytes + (p.plan.range != nullptr ? 2048 : 1024));
        for (int c = 0; c < D / 64; ++c) {
          tma_load_4d(dst + c * kAttnTile * 128, &map_q, &bar.full[st], c * 64, it.t * kAttnTile, h, b);
          tma_load_4d(dst + S::kTileBytes + c * kAttnTile * 128, &map_do, &bar.full[st], c * 64, it.t * kAttnTile, h, b);
        }
        bulk_g2s(rd, p.stats + ((static_cast<int64_t>(b) * p.hq + h) * bp.nq + it.t) * 2 * kAttnTile, 1024, &bar.full[st]);
        if (p.plan.range != nullptr)
          bulk_g2s(rd + 1024, p.plan.range + (static_cast<int64_t>(b) * bp.nq + it.t) * kAttnTile, 1024, &bar.full[st]);
      }
      loads = j;
    }
    if (!some) Guard::drain(&bar.fixed_full, 0);
    __syncwarp();
  } else if (warp == kIssuer) {
    if (some) {
      constexpr uint32_t kScores = mma_desc<T>(128, 128, false, false);
      constexpr uint32_t kRows = mma_desc<T>(128, D, false, true);
      const uint64_t dk = by_columns(smem_addr(sk)), dv = by_columns(smem_addr(sv));
      const uint64_t dqd = by_columns(smem_addr(sqd)), dqd_rows = by_rows(smem_addr(sqd));
      ok = guard.wait_warp(&bar.fixed_full, 0);
      auto stage = [&](int j) { return static_cast<uint64_t>((j % S::kStages) * (2 * S::kTileBytes / 16)); };
      auto arrived = [&](int j) {  // Q and dO of step j; rows without keys cleared
        ok = ok && guard.wait_warp(&bar.full[j % S::kStages], (j / S::kStages) & 1);
        if (!ok || it.full) return;
        const uint4 w = attn_tile_qdead(p, b, it.t);
        if (any_bit(w)) {
          zero_dead_rows<kAttnTile>(sqd + (j % S::kStages) * 2 * S::kTileBytes, 2 * (D / 64), {w.x, w.y, w.z, w.w}, lane);
          fence_proxy_async_smem();
          __syncwarp();
        }
      };
      auto scores = [&](int j) {
        if (elect_one()) {
          mma_scores<D>(tmem + kColS, dk, dqd + stage(j), kScores);
          mma_commit(&bar.s_full);
        }
        __syncwarp();
      };
      auto products = [&](int j) {
        if (elect_one()) {
          mma_scores<D>(tmem + kColDP, dv, dqd + (stage(j) + S::kTileBytes / 16), kScores);
          mma_commit(&bar.dp_full);
        }
        __syncwarp();
      };
      auto add_dv = [&](int j) {
        if (elect_one()) {
          mma_rows<kPartCols>(tmem + kColDV, tmem + kColP, dqd_rows + (stage(j) + S::kTileBytes / 16), kRows, j > 0);
          mma_commit(&bar.first_done);
        }
        __syncwarp();
      };
      auto add_dk = [&](int j) {
        if (elect_one()) {
          mma_rows<kPartCols>(tmem + kColDK, tmem + kColDS, dqd_rows + stage(j), kRows, j > 0);
          mma_commit(&bar.empty[j % S::kStages]);
          mma_commit(&bar.second_done);
        }
        __syncwarp();
      };
      arrived(0);
      if (ok) {
        scores(0);
        products(0);
      }
      bool more = ok;
      for (int j = 0; more && ok; ++j) {
        more = it.next();
        if (!(ok = guard.wait_warp(&bar.p_full, j & 1))) break;
        tc_fence_after();
        if (kOwn) {
          if (more) {
            arrived(j + 1);
            if (!ok) break;
            scores(j + 1);
          }
          add_dv(j);
        } else {
          add_dv(j);
          if (more) {
            arrived(j + 1);
            if (!(ok = ok && guard.wait_warp(&bar.first_done, j & 1))) break;
            scores(j + 1);
          }
        }
        if (!(ok = guard.wait_warp(&bar.ds_full, j & 1))) break;
        tc_fence_after();
        if (kOwn) {
          if (more) products(j + 1);
          add_dk(j);
        } else {
          add_dk(j);
          if (more) {
            if (!(ok = guard.wait_warp(&bar.second_done, j & 1))) break;
            products(j + 1);
          }
        }
      }
    }
  } else {
    const int r = (warp % 4) * 32 + lane, part = warp / 4;
    const int key = key0 + r;
    const Pair c2(bp.sc.c, bp.sc.c), inv2(bp.sc.cap_inv, bp.sc.cap_inv), one2(1.f, 1.f), minus2(-1.f, -1.f);
    const Pair unshift2(prob_unshift<T>(), prob_unshift<T>());
    const float masked = MODE == kCapped ? bp.sc.masked : -INFINITY;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
    bool more = some;
    int j = 0;
    for (; more; ++j) {
      const int st = j % S::kStages;
      const float* stats = reinterpret_cast<const float*>(rows + st * S::kRowBytes) + part * kPart;
      const int2* range = reinterpret_cast<const int2*>(rows + st * S::kRowBytes + 1024) + part * kPart;
      const int row0 = it.t * kAttnTile + part * kPart;
      const bool full = it.full;
      const float slope = MODE != kPlain && p.slopes != nullptr ? p.slopes[hk * group + it.g] * kLog2e : 0.f;
      more = it.next();
      if (!(ok = guard.wait_warp(&bar.full[st], (j / S::kStages) & 1) && guard.wait_warp(&bar.s_full, j & 1))) break;
      tc_fence_after();
      float pf[kPart];  // scores, then probability times the cap's factor
      tmem_ld32(lanes + kColS + part * kPart, reinterpret_cast<uint32_t*>(pf));
      tmem_wait_ld();
      if (MODE == kCapped) cap_scores(pf, bp.sc);
      const int first_pos = row0 + p.sk - p.sq;
      if (!full) {
        if (p.plan.range != nullptr) {
#pragma unroll
          for (int c = 0; c < kPart; c += 2) {
            const int4 v = *reinterpret_cast<const int4*>(range + c);
            pf[c] = key >= v.x && key < v.y ? pf[c] : masked;
            pf[c + 1] = key >= v.z && key < v.w ? pf[c + 1] : masked;
          }
        } else if (p.causal) {  // rows from position `key` on
#pragma unroll
          for (int c = 0; c < kPart; ++c) pf[c] = c >= key - first_pos ? pf[c] : masked;
        }
      }
      uint32_t w[kPart / 2];
      // Distances are row - key here.  With a known sign (masked pairs do not count) they go two at a time.
      const float d0 = static_cast<float>(first_pos - key);
      const bool ahead = MODE != kPlain &&
                         __all_sync(0xffffffffu, first_pos >= key || (p.causal && p.plan.range == nullptr));
      const float base = prob_shift<T>() - slope * d0;
      const Pair shift2(prob_shift<T>(), prob_shift<T>());
#pragma unroll
      for (int c = 0; c < kPart; c += 4) {
        const float4 nl = *reinterpret_cast<const float4*>(stats + c);
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const Pair x(pf[c + e], pf[c + e + 1]);
          Pair add = e == 0 ? Pair(nl.x, nl.y) : Pair(nl.z, nl.w);
          if (MODE != kPlain) {
            if (ahead)
              add = add2(add, Pair(fmaf(-slope, static_cast<float>(c + e), base), fmaf(-slope, static_cast<float>(c + e + 1), base)));
            else
              add = add2(add, Pair(fmaf(-slope, fabsf(d0 + (c + e)), prob_shift<T>()),
                                   fmaf(-slope, fabsf(d0 + (c + e + 1)), prob_shift<T>())));
          } else if (prob_shift<T>() != 0.f) {
            add = add2(add, shift2);
          }
          float p0, p1;
          (MODE == kCapped ? add2(x, add) : fma2(x, c2, add)).split(p0, p1);
          p0 = ex2(p0);
          p1 = ex2(p1);
          w[(c + e) / 2] = pack2<T>(p0, p1);
          Pair f(p0, p1);
          if (MODE == kCapped) {  // 1 - tanh^2, from the score without the bias
            const Pair u = mul2(x, inv2);
            f = mul2(f, fma2(mul2(u, minus2), u, one2));
          }
          if (prob_unshift<T>() != 1.f) f = mul2(f, unshift2);
          f.split(pf[c + e], pf[c + e + 1]);
        }
      }
      if (kOwn && j > 0) {  // the last P has been read
        if (!(ok = guard.wait_warp(&bar.first_done, (j - 1) & 1))) break;
        tc_fence_after();
      }
      tmem_st16(lanes + kColP + part * kPartCols, w);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bar.p_full);
      if (!(ok = guard.wait_warp(&bar.dp_full, j & 1))) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kPart / 32; ++c) {
        float dp[32];
        tmem_ld32(lanes + kColDP + part * kPart + c * 32, reinterpret_cast<uint32_t*>(dp));
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 dl = *reinterpret_cast<const float4*>(stats + kAttnTile + c * 32 + e);
          mul2(Pair(pf[c * 32 + e], pf[c * 32 + e + 1]), fma2(Pair(dl.x, dl.y), minus2, Pair(dp[e], dp[e + 1]))).split(dp[e], dp[e + 1]);
          mul2(Pair(pf[c * 32 + e + 2], pf[c * 32 + e + 3]), fma2(Pair(dl.z, dl.w), minus2, Pair(dp[e + 2], dp[e + 3])))
              .split(dp[e + 2], dp[e + 3]);
        }
        if (!full) {  // a masked pair is zero, whatever its product is
#pragma unroll
          for (int e = 0; e < 32; ++e) dp[e] = pf[c * 32 + e] == 0.f ? 0.f : dp[e];
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) w[c * 16 + e / 2] = pack2<T>(dp[e], dp[e + 1]);
      }
      if (kOwn && j > 0) {  // the last dS has been read
        if (!(ok = guard.wait_warp(&bar.second_done, (j - 1) & 1))) break;
        tc_fence_after();
      }
      tmem_st16(lanes + kColDS + part * kPartCols, w);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bar.ds_full);
    }
    if (ok && some) {
      ok = guard.wait_warp(&bar.second_done, (j - 1) & 1);
      tc_fence_after();
    }
  }
  __syncthreads();
  ok = over<S::kStages>(bar, &raised, true, loads, warp);  // the places of K and V take their gradients
  if (warp < 8) {
    const int col = warp / 4 * (D / 2), row = (warp % 4) * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
    stage_tmem_row<T, D / 2>(lanes + kColDV + col, sv, row, col, prob_unshift<T>(), some, ok);
    stage_tmem_row<T, D / 2>(lanes + kColDK + col, sk, row, col, p.scale, some, ok);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0) {
    store_tile<D>(&map_dv, sv, key0, hk, b);
    store_tile<D>(&map_dk, sk, key0, hk, b);
    bulk_wait_read();
  }
  if (warp == kIssuer) tmem_free(tmem, 512);
}

template <typename T, int D, Scores MODE>
cudaError_t run(const BwdParams& bp, cudaStream_t s) {
  const AttnParams& p = bp.a;
  CUtensorMap q, g, k, v, dq, dk, dv;
  if (!attn_map(&q, p.q, p, p.hq, p.sq, kAttnTile, 1) || !attn_map(&g, p.dout, p, p.hq, p.sq, kAttnTile, 1) ||
      !attn_map(&k, p.k, p, p.hk, p.sk, kAttnTile, 1) || !attn_map(&v, p.v, p, p.hk, p.sk, kAttnTile, 1) || !attn_map(&dq, p.dq, p, p.hq, p.sq, kAttnTile, 1) ||
      !attn_map(&dk, p.dk, p, p.hk, p.sk, kAttnTile, 1) || !attn_map(&dv, p.dv, p, p.hk, p.sk, kAttnTile, 1))
    return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(dq_kernel<T, D, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(dkv_kernel<T, D, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
  if (e != cudaSuccess) return e;
  dq_kernel<T, D, MODE>
      <<<static_cast<unsigned>(static_cast<int64_t>(bp.nq) * p.b * p.hq), kThreads, Shape<D>::kSmem, s>>>(q, g, k, v, dq, bp);
  dkv_kernel<T, D, MODE>
      <<<static_cast<unsigned>(static_cast<int64_t>(bp.nk) * p.b * p.hk), kThreads, Shape<D>::kSmem, s>>>(q, g, k, v, dk, dv, bp);
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t by_scores(const BwdParams& bp, cudaStream_t s) {
  switch (scores_of(bp.a)) {
    case kPlain: return run<T, D, kPlain>(bp, s);
    case kBiased: return run<T, D, kBiased>(bp, s);
    case kCapped: return run<T, D, kCapped>(bp, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

namespace launch {

cudaError_t attention_tc_backward(const AttnParams& p, cudaStream_t s) {
  BwdParams bp{p, ScoreScale::of(p), (p.sq + kAttnTile - 1) / kAttnTile, (p.sk + kAttnTile - 1) / kAttnTile, attn_status_ptr()};
  bp.a.wait_limit = attn_wait_limit();
  if (p.dt == kBF16) return p.d <= 64 ? by_scores<__nv_bfloat16, 64>(bp, s) : by_scores<__nv_bfloat16, 128>(bp, s);
  return p.d <= 64 ? by_scores<__half, 64>(bp, s) : by_scores<__half, 128>(bp, s);
}

}  // namespace launch
}  // namespace bitscom_b200
