// Masked attention forward on the 5th-generation tensor cores.
//
// One CTA holds a tile of 128 rows of queries and walks over its visible keys,
// 64 at a time: S = Q K^T into TMEM, softmax with the running maximum and sum in
// registers, P as 16-bit values back into TMEM over the scores they came from, O += P V
// with P as the TMEM operand.  S, P and O never leave the SM.
//
//   warps 0-3  softmax: a thread takes the 64 scores of a row
//   warp 4     copies of K and V (and Q, D = 128) through tensor maps
//   warp 5     MMAs; clears padding rows of a tile
//
// S has two places in TMEM: the scores of the tile after next are formed when this
// tile's P has been read, so the softmax warps find theirs ready.  D = 64 keeps Q in TMEM
// as well, which halves what S reads from shared memory.  Two CTAs share an SM (256 TMEM
// columns each), one's start and end beside the other's work.
//
// What bounds it: a score costs one exponential, 16 a clock and SM, and 4 D
// operations.  No pipe is full: at D = 64 that of the exponentials is busy 59 % of the
// time and the tensor cores 27 %, and warps wait most for instructions of fixed
// latency (TMEM loads and stores, maxima, votes, barriers), which a tile of 64 keys pays
// once.  16 heads x 4096 rows, causal: D = 64 60 us (570 TFLOP/s), with distance bias 88 us,
// capped 95 us; D = 128 78 us (880 TFLOP/s), capped 104 us.  One query of 16 heads on 4 over 8
// caches of 32768 x 128: 85 us, 92 % of a copy's bandwidth.  A CTA of three tiles alone takes
// 6.8 us with its launch, so short rows are bound by start and end.
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
#include <atomic>

#include "attention_tc.cuh"
#include "attention_tc_host.h"

namespace bitscom_b200 {

namespace {

__device__ int attn_status = 0;
std::atomic<int64_t> wait_limit{kWaitLimitClocks};

constexpr float kFollow = 4.f;
constexpr int kCols = 64;  // scores of a row that a thread takes

template <int D>
struct Shape {
  static constexpr int kKeys = 64;
  static constexpr int kSoftmax = 128;  // threads
  static constexpr int kThreads = kSoftmax + 64;
  static constexpr bool kTmemQ = D == 64;  // D = 128 fills TMEM with S and O
  static constexpr int kColO = 2 * kKeys, kColQ = kColO + D;
  static constexpr int kTmem = 256;
  static constexpr int kQBytes = kTmemQ ? 0 : kAttnTile * D * 2;
  static constexpr int kTileBytes = kKeys * D * 2;
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kSmem = kQBytes + 2 * kStages * kTileBytes + 1024;
};

struct FwdParams {
  AttnParams a;
  ScoreScale sc;
  int packed;  // query heads of one key head in one tile
  int tiles_q;
  int* status;
};

struct Barriers {
  uint64_t q_full, pv_done, o_full, drain;
  uint64_t s_full[2], p_full[2];  // by tile parity
  uint64_t k_full[3], k_empty[3], v_full[3], v_empty[3];
};

template <typename T, int D, Scores MODE>
__global__ void __launch_bounds__(Shape<D>::kThreads, 2)
    fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o,
               const __grid_constant__ CUtensorMap map_lo,
               const __grid_constant__ FwdParams fp) {
  using S = Shape<D>;
  constexpr int kKeys = S::kKeys, kStages = S::kStages;
  const AttnParams& p = fp.a;
  extern __shared__ char smem_raw[];
  __shared__ Barriers bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int raised, loads_k, loads_v;
  char* sq = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* sk = sq + S::kQBytes;
  char* sv = sk + kStages * S::kTileBytes;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  constexpr int kCopier = S::kSoftmax / 32, kIssuer = kCopier + 1;
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

  const int4 tr = [&] {
    if (fp.packed && p.plan.tile == nullptr)  // all rows of the row tile at once
      return p.causal ? make_int4(0, p.sk, 0, max(0, p.sk - p.sq + 1)) : make_int4(0, p.sk, 0, p.sk);
    return attn_tile_range(p, b, qt);
  }();
  int key_lo = tr.x, key_hi = tr.y;
  if (p.splits > 1) {
    key_lo = max(key_lo, split * p.split_tiles * kAttnTile);
    key_hi = min(key_hi, (split + 1) * p.split_tiles * kAttnTile);
  }
  const int t0 = key_lo / kKeys;
  const int n = max(0, (key_hi + kKeys - 1) / kKeys - t0);
  const int kv_head = fp.packed ? h : h / group;
  auto load_k = [&](int j) {
    const int st = j % kStages;
    mbar_arrive_expect_tx(&bar.k_full[st], S::kTileBytes);
    for (int c = 0; c < D / 64; ++c)
      tma_load_4d(sk + st * S::kTileBytes + c * kKeys * 128, &map_k, &bar.k_full[st], c * 64, (t0 + j) * kKeys, kv_head, b);
  };
  auto load_v = [&](int j) {
    const int st = j % kStages;
    mbar_arrive_expect_tx(&bar.v_full[st], S::kTileBytes);
    for (int c = 0; c < D / 64; ++c)
      tma_load_4d(sv + st * S::kTileBytes + c * kKeys * 128, &map_v, &bar.v_full[st], c * 64, (t0 + j) * kKeys, kv_head, b);
  };

  // Everything that takes long starts before the block meets: TMEM, the first copies, Q.
  const int r = (warp % 4) * 32 + lane;  // softmax warps: row of the tile
  const int i = fp.packed ? r % p.sq : qt * kAttnTile + r;
  const int head = fp.packed ? h * group + r / p.sq : h;
  const bool valid = fp.packed ? r < group * p.sq : i < p.sq;
  uint4 q[8];
  if (warp == kIssuer) {
    tmem_alloc(&tmem_slot, S::kTmem);
  } else if (warp == kCopier) {
    if (elect_one()) {
      raised = loads_k = loads_v = 0;
      for (int c = 0; c < kStages; ++c) {
        mbar_init(&bar.k_full[c], 1);
        mbar_init(&bar.k_empty[c], 1);
        mbar_init(&bar.v_full[c], 1);
        mbar_init(&bar.v_empty[c], 1);
      }
      mbar_init(&bar.q_full, S::kTmemQ ? S::kSoftmax : 1);
      mbar_init_fence();
      if (!S::kTmemQ && n > 0) {
        mbar_arrive_expect_tx(&bar.q_full, (fp.packed ? group * p.sq : kAttnTile) * D * 2);
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(sq + c * kAttnTile * 128, &map_q, &bar.q_full, c * 64, fp.packed ? 0 : qt * kAttnTile,
                      fp.packed ? h * group : h, b);
      }
      for (int j = 0; j < min(n, kStages); ++j) {
        load_k(j);
        load_v(j);
      }
      mbar_init(&bar.pv_done, 1);
      mbar_init(&bar.o_full, 1);
      mbar_init(&bar.drain, 1);
      for (int c = 0; c < 2; ++c) {
        mbar_init(&bar.s_full[c], p.wait_limit == 0 ? 2 : 1);
        mbar_init(&bar.p_full[c], S::kSoftmax);
      }
      mbar_init_fence();
    }
    __syncwarp();
  } else if (S::kTmemQ && n > 0) {  // Q is the TMEM operand of S
    const T* src = static_cast<const T*>(p.q.ptr) + b * p.q.sb + head * p.q.sh + i * p.q.ss;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      q[c] = valid && c * 8 < p.d ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0, 0, 0, 0);
  } else if (!S::kTmemQ && fp.packed && !valid) {
    // The copy of packed rows leaves the tile's other rows as the last kernel left them; their scores take
    // part in the warp's votes (which tanh, whether the maximum is followed), so they are zeros.
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        *reinterpret_cast<uint4*>(sq + c * kAttnTile * 128 + r * 128 + e * 16) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const Guard guard{&raised, fp.status, p.wait_limit};

  if (warp == kCopier) {
    if (n > 0 && elect_one()) {
      int k_loads = min(n, kStages), v_loads = k_loads;
      for (int j = kStages; j < n; ++j) {
        const int st = j % kStages, ph = (j / kStages) & 1;
        if (!guard.wait(&bar.k_empty[st], ph ^ 1)) break;
        load_k(j);
        ++k_loads;
        if (!guard.wait(&bar.v_empty[st], ph ^ 1)) break;
        load_v(j);
        ++v_loads;
      }
      loads_k = k_loads;
      loads_v = v_loads;
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    if (n > 0) {
      constexpr uint32_t kQK = mma_desc<T>(128, kKeys, false, false);
      constexpr uint32_t kPV = mma_desc<T>(128, D, false, true);
      const uint64_t dq = smem_desc(smem_addr(sq), 16, 1024), dk = smem_desc(smem_addr(sk), 16, 1024),
                     dv = smem_desc(smem_addr(sv), kKeys * 128, 1024);
      // Padding keys are cleared, whatever they hold.
      auto clear_dead = [&](char* tile, int j) {
        const int first = (t0 + j) * kKeys;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(
                                  &p.plan.kdead[static_cast<int64_t>(b) * ((p.sk + kAttnTile - 1) / kAttnTile) + first / kAttnTile]) +
                              first % kAttnTile / 32;
        uint32_t w[kKeys / 32], any = 0;
#pragma unroll
        for (int i = 0; i < kKeys / 32; ++i) any |= w[i] = src[i];
        if (any != 0u) {
          zero_dead_rows<kKeys>(tile, D / 64, w, lane);
          fence_proxy_async_smem();
          __syncwarp();
        }
      };
      bool ok = guard.wait_warp(&bar.q_full, 0);
      auto k_ready = [&](int j) {
        const int st = j % kStages;
        ok = ok && guard.wait_warp(&bar.k_full[st], (j / kStages) & 1);
        if (ok && p.plan.kdead != nullptr) clear_dead(sk + st * S::kTileBytes, j);
      };
      auto scores = [&](int j) {
        if (elect_one()) {
          const uint64_t d = dk + (j % kStages) * (S::kTileBytes / 16);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t dkk = d + ((k / 4) * kKeys * 128 + (k % 4) * 32) / 16;
            if (S::kTmemQ)
              mma_ts(tmem + (j & 1) * kKeys, tmem + S::kColQ + k * 8, dkk, kQK, k > 0);
            else
              mma_ss(tmem + (j & 1) * kKeys, dq + ((k / 4) * kAttnTile * 128 + (k % 4) * 32) / 16, dkk, kQK, k > 0);
          }
          mma_commit(&bar.k_empty[j % kStages]);
          mma_commit(&bar.s_full[j & 1]);
        }
        __syncwarp();
      };
      for (int j = 0; j < 2 && j < n; ++j) {
        k_ready(j);
        tc_fence_after();
        if (ok) scores(j);
      }
      for (int j = 0; j < n && ok; ++j) {
        const int st = j % kStages;
        if (!(ok = guard.wait_warp(&bar.v_full[st], (j / kStages) & 1))) break;
        if (p.plan.kdead != nullptr) clear_dead(sv + st * S::kTileBytes, j);
        if (!(ok = guard.wait_warp(&bar.p_full[j & 1], (j / 2) & 1))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t d = dv + st * (S::kTileBytes / 16);
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            mma_ts(tmem + S::kColO, tmem + (j & 1) * kKeys + k * 8, d + k * 128, kPV, j > 0 || k > 0);
          mma_commit(&bar.v_empty[st]);
          mma_commit(j + 1 < n ? &bar.pv_done : &bar.o_full);
        }
        __syncwarp();
        if (j + 2 < n) {  // its S takes the place of this P
          k_ready(j + 2);
          if (!(ok = ok && guard.wait_warp(&bar.pv_done, j & 1))) break;
          scores(j + 2);
        }
      }
    }
  } else {
    const int2 range = valid ? attn_row_range(p, b, i) : make_int2(0, 0);
    const bool warp_works = __any_sync(0xffffffffu, range.y > range.x);
    const int pos = i + p.sk - p.sq;
    const float slope = MODE != kPlain && p.slopes != nullptr ? p.slopes[valid ? head : 0] * kLog2e : 0.f;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    if (S::kTmemQ && n > 0) {
      tmem_st32(lanes + S::kColQ, reinterpret_cast<const uint32_t*>(q));
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bar.q_full);
    }
    for (int j = 0; j < n; ++j) {
      const uint32_t col_s = lanes + (j & 1) * kKeys;
      if (!(ok = guard.wait_warp(&bar.s_full[j & 1], (j / 2) & 1))) break;
      tc_fence_after();
      if (!warp_works) {  // rows of no use: their P is never looked at
        mbar_arrive(&bar.p_full[j & 1]);
        continue;
      }
      const int key0 = (t0 + j) * kKeys;
      float s[kCols];
      tmem_ld32(col_s, reinterpret_cast<uint32_t*>(s));
      tmem_ld32(col_s + 32, reinterpret_cast<uint32_t*>(s) + 32);
      tmem_wait_ld();
      if (MODE == kCapped) cap_scores(s, fp.sc);
      if (MODE == kBiased || (MODE == kCapped && slope != 0.f)) {
        const bool behind = __all_sync(0xffffffffu, key0 + kCols - 1 <= pos);
        bias_scores(s, MODE == kBiased ? fp.sc.c : 1.f, slope, static_cast<float>(key0 - pos), behind);
      }
      if (!(tr.z <= key0 && tr.w >= key0 + kCols)) {
        const unsigned len = static_cast<unsigned>(range.y - range.x), from = static_cast<unsigned>(key0 - range.x);
#pragma unroll
        for (int c = 0; c < kCols; ++c) s[c] = from + c < len ? s[c] : -INFINITY;
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c < kCols - 4; c += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(fmaxf(mx[e], s[c + e]), s[c + 4 + e]);
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[kCols - 4 + e]);
      float best = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      if (MODE == kPlain) best *= fp.sc.c;  // the factor is positive
      if (__any_sync(0xffffffffu, best > m + kFollow)) {
        const float mn = fmaxf(m, best);
        const float f = mn == -INFINITY ? 1.f : ex2(m - mn);
        m = mn;
        l *= f;
        if (j > 0) {  // S(j) came after the product j - 2: j - 1 is the one to wait for
          if (!(ok = guard.wait_warp(&bar.pv_done, (j - 1) & 1))) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 8; ++c) {
            const uint32_t at = lanes + S::kColO + c * 8;
            uint32_t o[8];
            tmem_ld8(at, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st8(at, o);
          }
        }
      }
      const float ref = prob_shift<T>() - (m == -INFINITY ? 0.f : m);
      const Pair ref2(ref, ref), c2(fp.sc.c, fp.sc.c);
      Pair sum[2] = {Pair(0.f, 0.f), Pair(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const Pair v(s[c * 32 + e * 2], s[c * 32 + e * 2 + 1]);
          float x, y;
          (MODE != kPlain ? add2(v, ref2) : fma2(v, c2, ref2)).split(x, y);
          x = ex2(x);
          y = ex2(y);
          sum[e & 1] = add2(sum[e & 1], Pair(x, y));
          w[e] = pack2<T>(x, y);
        }
        tmem_st16(col_s + c * 16, w);
      }
      float even, odd;
      add2(sum[0], sum[1]).split(even, odd);
      l += even + odd;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bar.p_full[j & 1]);
    }
    if (ok && n > 0) {
      ok = guard.wait_warp(&bar.o_full, 0);
      tc_fence_after();
    }
    // A row that sees nothing is zero; after a wait that ran out, rows are NaN.
    const bool none = l == 0.f && m == -INFINITY;
    const float f = !ok ? __int_as_float(0x7fc00000) : (none ? 0.f : 1.f / l);
    const int64_t row = (static_cast<int64_t>(b) * p.hq + head) * p.sq + i;
    const bool staged = ok && !fp.packed && p.splits == 1;
    // With o_full all copies are done and read, their place takes the warp's 32 rows, sub-tiles of 64 columns.
    char* tile = sk + warp * 4096 * (D / 64);
    char* low = tile + kAttnTile * D * 2;
    if (__any_sync(0xffffffffu, valid)) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        if (n > 0 && ok) {
          tmem_ld32(lanes + S::kColO + c * 32, reinterpret_cast<uint32_t*>(o));
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = (n > 0 && !none) || !ok ? (ok ? o[e] : 1.f) * f : 0.f;
        if (staged) {
          if (p.lo.ptr != nullptr)
            stage_row<T, true>(tile + c / 2 * 4096, low + c / 2 * 4096, lane, c % 2 * 4, o);
          else
            stage_row<T, false>(tile + c / 2 * 4096, low + c / 2 * 4096, lane, c % 2 * 4, o);
        } else if (valid) {  // few rows: straight from the thread
          const int col = c * 32;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (col + e >= p.d) continue;
            if (p.splits > 1) {
              float* dst = p.part_o + (split * (static_cast<int64_t>(p.b) * p.hq * p.sq) + row) * p.d + col + e;
              *reinterpret_cast<float4*>(dst) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
              *reinterpret_cast<float4*>(dst + 4) = make_float4(o[e + 4], o[e + 5], o[e + 6], o[e + 7]);
            } else {
              const int64_t at = b * p.o.sb + head * p.o.sh + i * p.o.ss + col + e;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const T hi = from_f32<T>(o[e + k]);
                static_cast<T*>(p.o.ptr)[at + k] = hi;
                if (p.lo.ptr != nullptr) static_cast<T*>(p.lo.ptr)[at + k] = from_f32<T>(o[e + k] - to_f32<T>(hi));
              }
            }
          }
        }
      }
      if (staged) {
        fence_proxy_async_smem();
        __syncwarp();
        if (elect_one()) {
          for (int c = 0; c < D / 64; ++c) {
            tma_store_4d(&map_o, tile + c * 4096, c * 64, qt * kAttnTile + warp * 32, head, b);
            if (p.lo.ptr != nullptr) tma_store_4d(&map_lo, low + c * 4096, c * 64, qt * kAttnTile + warp * 32, head, b);
          }
          bulk_commit();
          bulk_wait_read();
        }
        __syncwarp();
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
  if (raised) {  // a wait ran out: no copy or MMA may be in flight when TMEM is freed and the block leaves
    if (warp == kCopier && elect_one()) {
      if (!S::kTmemQ && n > 0) Guard::drain(&bar.q_full, 0);
      for (int j = max(0, loads_k - kStages); j < loads_k; ++j) Guard::drain(&bar.k_full[j % kStages], (j / kStages) & 1);
      for (int j = max(0, loads_v - kStages); j < loads_v; ++j) Guard::drain(&bar.v_full[j % kStages], (j / kStages) & 1);
    }
    if (warp == kIssuer && elect_one()) {
      mma_commit(&bar.drain);
      Guard::drain(&bar.drain, 0);
    }
    __syncthreads();
  }
  if (warp == kIssuer) tmem_free(tmem, S::kTmem);
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

template <typename T, int D, Scores MODE>
cudaError_t run(const FwdParams& fp, cudaStream_t s) {
  const AttnParams& p = fp.a;
  CUtensorMap q{}, k, v, o{}, lo{};
  if (!Shape<D>::kTmemQ && !attn_map(&q, p.q, p, p.hq, p.sq, fp.packed ? p.sq : kAttnTile, fp.packed ? p.hq / p.hk : 1))
    return cudaErrorInvalidValue;
  if (!fp.packed && p.splits == 1 &&
      (!attn_map(&o, p.o, p, p.hq, p.sq, 32, 1) || (p.lo.ptr != nullptr && !attn_map(&lo, p.lo, p, p.hq, p.sq, 32, 1))))
    return cudaErrorInvalidValue;
  if (!attn_map(&k, p.k, p, p.hk, p.sk, Shape<D>::kKeys, 1) || !attn_map(&v, p.v, p, p.hk, p.sk, Shape<D>::kKeys, 1))
    return cudaErrorInvalidValue;
  const auto kernel = fwd_kernel<T, D, MODE>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
  if (e != cudaSuccess) return e;
  const int64_t blocks = static_cast<int64_t>(fp.tiles_q) * p.b * (fp.packed ? p.hk : p.hq) * p.splits;
  kernel<<<static_cast<unsigned>(blocks), Shape<D>::kThreads, Shape<D>::kSmem, s>>>(q, k, v, o, lo, fp);
  if (p.splits > 1) {
    const int64_t rows = static_cast<int64_t>(p.b) * p.hq * p.sq;
    join_kernel<T><<<static_cast<unsigned>((rows + 3) / 4), 128, 0, s>>>(fp);
  }
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t by_scores(const FwdParams& fp, cudaStream_t s) {
  switch (scores_of(fp.a)) {
    case kPlain: return run<T, D, kPlain>(fp, s);
    case kBiased: return run<T, D, kBiased>(fp, s);
    case kCapped: return run<T, D, kCapped>(fp, s);
  }
  return cudaErrorInvalidValue;
}

bool packs(const AttnParams& p) { return p.hq > p.hk && p.hq / p.hk * p.sq <= kAttnTile; }

}  // namespace

namespace {

// The driver's encoder, looked up at run time: the module has to load on machines without a driver.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static const EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found);
    return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(p) : nullptr;
  }();
  return f;
}

}  // namespace

bool attn_map(CUtensorMap* m, const AttnTensor& t, const AttnParams& p, int heads, int len, int box_rows, int box_heads) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.d), static_cast<cuuint64_t>(len), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(p.b)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(t.ss) * 2, static_cast<cuuint64_t>(t.sh) * 2,
                                 static_cast<cuuint64_t>(t.sb) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(box_heads), 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const EncodeTiled encode = encoder();
  if (encode == nullptr) return false;
  return encode(m, p.dt == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                                t.ptr, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t attn_wait_limit() { return wait_limit.load(); }

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

int64_t attention_wait_limit(int64_t clocks) { return wait_limit.exchange(clocks); }

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
  fp.sc = ScoreScale::of(p);
  fp.packed = packs(p);
  fp.tiles_q = fp.packed ? 1 : (p.sq + kAttnTile - 1) / kAttnTile;
  fp.status = attn_status_ptr();
  fp.a.wait_limit = attn_wait_limit();
  if (p.dt == kBF16) return p.d <= 64 ? by_scores<__nv_bfloat16, 64>(fp, s) : by_scores<__nv_bfloat16, 128>(fp, s);
  return p.d <= 64 ? by_scores<__half, 64>(fp, s) : by_scores<__half, 128>(fp, s);
}

}  // namespace launch
}  // namespace bitscom_b200
