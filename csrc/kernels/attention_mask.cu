// Mask plans of the attention kernels: from document ids and prefix lengths to
// the interval of keys that each row sees, and its bounds for tiles of rows.
//
// A document is a run of equal ids, so its interval is found by looking for
// the nearest change of id on either side.  One CTA takes one tile of 128 rows:
// changes inside the tile come from a scan in shared memory, a run that reaches
// over the tile's edge is followed outwards 512 ids at a time.  One launch,
// no order between CTAs, about 4 us for 8 rows of 1024 tokens (launch bound);
// a single document of 128K tokens costs each CTA at most 256 such steps.
#include <cuda_runtime.h>

#include "attention.h"

namespace bitscom_b200 {
namespace {

constexpr int kThreads = 512;

struct Ids {
  const void* p;
  int bytes;
  int64_t ss;
  __device__ int64_t at(int64_t j) const {
    return bytes == 8 ? static_cast<const long long*>(p)[j * ss] : static_cast<const int*>(p)[j * ss];
  }
};

__global__ void __launch_bounds__(kThreads) plan_kernel(const void* ids_base, int ids_bytes, int64_t ids_sb,
                                                        int64_t ids_ss, const void* prefix, int prefix_bytes,
                                                        int causal, int sq, int sk, int nq, int nk, PlanView plan) {
  const int t = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  __shared__ long long id[kAttnTile];
  __shared__ int start[kAttnTile], end[kAttnTile];
  __shared__ uint32_t begins[4];
  __shared__ int found;
  __shared__ int red[4][4];
  const bool docs = ids_base != nullptr;
  Ids ids{docs ? static_cast<const char*>(ids_base) + b * ids_sb * ids_bytes : nullptr, ids_bytes, ids_ss};

  if (t < nk && tid < kAttnTile) {  // padding among the keys of key tile t
    const int j = t * kAttnTile + tid;
    const bool dead = docs && j < sk && ids.at(j) < 0;
    const uint32_t m = __ballot_sync(0xffffffffu, dead);
    if ((tid & 31) == 0) reinterpret_cast<uint32_t*>(&plan.kdead[static_cast<int64_t>(b) * nk + t])[tid >> 5] = m;
  }
  if (t >= nq) return;

  const int off = sk - sq;
  const int first = t * kAttnTile + off;  // position of the tile's first row; negative when Sq > Sk
  const int rows = min(kAttnTile, sq - t * kAttnTile);
  long long p_len = 0;
  if (prefix != nullptr)
    p_len = prefix_bytes == 8 ? static_cast<const long long*>(prefix)[b] : static_cast<const int*>(prefix)[b];
  const int plen = static_cast<int>(p_len < 0 ? 0 : (p_len > sk ? sk : p_len));

  if (docs) {
    if (tid < kAttnTile) id[tid] = tid < rows && first + tid >= 0 ? ids.at(first + tid) : -1;
    __syncthreads();
    if (tid < kAttnTile) {  // bit r: row r begins a run (row 0 counts as one, and so do the rows past the end)
      const uint32_t m = __ballot_sync(0xffffffffu, tid == 0 || tid >= rows || id[tid] != id[tid - 1]);
      if ((tid & 31) == 0) begins[tid >> 5] = m;
    }
    __syncthreads();
    if (tid < rows) {
      int w = tid >> 5;
      uint32_t m = begins[w] & (0xffffffffu >> (31 - (tid & 31)));  // begins up to this row
      while (m == 0u) m = begins[--w];
      start[tid] = first + w * 32 + 31 - __clz(m);
      w = tid >> 5;
      m = (tid & 31) == 31 ? 0u : begins[w] & (0xffffffffu << ((tid & 31) + 1));  // begins behind it
      while (m == 0u && ++w < 4) m = begins[w];
      end[tid] = first + (m == 0u ? rows : min(rows, w * 32 + __ffs(m) - 1));
    }
    __syncthreads();
    // The first row's run to the left of the tile, and the last row's to the right.
    int left = max(first, 0), right = first + rows;
    if (first > 0 && id[0] >= 0) {
      const long long want = id[0];
      for (int hi = first; hi > 0; hi -= kThreads) {
        if (tid == 0) found = -1;
        __syncthreads();
        const int j = hi - 1 - tid;
        if (j >= 0 && ids.at(j) != want) atomicMax(&found, j);
        __syncthreads();
        const int f = found;
        __syncthreads();
        if (f >= 0) { left = f + 1; break; }
        left = max(0, hi - kThreads);
      }
    }
    if (right > 0 && right < sk && id[rows - 1] >= 0 && (!causal || prefix != nullptr)) {
      const long long want = id[rows - 1];
      for (int lo = right; lo < sk; lo += kThreads) {
        if (tid == 0) found = sk;
        __syncthreads();
        const int j = lo + tid;
        if (j < sk && ids.at(j) != want) atomicMin(&found, j);
        __syncthreads();
        const int f = found;
        __syncthreads();
        if (f < sk) { right = f; break; }
        right = min(sk, lo + kThreads);
      }
    }
    if (tid < rows) {
      if (start[tid] == first) start[tid] = left;
      if (end[tid] == first + rows) end[tid] = right;
    }
  }

  // The interval of each row, and its bounds over the tile (4 warps).
  if (tid < kAttnTile) {
    int lo = 0, hi = 0;
    if (tid < rows) {
      const int pos = first + tid;
      if (docs) {
        if (pos >= 0 && id[tid] >= 0) {
          lo = start[tid];
          hi = causal ? max(pos + 1, min(plen, end[tid])) : end[tid];
        }
      } else {
        hi = causal ? max(pos + 1, plen) : sk;
      }
      if (hi <= lo) lo = hi = 0;
    }
    plan.range[(static_cast<int64_t>(b) * nq + t) * kAttnTile + tid] = make_int2(lo, hi);
    const bool some = hi > lo;
    const uint32_t dead = __ballot_sync(0xffffffffu, tid < rows && !some);
    const int w = tid >> 5;
    if ((tid & 31) == 0) reinterpret_cast<uint32_t*>(&plan.qdead[static_cast<int64_t>(b) * nq + t])[w] = dead;
    const int big = 0x7fffffff;
    const int v0 = __reduce_min_sync(0xffffffffu, some ? lo : big);
    const int v1 = __reduce_max_sync(0xffffffffu, some ? hi : 0);
    // Rows past the end are no reason to look at a mask.
    const int v2 = __reduce_max_sync(0xffffffffu, tid < rows ? (some ? lo : big) : 0);
    const int v3 = __reduce_min_sync(0xffffffffu, tid < rows ? hi : big);
    if ((tid & 31) == 0) {
      red[w][0] = v0;
      red[w][1] = v1;
      red[w][2] = v2;
      red[w][3] = v3;
    }
  }
  __syncthreads();
  if (tid == 0) {
    int4 r = make_int4(red[0][0], red[0][1], red[0][2], red[0][3]);
    for (int w = 1; w < 4; ++w) {
      r.x = min(r.x, red[w][0]);
      r.y = max(r.y, red[w][1]);
      r.z = max(r.z, red[w][2]);
      r.w = min(r.w, red[w][3]);
    }
    if (r.y == 0) r.x = 0;
    plan.tile[static_cast<int64_t>(b) * nq + t] = r;
  }
}

}  // namespace

namespace launch {

void attention_plan(const void* ids, int ids_bytes, int64_t ids_sb, int64_t ids_ss, const void* prefix,
                    int prefix_bytes, int causal, int b, int sq, int sk, PlanView plan, cudaStream_t s) {
  const int nq = (sq + kAttnTile - 1) / kAttnTile, nk = (sk + kAttnTile - 1) / kAttnTile;
  if (b == 0 || (nq == 0 && nk == 0)) return;
  plan_kernel<<<dim3(nq > nk ? nq : nk, b), kThreads, 0, s>>>(ids, ids_bytes, ids_sb, ids_ss, prefix, prefix_bytes,
                                                              causal, sq, sk, nq, nk, plan);
}

}  // namespace launch
}  // namespace bitscom_b200
