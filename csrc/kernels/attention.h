// Masked attention: parameters shared by the kernels, their launchers and the
// argument checks (csrc/ops/attention_ops.cpp).
//
//   s_ij = scale * q_i.k_j;  s = cap * tanh(s / cap) when cap > 0
//   s   -= slope_h * |pos_i - j|           pos_i = i + Sk - Sq
//   o_i  = sum_j softmax_j(s_ij) v_j       over the keys lo_i <= j < hi_i
//
// Every mask offered (causal, documents, prefix) leaves each row one interval
// of keys, so a mask is two integers a row.  Without documents and prefixes
// the interval is computed in the kernel; otherwise `plan` holds it (laid out
// by PlanView, written by attention_plan()).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "launchers.h"

namespace bitscom_b200 {

// Rows and keys are cut into tiles of 128 everywhere a plan is read.
constexpr int kAttnTile = 128;

// The parts of a mask plan inside one int32 buffer (every part 16-byte aligned).
struct PlanView {
  int2* range;   // [B][nq * 128] visible keys [lo, hi) of each row; (0, 0) sees none, like the rows past the end
  int4* tile;    // [B][nq]   of a tile's rows: min lo, max hi of those that see a key; max lo, min hi of all
  uint4* qdead;  // [B][nq]   bit r: row r of the tile sees no key
  uint4* kdead;  // [B][nk]   bit r: key r of the tile is padding (seen by no row)
  __host__ __device__ static int64_t words(int64_t b, int64_t sq, int64_t sk) {
    const int64_t nq = (sq + kAttnTile - 1) / kAttnTile, nk = (sk + kAttnTile - 1) / kAttnTile;
    return b * nq * kAttnTile * 2 + b * nq * 8 + b * nk * 4;
  }
  __host__ __device__ static PlanView of(int* base, int64_t b, int64_t sq, int64_t sk) {
    PlanView v{nullptr, nullptr, nullptr, nullptr};
    if (base == nullptr) return v;
    const int64_t nq = (sq + kAttnTile - 1) / kAttnTile;
    v.range = reinterpret_cast<int2*>(base);
    int* p = base + b * nq * kAttnTile * 2;
    v.tile = reinterpret_cast<int4*>(p);
    v.qdead = reinterpret_cast<uint4*>(p + b * nq * 4);
    v.kdead = reinterpret_cast<uint4*>(p + b * nq * 8);
    return v;
  }
};

struct AttnTensor {  // [B, H, S, D] with D contiguous; strides in elements
  void* ptr;
  int64_t sb, sh, ss;
};

struct AttnParams {
  AttnTensor q, k, v, o, dout, dq, dk, dv;
  AttnTensor lo;  // o minus its rounding to the tensors' type, laid out like o (null: not kept)
  float* lse;    // [B][Hq][Sq] log2 of the softmax denominator, +inf for a row without keys
  float* delta;  // [B][Hq][Sq] sum_d dout * o (backward, elementary form)
  float* stats;  // [B][Hq][nq][2][128] minus log2 of the denominator (-inf without keys, and past the end), delta
  const float* slopes;  // [Hq] or null
  PlanView plan;        // null pointers: causal or full from the lengths alone
  int b, hq, hk, sq, sk, d;
  int causal;
  float scale, cap;
  // Few rows over many keys: the keys are cut into `splits` ranges of
  // split_tiles tiles; each writes its own partial result, joined afterwards.
  int splits, split_tiles;
  float* part_o;    // [splits][B][Hq][Sq][D]
  float* part_lse;  // [splits][B][Hq][Sq]
  int64_t wait_limit;  // clocks that a wait of a tensor-core kernel may last; 0: the wait for scores runs out
  DType dt;
};

namespace launch {

// Builds a mask plan from document ids [B, Sk] (any integer width; id < 0 is
// padding; null: one document) and prefix lengths [B] (null: none).
void attention_plan(const void* ids, int ids_bytes, int64_t ids_sb, int64_t ids_ss, const void* prefix,
                    int prefix_bytes, int causal, int b, int sq, int sk, PlanView plan, cudaStream_t s);

// Elementary form in fp32 arithmetic for every type and head size up to 256.
void attention_simt_forward(const AttnParams& p, cudaStream_t s);
void attention_simt_backward(const AttnParams& p, cudaStream_t s);

// Tensor-core form: fp16 and bf16, head sizes up to 128 that are multiples of 8,
// rows on 16-byte boundaries.  The caller sets p.splits / split_tiles from attention_tc_splits and
// allocates part_o / part_lse when there are several.
void attention_tc_splits(const AttnParams& p, int sms, int* splits, int* split_tiles);
cudaError_t attention_tc_forward(const AttnParams& p, cudaStream_t s);

cudaError_t attention_tc_backward(const AttnParams& p, cudaStream_t s);

// 0, or 1 once a wait of a tensor-core kernel on the current device ran out (its
// outputs are NaN then); `reset` clears it.  Waits for the device.
int attention_status(bool reset);

// Limit of later launches' waits, of every device; returns the one before (at first about 4 s).  With 0 the
// barriers of the scores expect an arrival that never comes, so that their waits run out in every block.
int64_t attention_wait_limit(int64_t clocks);

}  // namespace launch
}  // namespace bitscom_b200
