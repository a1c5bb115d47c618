// Host side shared by the tensor-core attention kernels.
#pragma once

#include <cuda.h>

#include "attention.h"

namespace bitscom_b200 {

// Tensor map of a [B, H, S, D] tensor with a box of 64 x box_rows x box_heads.  The
// strides of dimensions longer than one are multiples of 16 bytes (the caller's check).
bool attn_map(CUtensorMap* m, const AttnTensor& t, const AttnParams& p, int heads, int len, int box_rows, int box_heads);

// The status word of the current device (see attention_status).
int* attn_status_ptr();

// Clocks that a wait of the next launch may last.
int64_t attn_wait_limit();

}  // namespace bitscom_b200
