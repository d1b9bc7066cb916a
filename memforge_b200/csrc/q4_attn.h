// The chunk kernel of attention over the 4-bit cache, as the dispatcher sees it.
#pragma once

#include "mf_attn.h"

namespace mf {

// Whether the tcgen05 kernel takes runs of this call (the rest stay with mma.sync).
bool q4_prefill_serves(const AttnParams& a, mf_dtype dtype);

// Serves every sequence with more than rows_cap rows per kv head.  a.kp: the pool, a.sb /
// a.sh its strides in bytes; width: entries of a block table's row; vec: q and out rows
// allow 16-byte accesses.
int launch_q4_prefill(const AttnParams& a, int width, int vec, int rows_cap, mf_dtype dtype,
                      cudaStream_t stream);

}  // namespace mf
