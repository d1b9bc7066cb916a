// The chunk kernel of attention over the 4-bit cache, as the dispatcher sees it.
#pragma once

#include "mf_attn.h"

namespace mf {

// Whether the tcgen05 kernel takes runs of this call (the rest stay with mma.sync).
bool q4_prefill_serves(const AttnParams& a, mf_dtype dtype);

// Whether the converting form may run in this build.
bool q4_converting_built();

// Serves every sequence with more than rows_cap rows per kv head.  a.kp: the pool, a.sb /
// a.sh its strides in bytes; width: entries of a block table's row; vec: q and out rows
// allow 16-byte accesses.
int launch_q4_prefill(const AttnParams& a, int width, int vec, int rows_cap,
                      cudaStream_t stream);

// The same over a copy of the cache that the call expands to fp16 in the workspace first:
// faster where many row tiles read a key, at 512 bytes per token and kv head.
struct Q4Scratch {
  size_t q, scale, k, v, bytes;  // offsets, and their total
};
// The expanded form's workspace, or false where it does not serve (rows that are not 16-byte
// aligned) or would exceed its limit.
bool q4_expand_plan(const AttnParams& a, int width, int vec, mf_dtype dtype, Q4Scratch& sc);
int launch_q4_expanded(const AttnParams& a, int width, int rows_cap, const Q4Scratch& sc,
                       uint8_t* ws, cudaStream_t stream);

}  // namespace mf
