// The 4-bit KV record, shared by the kernels that read or write it.
//
// Record of one (block of 16 tokens, kv head), 16 * D + 128 contiguous bytes:
//   [0, 8D)       K codes: token t's row at t * D/2, even dim in the low nibble
//   [8D, 16D)     V codes in the order the P V product's A operand wants them:
//                 [C][t >> 3][8 groups][(t >> 1) & 3][W words][t & 1][2 bytes],
//                 C = max(1, D / 128), W = min(4, D / 32); chunk c, group g, word w
//                 hold dims 128 c + 4W g + 4w .. + 3 (even dim in the low nibble)
//   [16D, +64)    K parameters: fp16 (scale, base) per token
//   [16D+64, +64) V parameters
// A value is code * scale + base.  In a V word the two 16-bit halves are tokens
// 2i and 2i + 1, so a mask leaves a pair of codes of neighbouring tokens, which is
// what one register of mma.sync's A fragment holds: no byte permutes.
#pragma once

#include "mf_internal.h"

namespace mf {
namespace q4 {

constexpr int BLOCK = 16;

__host__ __device__ constexpr int record_bytes(int d) { return 16 * d + 128; }
__host__ __device__ constexpr bool head_dim_ok(int d) { return d == 64 || d == 128 || d == 256; }

// Byte offset of the 16-bit piece that holds V dims 4j .. 4j+3 of token t.
template <int D>
MF_DEVINL int v_piece(int t, int j) {
  constexpr int W = D / 32 < 4 ? D / 32 : 4;
  constexpr int PC = D < 128 ? D / 4 : 32;  // pieces per chunk
  const int c = j / PC, jj = j % PC;
  const int g = jj / W, w = jj % W;
  return 8 * D + ((((c * 2 + (t >> 3)) * 8 + g) * 4 + ((t >> 1) & 3)) * W + w) * 4 + (t & 1) * 2;
}

}  // namespace q4

}  // namespace mf
