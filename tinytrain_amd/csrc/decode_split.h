// How the decode kernels (fa_decode.hip, fa_decode_mx.hip) deal a unit, one (batch, KV head), to the
// workgroups of a split call.
#pragma once

#include <hip/hip_runtime.h>

namespace ttfa {

// Workgroups of a unit that have work: its nb blocks, 2^log2_min each at least (a power of two:
// a quotient would stand between the length's load and the first block's).
__device__ __forceinline__ int used_chunks(int nb, int n_chunks, int log2_min) {
  return max(min((nb + (1 << log2_min) - 1) >> log2_min, n_chunks), 1);
}

// Places by which chunk `chunk` turns its units (n_units >= 8).  Consecutive workgroups go to the
// XCDs in turn, and those of an XCD to its 32 CUs: 37 = 4 * 8 + 5 moves a unit's chunks to
// other XCDs and other CUs.  Fewer units have more chunks, whose own numbers do that.
__device__ __forceinline__ int chunk_turn(int chunk, int n_units) {
  int turn = chunk * (n_units >= 64 ? 37 : 5);
  if (n_units < 32) turn &= 7;
  while (turn >= n_units) turn -= n_units;  // at most five times
  return turn;
}

}  // namespace ttfa
