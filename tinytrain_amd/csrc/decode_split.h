// How the decode kernels (fa_decode.hip, fa_decode_mx.hip) deal a unit, one (batch, KV head), to the
// workgroups of a split call.  Each of them turns a unit's chunks over the XCDs by a rule of its own.
#pragma once

#include <hip/hip_runtime.h>

namespace ttfa {

// Workgroups of a unit that have work: its nb blocks, 2^log2_min each at least (a power of two:
// a quotient would stand between the length's load and the first block's).
__device__ __forceinline__ int used_chunks(int nb, int n_chunks, int log2_min) {
  return max(min((nb + (1 << log2_min) - 1) >> log2_min, n_chunks), 1);
}

}  // namespace ttfa
