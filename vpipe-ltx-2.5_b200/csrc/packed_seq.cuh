// packed_seq.cuh -- finding a work slot's sequence on the device.
#pragma once

#include "packed_index.h"
#include "ptx.cuh"

namespace ltx {

// The sequence that owns work slot `slot`: the last s with slot_base <= slot.
// The whole warp searches, 32 ways at a time.
__device__ __forceinline__ int find_seq(const int* cu, int seqs, int rows, int tile, int extra,
                                        int slot)
{
  int lo = 0, hi = seqs;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + (int)lane_id() * step;
    const bool below = lane_id() == 0 ||
        (at < hi && slot_base(clamp_int(cu[at], 0, rows), at, tile, extra) <= slot);
    const int last = 31 - __clz((int)__ballot_sync(0xffffffffu, below));
    lo += last * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

}  // namespace ltx
