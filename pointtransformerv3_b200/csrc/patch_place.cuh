// Where a pair of points looks into a head's table of biases, and where a block of keys leaves the table's gradient (patch_attn.cuh); plain
// C++, so that both can be checked on the host.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define PTV3_PLACE __host__ __device__ __forceinline__
#else
#define PTV3_PLACE static inline
#endif

namespace ptv3 {

// A coordinate within its sequence's box, [lowest, lowest + extent], counted from `lowest`.  Points outside the box, which are there where
// coordinates have changed since the plan's rows were made, count as on its border, so that no offset is larger than the extent,
// whatever is read.
PTV3_PLACE int pa_held(int coord, int lowest, int extent)
{
    const uint32_t v = (uint32_t)coord - (uint32_t)lowest;
    return (int)(v < (uint32_t)extent ? v : (uint32_t)extent);
}
// This point's share of an entry's address: subtracting `sign` times pa_other of the other point gives the address
PTV3_PLACE int pa_mine(int first, int reach, int held, int sign, int step) { return first + ((reach + sign * held) << step); }
PTV3_PLACE int pa_other(int held, int step) { return held << step; }

// Number of a block of `rows` keys, tile `tile` of a sequence that starts at row `start`: below n_pad / rows + n_seq, whatever the longest
// sequence is.  Sequences have a number to spare at most, behind their last tile: where pa_bin_end is above that tile's number and one.
PTV3_PLACE int64_t pa_bin_block(int start, int rows, int seq, int tile) { return (int64_t)(start / rows) + seq + tile; }
// first number of the next sequence
PTV3_PLACE int64_t pa_bin_end(int end, int rows, int seq) { return (int64_t)(end / rows) + seq + 1; }

}  // namespace ptv3
