// Host build of the addresses of look-ups into a table of biases.
#include "../../pointtransformerv3_b200/csrc/patch_place.cuh"

using namespace ptv3;

// addresses of the entries of n pairs (mine[i], other[i]) of a sequence whose coordinates are in [lowest, lowest + extent]
extern "C" void host_places(const int32_t* mine, const int32_t* other, int64_t n, int lowest, int extent, int first, int reach,
                            int sign, int step, int32_t* out)
{
    for (int64_t i = 0; i < n; ++i)
        out[i] = pa_mine(first, reach, pa_held(mine[i], lowest, extent), sign, step) -
                 sign * pa_other(pa_held(other[i], lowest, extent), step);
}

// numbers that a sequence's tiles of `rows` keys write, in order, and zero: at most `most`, their count
extern "C" int host_bins(int start, int length, int rows, int seq, int64_t* out)
{
    int n = 0;
    const int tiles = (length + rows - 1) / rows;
    for (int t = 0; t < (tiles ? tiles : 1); ++t) out[n++] = pa_bin_block(start, rows, seq, t);
    if (tiles && pa_bin_end(start + length, rows, seq) > out[n - 1] + 1) {
        out[n] = out[n - 1] + 1;
        ++n;
    }
    return n;
}
