// Patch attention with a learned relative position bias, and differential patch attention, forward and backward
// (ptv3_patch_attention_fwd / _bwd): what their files share.
//
//   maps = 1:  A = P1            maps = 2:  A = P1 - lam[h] P2          O = A V
//   P_m = softmax_j(scale q_m k_m^T + bias),  q_m, k_m of W / maps values, v of W values per head
//   backward, G = dO V^T:  delta_m = sum_j P_m G,  dS_1 = P_1 (G - delta_1),  dS_2 = -lam P_2 (G - delta_2),
//   dV = A^T dO,  dQ_m = scale dS_m K_m,  dK_m = scale dS_m^T Q_m,  dlam = -sum_i delta_2,
//   dtable[a][b] = sum of dS_1 over the pairs whose offset along axis a falls into bucket b
//
// A backward pass is two kernels, one that walks keys for each block of queries (delta, dQ) and one that walks
// queries for each block of keys (dK, dV, dtable): both compute scores and probabilities again from the softmax's saved
// reference value and sum, nothing of size L x L is stored and no float is added atomically, so results do not
// depend on the order of anything.
//
// delta in one walk: the stored result gives an estimate, delta' = dO . O (dO . O2 for the second map, whose O2 the
// forward pass leaves too), which is off by the rounding of O alone.  With E = sum_j P (G - delta'),
// delta = delta' + E and dQ = sum_j P (G - delta') K - E sum_j P K, exact however far the values' mean is from zero and
// however peaked a row is.  (A walk of its own for delta: 632 us for the differential rows of 100 000 x 64 where one walk took 376.)
//
// dtable: a pair adds its dS to three bins, as integers in shared memory, since integer sums do not depend on the order
// of the additions.  Their unit follows from what the queries of a window can add at most, sum_j |dS_ij| <= sum_j P |G -
// delta'| + |E| (`reach`), so that no bin overflows; after a window the bins go into floats.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "patch_place.cuh"

namespace ptv3 {

constexpr float PA_LOG2E = 1.4426950408889634f, PA_LN2 = 0.6931471805599453f;
// Where a running maximum starts: no finite score is lower, and what it leaves of a sum (2^(start - score)) is 0 or, at that score, 1.
constexpr float PA_LOWEST = -3.402823466e38f;
// Finite entries of a table are held within this, in powers of two, so that three of them and a product are finite: a row whose
// every key is masked by the lowest value of a type is softmax's row of its least masked keys, as it is in 64 bits.
constexpr float PA_FAR = 4.2535296e37f;               // 2^125
constexpr int PA_MAX_BOUND = 512;
constexpr int PA_MAX_COORD = 1 << 22;                 // coordinates of a bias lie within this of zero
constexpr int PA_TABLE_BYTES = 80 * 1024;             // shared memory for a head's table, so that two CTAs fit an SM;
constexpr int PA_BINS_BYTES = 2 * 352 * 32 * 4;       // for a table and its bins beside it

// What the kernels get: ptv3_patch_attention_args with the workspace carved up.
struct PatchArgs {
    const void* qkv;
    void* out;
    const int32_t* rows;        // point of every padded row; -1 - point where the row does not answer for it
    const int32_t* slot;        // of every padded row: < 0, or its row of `shared` (a point with a borrowed copy)
    const int32_t* cu;
    int n_pad, n_seq, max_seqlen, tiles, C, H;
    float scale;
    const int32_t* grid;        // n x 3, or NULL without a bias
    const void* table;          // (3 num) x H
    const int32_t* buckets;     // 2 bnd + 1, or NULL: every offset its own
    int num, bnd, table_bf16;
    const int32_t* extent;      // n_seq x 6: largest offset within a sequence along each axis, and its lowest coordinates
    const int32_t* owner;       // of every point: a row that answers for it (one of them, where an order holds it twice)
    uint32_t* status;           // or NULL
    const void* lam;            // H
    int lam_bf16;
    float* lse;                 // twice (H maps) x n_pad: the softmax's reference value in log2, then one over its sum (not the
                                // logarithm of the sum, in which a reference far from zero leaves no bits for the sum); or NULL
    const void* dout;
    void* dqkv;
    void* second;               // n x C: O2, with two maps
    float* delta;               // (H maps) x n_pad
    float* reach;               // H x n_pad: no row's sum of |dS| is larger; or NULL
    float* shared;              // rows of (dK, dV), 2C
    float* bins;                // per block of keys: H x 3 (2 bnd + 1), or NULL
    int bin_rows;               // rows of such a block, where blocks are numbered by rows (pa_bin_block); 0: by sequence and tile
};

// rows [start, start + L) of a sequence; L = 0 for what patch_rows_kernel reports
__device__ __forceinline__ int pa_sequence(const PatchArgs& a, int seq, int& start)
{
    start = a.cu[seq];
    const int end = a.cu[seq + 1];
    const bool ok = start >= 0 && end <= a.n_pad && end - start <= a.max_seqlen && end > start;
    return ok ? end - start : 0;
}

// Reports a point that more than one of the rows [first, end) answers for, and another therefore none: all but one of its rows find that
// out.  (A call, so that the kernels' registers stay as they are.)
static __device__ __noinline__ void pa_check_owners(const int32_t* rows, const int32_t* owner, uint32_t* status, int first, int end)
{
    for (int i = first + threadIdx.x; i < end; i += blockDim.x) {
        const int e = rows[i];
        if (e >= 0 && owner[e] != i) atomicOr(status, PTV3_STATUS_BAD_INDEX);
    }
}

// a coordinate of a bias (patch_rows_kernel reports one out of range; places in the table stay within it all the same)
__device__ __forceinline__ int pa_coord(const PatchArgs& a, int64_t p, int c)
{
    return min(max(a.grid[3 * p + c], -PA_MAX_COORD), PA_MAX_COORD);
}

__device__ __forceinline__ float pa_param(const void* p, int i, int bf16)
{
    return bf16 ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : ((const float*)p)[i];
}

// This head's table in shared memory, in powers of two, of the offsets that occur in a sequence: axis a holds offsets
// -reach[a] .. reach[a], entry e of it at (first[a] + e) copies + copy.  A lane reads the copy of its number: with 32
// copies, which most patches leave room for, look-ups of a warp never meet in a bank.  Offsets beyond the bound repeat its
// outermost entries (`far`), as long as that leaves room for eight copies: no look-up then has to be clamped.  With `bins`, there
// are as many copies of the bins, or half.
struct PatchTable {
    int reach[3], first[3], entries, copies_log2, bins_log2;
    bool clamps;
};
__device__ __forceinline__ PatchTable pa_table(const PatchArgs& a, int seq, int bytes, bool bins, bool far = true, int bins_most = 5)
{
    PatchTable t;
    t.clamps = false;
    for (int k = far ? 0 : 1; k < 2; ++k) {
        t.entries = 0;
#pragma unroll
        for (int c = 0; c < 3; ++c) {
            t.reach[c] = a.extent[6 * seq + c];
            if (k) t.reach[c] = min(a.bnd, t.reach[c]);
            t.first[c] = t.entries;
            t.entries += 2 * t.reach[c] + 1;
        }
        if (t.entries <= bytes >> (bins ? 6 : 5)) break;
        t.clamps = true;
    }
    t.copies_log2 = 5;
    t.bins_log2 = bins ? bins_most : 5;
    while (t.copies_log2 > 0 && 4 * ((t.entries << t.copies_log2) + (bins ? t.entries << t.bins_log2 : 0)) > bytes) {
        if (bins && t.bins_log2 == t.copies_log2) --t.bins_log2;
        else t.copies_log2 = t.bins_log2 = bins ? t.bins_log2 : t.bins_log2 - 1;
    }
    return t;
}
// axis and offset of an entry
__device__ __forceinline__ void pa_entry(const PatchTable& t, int i, int& axis, int& d)
{
    axis = i >= t.first[2] ? 2 : i >= t.first[1] ? 1 : 0;
    d = i - (axis == 2 ? t.first[2] + t.reach[2] : axis == 1 ? t.first[1] + t.reach[1] : t.reach[0]);
}
__device__ __forceinline__ void pa_load_table(const PatchArgs& a, const PatchTable& t, int h, float* tab, int tid,
                                              int threads)
{
    const int copies = 1 << t.copies_log2;
    for (int i = tid; i < t.entries; i += threads) {
        int axis, d;
        pa_entry(t, i, axis, d);
        const int e = min(max(d, -a.bnd), a.bnd) + a.bnd;
        int b = a.buckets ? a.buckets[e] : e;
        b = min(max(b, 0), a.num - 1);                     // (patch_rows_kernel reports one out of range)
        const float entry = pa_param(a.table, (axis * a.num + b) * a.H + h, a.table_bf16);
        const float v = fabsf(entry) < INFINITY ? fminf(fmaxf(entry * PA_LOG2E, -PA_FAR), PA_FAR) : entry;
        for (int c = 0; c < copies; ++c) tab[(i << t.copies_log2) + ((c + tid) & (copies - 1))] = v;
    }
}
// What the queries [q0, q0 + WINDOW) of a sequence can add to a bin at most, as a unit in which 2^30 of it are that.
// Lane t of four adds queries 2 t and 2 t + 1 of every eight, to copies of its own where there are four and
// more: the largest of four sums.  All threads of a block of 32 `WARPS`; `part`: WARPS x 4 floats
template <int WARPS, int WINDOW>
__device__ __forceinline__ float pa_unit(const PatchArgs& a, const PatchTable& table, int h, int start, int L, int q0,
                                         float* part)
{
    float v = 0.f;
    for (int j = threadIdx.x; j < WINDOW; j += 32 * WARPS)
        if (q0 + j < L) v += a.reach[(int64_t)h * a.n_pad + start + q0 + j];
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    v += __shfl_xor_sync(0xffffffffu, v, 16);
    __syncthreads();
    if ((threadIdx.x & 31) < 8 && (threadIdx.x & 1) == 0) part[(threadIdx.x / 32) * 4 + (threadIdx.x & 31) / 2] = v;
    __syncthreads();
    float top = 0.f, all = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        float sum = 0.f;
        for (int w = 0; w < WARPS; ++w) sum += part[4 * w + t];
        top = fmaxf(top, sum);
        all += sum;                        // (a NaN among them is kept by this one)
    }
    return (table.bins_log2 >= 2 && all == all ? top : all) * (1.f / 1073741824.f);
}
__device__ __forceinline__ float pa_per_unit(float unit)
{
    const float v = unit > 0.f ? 1.f / unit : 0.f;
    return v < INFINITY ? v : 0.f;
}
// bins into floats, bins cleared
__device__ __forceinline__ void pa_flush(const PatchTable& t, int* hist, float* sums, float unit, int threads)
{
    const int copies = 1 << t.bins_log2;
    for (int i = threadIdx.x; i < t.entries; i += threads) {
        float v = 0.f;
        for (int c = 0; c < copies; ++c) {
            int* at = hist + (i << t.bins_log2) + ((c + i) & (copies - 1));
            v += (float)*at;
            *at = 0;
        }
        sums[i] = fmaf(v, unit, sums[i]);
    }
}
// The bins of a block of keys and head; of a tile without keys, zeros are left there where nobody else does, and NULL is returned
template <int ROWS>
__device__ __forceinline__ float* pa_bins(const PatchArgs& a, int seq, int tile, int h, int start, int L, int threads)
{
    const int64_t size = 3 * (2 * a.bnd + 1);
    auto at = [&](int64_t block) { return a.bins + (block * a.H + h) * size; };
    auto clear = [&](int64_t block) {
        for (int i = threadIdx.x; i < size; i += threads) at(block)[i] = 0.f;
    };
    const bool empty = tile * ROWS >= L;
    if (!a.bin_rows) {
        const int64_t block = (int64_t)seq * a.tiles + tile;
        if (empty) clear(block);
        return empty ? nullptr : at(block);
    }
    const int first = min(max(start, 0), a.n_pad);          // (of a sequence that does not hold)
    const int64_t block = pa_bin_block(first, ROWS, seq, tile);
    if (empty) {
        if (tile == 0) clear(block);
        return nullptr;
    }
    if ((tile + 1) * ROWS >= L && pa_bin_end(first + L, ROWS, seq) > block + 1) clear(block + 1);
    return at(block);
}
// a block's sums of all offsets within the bound, those beyond with the outermost
__device__ __forceinline__ void pa_store_bins(const PatchArgs& a, const PatchTable& t, const float* sums, float* bins, int threads)
{
    const int ne = 2 * a.bnd + 1;
    for (int i = threadIdx.x; i < 3 * ne; i += threads) {
        const int axis = i / ne, d = i - axis * ne - a.bnd, r = axis == 0 ? t.reach[0] : axis == 1 ? t.reach[1] : t.reach[2];
        const float* at = sums + (axis == 0 ? 0 : axis == 1 ? t.first[1] : t.first[2]) + r;
        const int lo = d == -a.bnd ? -r : max(d, -r), hi = d == a.bnd ? r : min(d, r);
        float v = 0.f;
        for (int k = lo; k <= hi; ++k) v += at[k];
        bins[i] = v;
    }
}

enum { PA_FWD = 0, PA_ROWS = 1, PA_COLS = 2 };
// fp32 (patch_attn_fma.cu) and bf16 (patch_attn_mma.cu): a pass queued, `tiles` set by the rows that its blocks have
int launch_patch_fma(const PatchArgs& a, int width, int maps, int pass, cudaStream_t stream);
int launch_patch_mma(const PatchArgs& a, int width, int maps, int pass, cudaStream_t stream);
// rows of a block of the pass over columns with a bias, whose blocks leave bins (PatchArgs::bin_rows)
int patch_fma_cols_rows(int64_t longest, int width);
int patch_mma_cols_rows(int64_t n_seq, int64_t longest, int heads, int width);

}  // namespace ptv3
