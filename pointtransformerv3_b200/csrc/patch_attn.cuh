// Patch attention with a learned relative position bias, and differential patch attention, forward and backward
// (ptv3_patch_attention_fwd / _bwd): what their files share.
//
//   maps = 1:  A = P1            maps = 2:  A = P1 - lam[h] P2          O = A V
//   P_m = softmax_j(scale q_m k_m^T + bias),  q_m, k_m of W / maps values, v of W values per head
//   backward, G = dO V^T:  delta_m = sum_j P_m G,  dS_1 = P_1 (G - delta_1),  dS_2 = -lam P_2 (G - delta_2),
//   dV = A^T dO,  dQ_m = scale dS_m K_m,  dK_m = scale dS_m^T Q_m,  dlam = -sum_i delta_2,
//   dtable[a][b] = sum of dS_1 over the pairs whose offset along axis a falls into bucket b
//
// A backward pass is two kernels, one that walks keys for each block of queries (delta, dQ, dtable) and one that walks
// queries for each block of keys (dK, dV): both compute scores and probabilities again from the saved logarithm
// of the softmax's sum, nothing of size L x L is stored and no float is added atomically, so results do not
// depend on the order of anything.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace ptv3 {

constexpr float PA_LOG2E = 1.4426950408889634f, PA_LN2 = 0.6931471805599453f;
constexpr int PA_MAX_BOUND = 512;
constexpr int PA_MAX_COORD = 1 << 22;                 // coordinates of a bias lie within this of zero
constexpr int PA_TABLE_BYTES = 3 * 129 * 32 * 4;      // shared memory that copies of a head's table may take

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
    int copies_log2;            // the table in shared memory: that many copies, interleaved, one per lane or so
    const void* lam;            // H
    int lam_bf16;
    float* lse;                 // (H maps) x n_pad: log2 of the sum, or NULL
    const void* dout;
    void* dqkv;
    float* delta;               // (H maps) x n_pad
    float* shared;              // rows of (dK, dV), 2C
    float* bins;                // per block of queries: H x 3 (2 bnd + 1), or NULL
};

// rows [start, start + L) of a sequence; L = 0 for what ptv3_patch_rows reports
__device__ __forceinline__ int pa_sequence(const PatchArgs& a, int seq, int& start)
{
    start = a.cu[seq];
    const int end = a.cu[seq + 1];
    const bool ok = start >= 0 && end <= a.n_pad && end - start <= a.max_seqlen && end > start;
    return ok ? end - start : 0;
}

__device__ __forceinline__ float pa_param(const void* p, int i, int bf16)
{
    return bf16 ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : ((const float*)p)[i];
}

// This head's table in shared memory, in powers of two: entry e of axis a at ((a (2 bnd + 1) + e) << copies) + copy.
// A lane reads the copy of its number: with 32 copies look-ups of a warp never meet in a bank.
__device__ __forceinline__ void pa_load_table(const PatchArgs& a, int h, float* tab, int tid, int threads)
{
    const int ne = 2 * a.bnd + 1, copies = 1 << a.copies_log2;
    for (int i = tid; i < 3 * ne; i += threads) {
        const int axis = i / ne, e = i - axis * ne;
        int b = a.buckets ? a.buckets[e] : e;
        b = min(max(b, 0), a.num - 1);                     // (ptv3_patch_rows reports one out of range)
        const float v = pa_param(a.table, (axis * a.num + b) * a.H + h, a.table_bf16) * PA_LOG2E;
        for (int c = 0; c < copies; ++c) tab[(i << a.copies_log2) + ((c + tid) & (copies - 1))] = v;
    }
}

enum { PA_FWD = 0, PA_ROWS = 1, PA_COLS = 2 };
// fp32 (patch_attn_fma.cu) and bf16 (patch_attn_mma.cu); ..._rows: rows of a block, in which `tiles` counts
int launch_patch_fma(const PatchArgs& a, int width, int maps, int pass, cudaStream_t stream);
int launch_patch_mma(const PatchArgs& a, int width, int maps, int pass, cudaStream_t stream);
int patch_fma_rows(int width);
int patch_mma_rows();

}  // namespace ptv3
