// Patch attention with a learned relative position bias, and differential patch attention: entry points, the map from padded rows
// to points, and the sums behind the backward pass (patch_attn.cuh has the mathematics).
#include "patch_attn.cuh"
#include "../../include/ptv3_b200.h"

namespace ptv3 {

// ---- rows of a plan ---------------------------------------------------------------------------------------
// Points are looked up once (rows[P] = order[pad[P]], or -1 - that where unpad[pad[P]] != P: the row was borrowed by
// another patch and answers for nothing), so that the attention kernels load one word per row and not three in a chain.
// Keys and values of a borrowed row have a gradient all the same, and a point has at most one such row beside its
// own: for a backward pass both get a row of its side buffer (slots 2 i and 2 i + 1; `slot` comes in filled with -1, and so
// does the counter behind it).  With a bias the first blocks take a sequence each, and find the largest offset of two of its
// points along each axis.
// (Neither this kernel nor the attention kernels let the one behind them start early: blocks that come while others run are placed
// where there is room at that time, not evenly.  12 000 x 32 in fp32, forward and backward: 167 us, 191 if this one did.)
struct PatchPlan {
    const int64_t *order, *pad, *unpad;
    const int32_t *cu, *grid, *buckets;
    int n, n_pad, n_seq, max_seqlen, n_entries, num, n_extents;
    int32_t *rows, *slot, *extent, *owner;      // slot: n_pad, then a point for each of n_pad - n, then the counter; or NULL
    uint32_t* status;
};

__device__ __forceinline__ void patch_extent(const PatchPlan& p, int seq)
{
    __shared__ int lo_s[8][3], hi_s[8][3];
    int lo[3], hi[3];
    PatchArgs a = {};
    a.cu = p.cu;
    a.grid = p.grid;
    a.n_pad = p.n_pad;
    a.max_seqlen = p.max_seqlen;
    int start;
    const int L = pa_sequence(a, seq, start);
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        lo[c] = PA_MAX_COORD;
        hi[c] = -PA_MAX_COORD;
    }
#pragma unroll 4
    for (int i = threadIdx.x; i < L; i += 256) {
        const int64_t pd = p.pad[start + i];
        int64_t e = pd >= 0 && pd < p.n ? p.order[pd] : 0;
        if (e < 0 || e >= p.n || p.unpad[pd >= 0 && pd < p.n ? pd : 0] < 0 ||
            p.unpad[pd >= 0 && pd < p.n ? pd : 0] >= p.n_pad)
            e = 0;                               // (what such a row is taken as: point 0)
#pragma unroll
        for (int c = 0; c < 3; ++c) {
            const int v = pa_coord(a, e, c);
            lo[c] = min(lo[c], v);
            hi[c] = max(hi[c], v);
        }
    }
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        lo[c] = __reduce_min_sync(0xffffffffu, lo[c]);
        hi[c] = __reduce_max_sync(0xffffffffu, hi[c]);
        if ((threadIdx.x & 31) == 0) {
            lo_s[threadIdx.x / 32][c] = lo[c];
            hi_s[threadIdx.x / 32][c] = hi[c];
        }
    }
    __syncthreads();
    if (threadIdx.x < 3) {
        int l = lo_s[0][threadIdx.x], h = hi_s[0][threadIdx.x];
        for (int w = 1; w < 8; ++w) {
            l = min(l, lo_s[w][threadIdx.x]);
            h = max(h, hi_s[w][threadIdx.x]);
        }
        p.extent[6 * seq + threadIdx.x] = max(h - l, 0);
        p.extent[6 * seq + 3 + threadIdx.x] = l;
    }
}

__global__ void __launch_bounds__(256) patch_rows_kernel(const PatchPlan p)
{
    pdl_wait();
    if ((int)blockIdx.x < p.n_extents) {
        patch_extent(p, blockIdx.x);
        return;
    }
    bool bad = false;
    const int n_slots = p.n_pad - p.n;
    int32_t *slot_point = p.slot + p.n_pad, *taken = slot_point + n_slots;
    const int most = max(max(p.n_pad, p.n_seq + 1), p.n_entries);
    for (int i = ((int)blockIdx.x - p.n_extents) * 256 + (int)threadIdx.x; i < most;
         i += ((int)gridDim.x - p.n_extents) * 256) {
        if (i < p.n_pad) {
            const int64_t pd = p.pad[i];
            const bool in = pd >= 0 && pd < p.n;
            const int64_t e = in ? p.order[pd] : -1, own = in ? p.unpad[pd] : -1;
            const bool good = e >= 0 && e < p.n && own >= 0 && own < p.n_pad;
            bad |= !good;
            if (good && own != i) {
                const bool right = n_slots > 0 && p.pad[own] == pd;
                bad |= !right;
                if (right && p.slot) {
                    const int s = atomicAdd(taken, 1) + 1;
                    bad |= s >= n_slots;
                    if (s < n_slots) {
                        p.slot[i] = 2 * s + 1;
                        // (a point with two borrowed rows has no place for the second)
                        bad |= atomicCAS(p.slot + own, -1, 2 * s) != -1;
                        slot_point[s] = (int32_t)e;
                    }
                }
            }
            p.rows[i] = !good ? -1 : own == i ? (int32_t)e : -1 - (int32_t)e;
            if (good && own == i) p.owner[e] = i;
        }
        if (i < p.n) {
            // every point has one row that answers for it
            bad |= p.unpad[i] < 0 || p.unpad[i] >= p.n_pad || p.pad[p.unpad[i]] != i;
            if (p.grid)
                for (int c = 0; c < 3; ++c)
                    bad |= p.grid[3 * (int64_t)i + c] < -PA_MAX_COORD || p.grid[3 * (int64_t)i + c] > PA_MAX_COORD;
        }
        if (i < p.n_seq)
            bad |= p.cu[i] < 0 || p.cu[i + 1] < p.cu[i] || p.cu[i + 1] - p.cu[i] > p.max_seqlen || (i == 0 && p.cu[0] != 0);
        if (i == p.n_seq) bad |= p.cu[p.n_seq] != p.n_pad;
        if (i < p.n_entries) bad |= p.buckets[i] < 0 || p.buckets[i] >= p.num;
    }
    if (bad && p.status) atomicOr(p.status, PTV3_STATUS_BAD_INDEX);
}

// ---- gradients of keys and values with a borrowed copy ------------------------------------------------------
template <typename T>
__device__ __forceinline__ void pa_store(T* p, float v);
template <> __device__ __forceinline__ void pa_store<float>(float* p, float v) { *p = v; }
template <> __device__ __forceinline__ void pa_store<__nv_bfloat16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T>
__global__ void __launch_bounds__(256) patch_shared_kernel(const float* shared, const int32_t* slot_point, int n_slots, int C,
                                                           T* dqkv)
{
    pdl_wait();
    const int64_t total = (int64_t)n_slots * 2 * C;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t s = i / (2 * C), c = i % (2 * C);
        const int p = slot_point[s];
        if (p >= 0) pa_store(dqkv + (int64_t)p * 3 * C + C + c, shared[4 * C * s + c] + shared[4 * C * s + 2 * C + c]);
    }
}

// ---- sums over blocks, in a fixed order ------------------------------------------------------------------------
constexpr int PA_FOLD = 64;      // rows added by a block of the first step

// out[block][i] = sum of PA_FOLD rows of in
__global__ void __launch_bounds__(256) patch_fold_kernel(const float* in, int64_t rows, int width, float* out)
{
    pdl_wait();
    const int64_t first = (int64_t)blockIdx.x * PA_FOLD;
    const int count = (int)min((int64_t)PA_FOLD, rows - first);
    const int i = blockIdx.y * 256 + threadIdx.x;
    if (i >= width) return;
    float v = 0.f;
#pragma unroll 8
    for (int r = 0; r < count; ++r) v += in[(first + r) * width + i];
    out[(int64_t)blockIdx.x * width + i] = v;
}

// One axis and head: sums of all rows by offset, then by bucket.
__global__ void __launch_bounds__(256) patch_table_kernel(const float* in, int64_t rows, int H, int bnd, int num,
                                                          const int32_t* buckets, void* dtable, int bf16)
{
    pdl_wait();
    __shared__ float sum[2 * PA_MAX_BOUND + 1];
    __shared__ int bucket[2 * PA_MAX_BOUND + 1];
    const int axis = blockIdx.x, h = blockIdx.y, ne = 2 * bnd + 1;
    const int64_t width = (int64_t)H * 3 * ne;
    for (int e = threadIdx.x; e < ne; e += 256) {
        float v = 0.f;
#pragma unroll 4
        for (int64_t r = 0; r < rows; ++r) v += in[r * width + (h * 3 + axis) * ne + e];
        sum[e] = v;
        bucket[e] = buckets ? min(max(buckets[e], 0), num - 1) : e;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < num; b += 256) {
        float v = 0.f;
        for (int e = 0; e < ne; ++e)
            if (bucket[e] == b) v += sum[e];
        const int at = (axis * num + b) * H + h;
        if (bf16) pa_store((__nv_bfloat16*)dtable + at, v);
        else pa_store((float*)dtable + at, v);
    }
}

// -sum of delta_2 over all rows, a head per block row: `parts` blocks leave partial sums, a block of a second launch
// adds them (the result in place of them); with one part that one launch does it all
__global__ void __launch_bounds__(256) patch_lam_kernel(const float* delta, int n_pad, int parts, float* partial, void* dlam,
                                                        int bf16)
{
    pdl_wait();
    __shared__ float warp_sum[8];
    const int h = blockIdx.y;
    float v = 0.f;
    if (dlam && parts > 1) {
        for (int i = threadIdx.x; i < parts; i += 256) v += partial[h * parts + i];
    } else {
        const float* row = delta + (int64_t)(2 * h + 1) * n_pad;
#pragma unroll 4
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n_pad; i += (int64_t)parts * 256) v -= row[i];
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x / 32] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        v = 0.f;
        for (int w = 0; w < 8; ++w) v += warp_sum[w];
        if (!dlam) partial[h * parts + blockIdx.x] = v;
        else if (bf16) pa_store((__nv_bfloat16*)dlam + h, v);
        else pa_store((float*)dlam + h, v);
    }
}

// (a caller's patch size may be more than there is)
static int longest(const ptv3_patch_attention_args* p)
{
    return (int)(p->max_seqlen < p->n_pad ? p->max_seqlen : p->n_pad);
}
// rows of a block that leaves bins
static int bin_rows(const ptv3_patch_attention_args* p)
{
    const int width = p->channels / p->heads;
    return p->dtype == PTV3_DTYPE_BF16 ? patch_mma_cols_rows(p->n_seq, longest(p), p->heads, width)
                                       : patch_fma_cols_rows(longest(p), width);
}
// Such blocks, heads apart: a tile's of every sequence, or as many as there are rows for (20 000 scenes of 20 points beside a patch of 1 024:
// 23 000 instead of 160 000).
static int64_t bin_blocks(const ptv3_patch_attention_args* p, bool& by_rows)
{
    const int rows = bin_rows(p);
    const int64_t tiles = (int64_t)p->n_seq * ceil_div(longest(p), rows), numbers = p->n_pad / rows + p->n_seq;
    by_rows = numbers < tiles;
    return by_rows ? numbers : tiles;
}

static int launch_patch(const ptv3_patch_attention_args* p, const PatchArgs& a, int pass, cudaStream_t stream)
{
    const int width = p->channels / p->heads;
    return p->dtype == PTV3_DTYPE_BF16 ? launch_patch_mma(a, width, p->maps, pass, stream)
                                       : launch_patch_fma(a, width, p->maps, pass, stream);
}

struct PatchWorkspace {
    float *delta, *reach, *shared, *bins, *folded, *partial;
    size_t bytes;
    int64_t blocks;      // that leave bins, heads apart
    bool by_rows;        // how they are numbered
    int parts;
};

static PatchWorkspace carve(const ptv3_patch_attention_args* p)
{
    Carver c(p->workspace);
    PatchWorkspace w = {};
    w.blocks = bin_blocks(p, w.by_rows);
    w.parts = p->n_pad > 16384 ? ceil_div(p->n_pad, 4096) : 1;
    w.delta = c.take<float>((size_t)p->heads * p->maps * p->n_pad);
    w.shared = c.take<float>((size_t)(p->n_pad - p->n) * 4 * p->channels);
    if (p->dtable) {
        w.reach = c.take<float>((size_t)p->heads * p->n_pad);
        const size_t width = (size_t)p->heads * 3 * (2 * p->pos_bnd + 1);
        w.bins = c.take<float>((size_t)w.blocks * width);
        w.folded = c.take<float>(w.blocks > PA_FOLD ? (size_t)ceil_div(w.blocks, PA_FOLD) * width : 0);
    }
    if (p->dlam) w.partial = c.take<float>((size_t)p->heads * w.parts);
    w.bytes = c.off;
    return w;
}

static int check_sizes(const ptv3_patch_attention_args* p, const char* what)
{
    PTV3_REQUIRE(p != nullptr, PTV3_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
    PTV3_REQUIRE(p->n >= 0 && p->n_pad >= p->n && p->n_pad <= 2 * p->n && p->n_seq >= (p->n > 0) && p->max_seqlen >= 1 && p->channels >= 1 && p->heads >= 1 &&
                     p->channels % p->heads == 0 && (p->maps == 1 || p->maps == 2),
                 PTV3_ERR_INVALID_ARGUMENT, "%s: bad sizes", what);
    const int width = p->channels / p->heads;
    PTV3_REQUIRE(width == 16 || width == 32 || width == 64, PTV3_ERR_UNSUPPORTED,
                 "%s: heads of %d values (supported: 16, 32, 64)", what, width);
    PTV3_REQUIRE(p->scale != 0.f && p->scale - p->scale == 0.f, PTV3_ERR_INVALID_ARGUMENT, "%s: scale %g", what, p->scale);
    PTV3_REQUIRE(p->dtype == PTV3_DTYPE_F32 || p->dtype == PTV3_DTYPE_BF16, PTV3_ERR_UNSUPPORTED, "%s: dtype %d", what,
                 p->dtype);
    // half of each: a point has at most two rows, and their slots are numbered in 32 bits too
    PTV3_REQUIRE(p->n_pad < (1ll << 30) && p->n_seq < (1 << 30), PTV3_ERR_UNSUPPORTED, "%s: more than 2^30 rows", what);
    if (p->maps == 2) {
        PTV3_REQUIRE(!p->grid_coord && !p->table, PTV3_ERR_UNSUPPORTED, "%s: no bias with two maps", what);
        PTV3_REQUIRE(p->lam_dtype == PTV3_DTYPE_F32 || p->lam_dtype == PTV3_DTYPE_BF16, PTV3_ERR_UNSUPPORTED,
                     "%s: dtype %d of lam", what, p->lam_dtype);
    } else {
        PTV3_REQUIRE(p->n == 0 || !p->grid_coord == !p->table, PTV3_ERR_INVALID_ARGUMENT,
                     "%s: a bias needs both coordinates and a table", what);
    }
    if (p->table) {
        PTV3_REQUIRE(p->pos_bnd >= 0 && p->pos_bnd <= PA_MAX_BOUND, PTV3_ERR_UNSUPPORTED, "%s: pos_bnd %d outside [0, %d]",
                     what, p->pos_bnd, PA_MAX_BOUND);
        PTV3_REQUIRE(p->buckets ? p->num_buckets >= 1 && p->num_buckets <= 2 * p->pos_bnd + 1
                                : p->num_buckets == 2 * p->pos_bnd + 1,
                     PTV3_ERR_INVALID_ARGUMENT, "%s: %d buckets of %d offsets", what, p->num_buckets, 2 * p->pos_bnd + 1);
        PTV3_REQUIRE(p->table_dtype == PTV3_DTYPE_F32 || p->table_dtype == PTV3_DTYPE_BF16, PTV3_ERR_UNSUPPORTED,
                     "%s: dtype %d of the table", what, p->table_dtype);
    }
    PTV3_REQUIRE((int64_t)p->n_seq * ceil_div(longest(p), 64) * p->heads < (1ll << 31), PTV3_ERR_UNSUPPORTED,
                 "%s: too many blocks (%d sequences of up to %d rows, %d heads)", what, p->n_seq, longest(p), p->heads);
    return PTV3_OK;
}

static PatchArgs device_args(const ptv3_patch_attention_args* p)
{
    PatchArgs a = {};
    a.qkv = p->qkv;
    a.out = p->out;
    a.rows = p->rows;
    a.slot = p->n_pad > p->n ? p->rows + p->n_pad : nullptr;
    a.cu = p->cu_seqlens;
    a.n_pad = (int)p->n_pad;
    a.n_seq = p->n_seq;
    a.max_seqlen = p->max_seqlen;
    a.C = p->channels;
    a.H = p->heads;
    a.scale = p->scale;
    a.grid = p->grid_coord;
    a.table = p->table;
    a.buckets = p->buckets;
    a.num = p->num_buckets;
    a.bnd = p->pos_bnd;
    a.table_bf16 = p->table_dtype == PTV3_DTYPE_BF16;
    int32_t* const extent = p->rows + 2 * p->n_pad + (p->n_pad - p->n) + 1;
    a.extent = p->grid_coord ? extent : nullptr;
    a.owner = extent + 6 * (int64_t)p->n_seq;
    a.status = p->status;
    a.second = p->second;
    a.lam = p->lam;
    a.lam_bf16 = p->lam_dtype == PTV3_DTYPE_BF16;
    a.lse = p->lse;
    return a;
}

}  // namespace ptv3

using namespace ptv3;

// the plan's rows, for the attention kernel behind it in the stream
static int launch_rows(const ptv3_patch_attention_args* a, cudaStream_t stream)
{
    const int64_t n = a->n, n_pad = a->n_pad;
    const int borrowed = (int)(n_pad - n);
    PatchPlan p = {a->order, a->pad, a->unpad, a->cu_seqlens, a->grid_coord, a->buckets, (int)n, (int)n_pad, a->n_seq,
                   a->max_seqlen, a->buckets ? 2 * a->pos_bnd + 1 : 0, a->num_buckets, a->grid_coord ? a->n_seq : 0, a->rows,
                   a->lse && borrowed ? a->rows + n_pad : nullptr, a->rows + 2 * n_pad + borrowed + 1,
                   a->rows + 2 * n_pad + borrowed + 1 + 6 * (int64_t)a->n_seq, a->status};
    if (p.slot) {
        const cudaError_t e = cudaMemsetAsync(p.slot, 0xff, (size_t)(n_pad + borrowed + 1) * 4, stream);
        PTV3_REQUIRE(e == cudaSuccess, PTV3_ERR_CUDA, "ptv3_patch_attention_fwd: %s", cudaGetErrorString(e));
    }
    const int64_t most = n_pad > a->n_seq + 1 ? n_pad : a->n_seq + 1;
    launch_dependent(patch_rows_kernel, dim3((unsigned)(p.n_extents + ceil_div(most, 256))), dim3(256), 0, stream, p);
    count_launches(1);
    return check_launch("ptv3_patch_attention_fwd");
}

extern "C" int ptv3_patch_attention_fwd(const ptv3_patch_attention_args* p, void* stream)
{
    int rc = check_sizes(p, "ptv3_patch_attention_fwd");
    if (rc != PTV3_OK) return rc;
    if (p->n == 0) return PTV3_OK;
    PTV3_REQUIRE((((uintptr_t)p->qkv | (uintptr_t)p->out | (uintptr_t)p->second) & 15) == 0, PTV3_ERR_INVALID_ARGUMENT,
                 "ptv3_patch_attention_fwd: unaligned rows");
    PTV3_REQUIRE(p->qkv && p->order && p->pad && p->unpad && p->rows && p->cu_seqlens && p->out && (p->maps == 1 || (p->lam && (!p->lse || p->second))),
                 PTV3_ERR_INVALID_ARGUMENT, "ptv3_patch_attention_fwd: null pointer");
    if ((rc = launch_rows(p, (cudaStream_t)stream)) != PTV3_OK) return rc;
    return launch_patch(p, device_args(p), PA_FWD, (cudaStream_t)stream);
}

extern "C" size_t ptv3_patch_attention_workspace_bytes(const ptv3_patch_attention_args* p)
{
    if (check_sizes(p, "ptv3_patch_attention_workspace_bytes") != PTV3_OK) return 0;
    ptv3_patch_attention_args q = *p;
    q.workspace = nullptr;
    return carve(&q).bytes;
}

extern "C" int ptv3_patch_attention_bwd(const ptv3_patch_attention_args* p, void* stream)
{
    int rc = check_sizes(p, "ptv3_patch_attention_bwd");
    if (rc != PTV3_OK) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    PatchArgs a = device_args(p);
    if (p->n > 0)
        PTV3_REQUIRE(p->qkv && p->order && p->pad && p->unpad && p->rows && p->cu_seqlens && p->out && p->lse && p->dout && p->dqkv &&
                         (p->maps == 1 || (p->lam && p->second)),
                     PTV3_ERR_INVALID_ARGUMENT, "ptv3_patch_attention_bwd: null pointer");
    PTV3_REQUIRE((((uintptr_t)p->qkv | (uintptr_t)p->out | (uintptr_t)p->second | (uintptr_t)p->dout | (uintptr_t)p->dqkv) &
                  15) == 0, PTV3_ERR_INVALID_ARGUMENT,
                 "ptv3_patch_attention_bwd: unaligned rows");
    PTV3_REQUIRE((!p->dtable || p->table) && (!p->dlam || p->maps == 2), PTV3_ERR_INVALID_ARGUMENT,
                 "ptv3_patch_attention_bwd: a gradient without its parameter");
    const PatchWorkspace w = carve(p);
    PTV3_REQUIRE(w.bytes == 0 || (p->workspace && p->workspace_bytes >= w.bytes), PTV3_ERR_WORKSPACE,
                 "ptv3_patch_attention_bwd: workspace of %zu bytes, %zu needed", p->workspace_bytes, w.bytes);
    const bool any = p->n > 0;
    if (any) {
        a.dout = p->dout;
        a.dqkv = p->dqkv;
        a.delta = w.delta;
        a.shared = w.shared;
        a.reach = w.reach;
        a.bins = w.bins;
        a.bin_rows = w.by_rows ? bin_rows(p) : 0;
        if ((rc = launch_patch(p, a, PA_ROWS, s)) != PTV3_OK) return rc;
        if ((rc = launch_patch(p, a, PA_COLS, s)) != PTV3_OK) return rc;
    }
    const int borrowed = (int)(p->n_pad - p->n);
    if (any && borrowed) {
        const int32_t* slot_point = p->rows + 2 * p->n_pad;
        const int64_t total = (int64_t)borrowed * 2 * a.C;
        const int blocks = (int)(total > 256ll * 8 * SMS * 16 ? 8 * SMS * 16 : ceil_div(total, 256));
        if (p->dtype == PTV3_DTYPE_F32)
            launch_dependent(patch_shared_kernel<float>, dim3(blocks), dim3(256), 0, s, w.shared, slot_point, borrowed, a.C,
                             (float*)p->dqkv);
        else
            launch_dependent(patch_shared_kernel<__nv_bfloat16>, dim3(blocks), dim3(256), 0, s, w.shared, slot_point, borrowed,
                             a.C, (__nv_bfloat16*)p->dqkv);
        count_launches(1);
    }
    if (p->dtable) {
        const int wide = a.H * 3 * (2 * a.bnd + 1);
        const float* sums = w.bins;
        int64_t rows = any ? w.blocks : 0;
        if (rows > PA_FOLD) {
            const int folded = ceil_div(rows, PA_FOLD);
            launch_dependent(patch_fold_kernel, dim3(folded, ceil_div(wide, 256)), dim3(256), 0, s, w.bins, rows, wide, w.folded);
            count_launches(1);
            sums = w.folded;
            rows = folded;
        }
        launch_dependent(patch_table_kernel, dim3(3, a.H), dim3(256), 0, s, sums, rows, a.H, a.bnd, a.num, a.buckets,
                         p->dtable, a.table_bf16);
        count_launches(1);
    }
    if (p->dlam) {
        // short launches in one step
        if (any && w.parts > 1) {
            launch_dependent(patch_lam_kernel, dim3(w.parts, a.H), dim3(256), 0, s, w.delta, a.n_pad, w.parts, w.partial,
                             nullptr, 0);
            count_launches(1);
        }
        launch_dependent(patch_lam_kernel, dim3(1, a.H), dim3(256), 0, s, w.delta, any ? a.n_pad : 0, w.parts, w.partial,
                         p->dlam, a.lam_bf16);
        count_launches(1);
    }
    return check_launch("ptv3_patch_attention_bwd");
}
