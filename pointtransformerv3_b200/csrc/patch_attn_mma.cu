// Patch attention with bias or of two maps, forward and backward, for bf16 on the tensor cores by mma.sync
// (patch_attn.cuh has the mathematics).
//
// A CTA of eight warps (or four) owns 128 rows (queries, or keys in the pass over columns) of one patch and head, a warp 16
// of them (or 32); the other side streams through shared memory in chunks of 64 rows, gathered by cp.async through the row list, two
// chunks ahead (three stages, one barrier a chunk).  Scores, probabilities and dS live in accumulator registers and are
// the A operands of the next product as they lie; rounding to bf16 happens there (probabilities, dS) and where results
// are stored, everything else is fp32.  Of a map there are 64 tensor FLOPs to an exponential at heads of 16: the exponential unit
// and instruction issue set the pace, which is why the products stay on mma.sync.
//
// The bias: coordinates are kept times the size of a table entry in bytes, so a look-up is a subtraction with a
// maximum, a minimum, a load and an addition; 32 copies of the table, one to a lane, keep loads and the integer
// additions of the table's gradient free of bank conflicts.
#include "patch_attn.cuh"
#include "mma_util.cuh"

namespace ptv3 {

// Rows of the other side in a stage.  Warps meet once a chunk: with 64 rows instead of 256 the three kernels of 100 000 x 64,
// differential, take 333, 378 and 386 us instead of 311, 343 and 349; a bias needs the room for its table.
template <int W, bool BIAS, int NT>
struct PmChunk {
    static constexpr int N = W == 16 && !BIAS && NT == 256 ? 256 : 64;
};
// Shared memory of a table, and of a table and its bins: smaller CTAs share an SM with more
template <int NT>
struct PmTableBytes {
    static constexpr int TABLE = PA_TABLE_BYTES * NT / 256, BINS = PA_BINS_BYTES * NT / 256;
};
constexpr int PM_STAGES = 3;
constexpr int PM_WINDOW = 256;     // queries between two clearings of the table's bins
constexpr float PM_NEAR = 1024.f;  // references this near zero leave the sum's logarithm 2^-14 of a power of two: less than bf16 shows
constexpr float PM_LAZY = 8.f;     // slack of the running maximum, in powers of two
// bytes for the sums of the bins: entries of a table of eight copies, or of the largest bound (patch_attn.cuh)
static int pm_sums_bytes(int bnd, int bins_bytes)
{
    return (3 * (2 * bnd + 1) > bins_bytes / 64 ? 3 * (2 * bnd + 1) : bins_bytes / 64) * 4;
}

template <int W, int CH>
struct PmStage {
    static constexpr int TILE = CH * W * 2;            // bytes of a matrix
    static constexpr int AUX = 2 * TILE;               // three words of each map and row
    static constexpr int GRID = AUX + 3 * CH * 4;      // coordinates, where there is a bias and one map; or the second map's words
    static constexpr int BYTES = GRID + 3 * CH * 4;
};

// byte offset of 16-byte chunk c of row r: chunks are exchanged so that the eight rows of an ldmatrix lie in different banks
template <int W>
__device__ __forceinline__ uint32_t pm_offset(int r, int c)
{
    constexpr int RB = 2 * W;
    return (uint32_t)(r * RB + ((c ^ ((r * RB >> 7) & (RB / 16 - 1))) << 4));
}

__device__ __forceinline__ void mma_bf16_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0)
{
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(b0));
}

// a coordinate in its sequence's box (of what the plan's rows hold, not of the coordinates as they are now)
__device__ __forceinline__ int pm_box(const PatchArgs& a, int seq, int coord, int c)
{
    return pa_held(coord, a.extent[6 * seq + 3 + c], a.extent[6 * seq + c]);
}
struct PmPlace {
    int h, tile, seq, start, L;
};
__device__ __forceinline__ PmPlace pm_place(const PatchArgs& a)
{
    PmPlace p;
    p.h = blockIdx.x % a.H;
    p.tile = blockIdx.x / a.H % a.tiles;
    p.seq = blockIdx.x / a.H / a.tiles;
    p.L = pa_sequence(a, p.seq, p.start);
    return p;
}
// Bias of a pair of points: coordinates in bytes of the table in shared memory
struct PmBias {
    int lo[3], hi[3];       // bounds of an entry's place, this lane's copy
};
__device__ __forceinline__ float pm_lds(uint32_t addr)
{
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ void pm_add_shared(uint32_t addr, int v)
{
    asm volatile("red.shared.add.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// The other side's rows: x and y (head h's W values of each), three words of each map (AUX), coordinates (BIAS).  The words are
// r, f and -delta of P = f 2^(score + r): near zero r takes the logarithm of the softmax's sum in, and f is 1 or -lam; a reference
// further off has no bits for it, so f is that over the sum, and the chunk is marked.  (100 000 x 64, columns: of two maps 320 us, 364 with f
// multiplied always.  With a bias, whose tables mask, always: 803 us, 784 without f.)  SPREAD: a thread has one coordinate of a row,
// not three, so that no warp comes late to a chunk (rows of heads of 16 447 -> 432 us; forward 397 -> 407, rows of heads of 32 293 -> 295).
template <int W, int MAPS, bool AUX, bool BIAS, bool SPREAD, int NT>
struct PmStream {
    static constexpr int CH = PmChunk<W, BIAS, NT>::N;
    static constexpr int RPP = NT / 4, NR = CH / RPP;
    // coordinates that a thread has at a time, and how often; with a bias it has one word of a row at a time, otherwise three
    static constexpr int GA = SPREAD ? 1 : 3, SLOTS = 3 / GA * CH, NG = BIAS ? (SLOTS + NT - 1) / NT : 1;
    static constexpr int NA = !AUX ? 1 : ((BIAS ? 3 : MAPS) * CH + NT - 1) / NT, AW = BIAS ? 1 : 3;
    static_assert(!(BIAS && MAPS == 2), "coordinates lie where the second map's words do");
    using S = PmStage<W, CH>;
    const PatchArgs& a;
    const __nv_bfloat16 *x, *y;
    int64_t xs, ys;
    int seq, start, L, h;
    bool owners;             // rows of y that answer for no point are taken as zeros
    int step;                // coordinates are kept times 2^step
    float second;            // factor of the second map
    int* marks;              // of the stages: 1 + the last chunk there with a reference far from zero
    unsigned char* smem;
    int e[NR], eg[NG], ea[NA], g[NG][GA];
    float aux[NA][AW];

    __device__ __forceinline__ int row_of(int chunk, int j) const
    {
        const int r = chunk * CH + j;
        return r < L ? a.rows[start + r] : INT_MIN;
    }
    // this thread's i-th coordinates of a chunk: of row k % CH, from axis k / CH on
    static __device__ __forceinline__ int grid_slot(int i) { return threadIdx.x + i * NT; }
    // (of rows beyond the last the last one's: places in the table stay within it)
    __device__ __forceinline__ void fetch_rows(int chunk)
    {
        if (BIAS)
#pragma unroll
            for (int i = 0; i < NG; ++i)
                if (grid_slot(i) < SLOTS) eg[i] = a.rows[start + min(chunk * CH + grid_slot(i) % CH, L - 1)];
    }
    __device__ __forceinline__ void fetch_grid()
    {
        if (BIAS)
#pragma unroll
            for (int i = 0; i < NG; ++i)
                if (grid_slot(i) < SLOTS)
#pragma unroll
                    for (int c = 0; c < GA; ++c)
                        g[i][c] = a.grid[3 * (int64_t)(eg[i] >= 0 ? eg[i] : -(eg[i] + 1)) + grid_slot(i) / CH + c];
    }
    // its i-th word, or three (with a bias other threads than the first have two of these)
    static __device__ __forceinline__ int aux_slot(int i) { return (BIAS ? (threadIdx.x + NT - CH) % NT : threadIdx.x) + i * NT; }
    __device__ __forceinline__ void fetch_aux(int chunk)
    {
        const int64_t all = (int64_t)a.H * MAPS * a.n_pad;
        if (AUX)
#pragma unroll
            for (int i = 0; i < NA; ++i) {
                const int k = aux_slot(i), what = k / CH;
                ea[i] = k < (BIAS ? 3 : MAPS) * CH ? row_of(chunk, k % CH) : INT_MIN;
#pragma unroll
                for (int c = 0; c < AW; ++c) aux[i][c] = 0.f;
                if (ea[i] < 0) continue;
                const int64_t at = (int64_t)(h * MAPS + (BIAS ? 0 : what)) * a.n_pad + start + chunk * CH + k % CH;
                if (BIAS) {
                    aux[i][0] = what == 2 ? a.delta[at] : a.lse[what == 1 ? at + all : at];
                } else {
                    aux[i][0] = a.lse[at];
                    aux[i][AW / 2] = a.lse[at + all];
                    aux[i][AW - 1] = a.delta[at];
                }
            }
    }
    // what issue(chunk) needs in registers
    __device__ __forceinline__ void fetch(int chunk)
    {
#pragma unroll
        for (int i = 0; i < NR; ++i) e[i] = row_of(chunk, (threadIdx.x >> 2) + RPP * i);
        fetch_grid();
        fetch_rows(chunk + 1);
        fetch_aux(chunk);
    }
    __device__ __forceinline__ void issue(int chunk)
    {
        if (chunk * CH < L) {
            unsigned char* st = smem + chunk % PM_STAGES * S::BYTES;
            constexpr int CPR = W / 8;
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int r = (threadIdx.x >> 2) + RPP * n;
                const bool there = e[n] != INT_MIN;
                const int64_t p = !there ? 0 : e[n] >= 0 ? e[n] : -(e[n] + 1);
#pragma unroll
                for (int i = 0; i < CPR / 2; ++i) {
                    const int o = (threadIdx.x & 3) + 4 * i, c = o % CPR;
                    if (o < CPR) cp_async16_zfill(smem_u32(st) + pm_offset<W>(r, c), x + p * xs + 8 * c, there);
                    else cp_async16_zfill(smem_u32(st) + S::TILE + pm_offset<W>(r, c), y + p * ys + 8 * c,
                                          there && !(owners && e[n] < 0));
                }
            }
            if (AUX)
#pragma unroll
                for (int i = 0; i < NA; ++i) {
                    const int k = aux_slot(i);
                    float* to = (float*)(st + S::AUX) + k;
                    // rows that are not there, or answer for no point: probabilities of nothing
                    const bool there = ea[i] >= 0;
                    if (BIAS) {
                        if (k < 3 * CH) to[0] = k < CH && !there ? -INFINITY : k / CH == 1 ? aux[i][0] : -aux[i][0];
                    } else if (k < MAPS * CH) {
                        const bool far = there && !(fabsf(aux[i][0]) < PM_NEAR);
                        const float f = k < CH ? 1.f : second, inv = aux[i][AW / 2];
                        to[0] = !there ? -INFINITY : far ? -aux[i][0] : log2f(inv) - aux[i][0];
                        to[MAPS * CH] = !there ? 0.f : far ? f * inv : f;
                        to[2 * MAPS * CH] = -aux[i][AW - 1];
                        if (far) marks[chunk % PM_STAGES] = chunk + 1;
                    }
                }
            if (BIAS)
#pragma unroll
                for (int i = 0; i < NG; ++i)
                    if (grid_slot(i) < SLOTS)
#pragma unroll
                        for (int c = 0; c < GA; ++c)
                            ((int*)(st + S::GRID))[c * CH + grid_slot(i)] =
                                pa_other(pm_box(a, seq, g[i][c], grid_slot(i) / CH + c), step);
        }
        cp_async_commit();
    }
    __device__ __forceinline__ void begin()
    {
        fetch_rows(0);
        fetch(0);
        issue(0);
        fetch(1);
        issue(1);
        fetch(2);
    }
    // chunk i has landed, its stage is returned; chunk i + 2 is on its way, what the one after needs is asked for
    __device__ __forceinline__ const unsigned char* next(int i)
    {
        cp_async_wait<1>();
        __syncthreads();
        issue(i + 2);
        fetch(i + 3);
        return smem + i % PM_STAGES * S::BYTES;
    }
    __device__ __forceinline__ void end()
    {
        cp_async_wait<0>();
        __syncthreads();
    }
};

// ---- fragments ----------------------------------------------------------------------------------------------
// A operand of 16 rows: W values of each, rows p0 and p1 of this lane (NULL: zeros)
template <int W>
__device__ __forceinline__ void pm_rows(const __nv_bfloat16* p0, const __nv_bfloat16* p1, uint32_t flip, uint32_t (&f)[W / 16][4])
{
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int k = 0; k < W / 16; ++k)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            f[k][2 * half] = p0 ? ((const uint32_t*)p0)[8 * k + 4 * half + t] ^ flip : 0u;
            f[k][2 * half + 1] = p1 ? ((const uint32_t*)p1)[8 * k + 4 * half + t] ^ flip : 0u;
        }
}

// s[rt][m] = 16 rows of this warp x 16 rows of the tile, transposed: MAPS sums of W / MAPS products each
template <int W, int MAPS, int RT>
__device__ __forceinline__ void pm_products(const uint32_t (&f)[RT][W / 16][4], uint32_t tile, int row0,
                                            float (&s)[RT][MAPS][2][4])
{
    const int lane = threadIdx.x & 31, r = row0 + (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;
#pragma unroll
    for (int x = 0; x < RT; ++x)
#pragma unroll
        for (int m = 0; m < MAPS; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[x][m][i][j] = 0.f;
#pragma unroll
    for (int k = 0; k < W / 16; ++k) {
        uint32_t b[4];
        ldmatrix_x4(b, tile + pm_offset<W>(r, 2 * k + c));
#pragma unroll
        for (int x = 0; x < RT; ++x) {
            if (W / MAPS == 8) {
                // a map's eight values are one half of the fragment
                mma_bf16_k8(s[x][0][0], f[x][k][0], f[x][k][1], b[0]);
                mma_bf16_k8(s[x][0][1], f[x][k][0], f[x][k][1], b[2]);
                mma_bf16_k8(s[x][MAPS - 1][0], f[x][k][2], f[x][k][3], b[1]);
                mma_bf16_k8(s[x][MAPS - 1][1], f[x][k][2], f[x][k][3], b[3]);
            } else {
                const int m = k * 16 / (W / MAPS);
                mma_bf16(s[x][m][0], f[x][k], b[0], b[1]);
                mma_bf16(s[x][m][1], f[x][k], b[2], b[3]);
            }
        }
    }
}

// the same for 8 rows of the tile
template <int W, int MAPS, int RT>
__device__ __forceinline__ void pm_products8(const uint32_t (&f)[RT][W / 16][4], uint32_t tile, int row0, float (&s)[RT][MAPS][4])
{
    const int lane = threadIdx.x & 31, r = row0 + (lane & 7), c = (lane >> 3) & 1;
#pragma unroll
    for (int x = 0; x < RT; ++x)
#pragma unroll
        for (int m = 0; m < MAPS; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[x][m][j] = 0.f;
#pragma unroll
    for (int k = 0; k < W / 16; ++k) {
        uint32_t b0, b1;
        asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];\n"
                     : "=r"(b0), "=r"(b1)
                     : "r"(tile + pm_offset<W>(r, 2 * k + c)));
#pragma unroll
        for (int x = 0; x < RT; ++x) {
            if (W / MAPS == 8) {
                mma_bf16_k8(s[x][0], f[x][k][0], f[x][k][1], b0);
                mma_bf16_k8(s[x][MAPS - 1], f[x][k][2], f[x][k][3], b1);
            } else {
                mma_bf16(s[x][k * 16 / (W / MAPS)], f[x][k], b0, b1);
            }
        }
    }
}

// acc += P x 16 rows of the tile (W values each); P of map m for the values of map m, or one P for all (MAPS = 1).  With
// `acc2` the same of P2 to that.
template <int W, int MAPS, int RT, bool TWO = false>
__device__ __forceinline__ void pm_accumulate(const uint32_t (&p)[RT][MAPS][4], uint32_t tile, int row0,
                                              float (&acc)[RT][W / 8][4], const uint32_t (&p2)[RT][MAPS][4],
                                              float (&acc2)[RT][W / 8][4])
{
    constexpr int D = W / MAPS;
    const int lane = threadIdx.x & 31, r = row0 + (lane & 15), c = lane >> 4;
#pragma unroll
    for (int k = 0; k < W / 16; ++k) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, tile + pm_offset<W>(r, 2 * k + c));
#pragma unroll
        for (int x = 0; x < RT; ++x) {
            mma_bf16(acc[x][2 * k], p[x][16 * k / D], b[0], b[1]);
            mma_bf16(acc[x][2 * k + 1], p[x][(16 * k + 8) / D], b[2], b[3]);
            if (TWO) {
                mma_bf16(acc2[x][2 * k], p2[x][16 * k / D], b[0], b[1]);
                mma_bf16(acc2[x][2 * k + 1], p2[x][(16 * k + 8) / D], b[2], b[3]);
            }
        }
    }
}

// whether places in the table have to be held within it
struct PmYes {
    static constexpr bool value = true;
};
struct PmNo {
    static constexpr bool value = false;
};

// ---- bias ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ void pm_bias_setup(const PatchTable& t, uint32_t base, PmBias& b)
{
    const int copy = (threadIdx.x & ((1 << t.copies_log2) - 1)) * 4, step = t.copies_log2 + 2;
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        b.lo[c] = (int)base + (t.first[c] << step) + copy;
        b.hi[c] = b.lo[c] + ((2 * t.reach[c]) << step);
    }
}
// row r's point, so that subtracting another's coordinates gives the entry's place
__device__ __forceinline__ void pm_bias_point(const PatchArgs& a, const PatchTable& t, const PmBias& b, const PmPlace& w, int r,
                                              int sign, int (&g)[3])
{
    const int e = a.rows[w.start + min(r, w.L - 1)];
    const int64_t p = e >= 0 ? e : -(e + 1);
#pragma unroll
    for (int c = 0; c < 3; ++c)
        g[c] = pa_mine(b.lo[c], t.reach[c], pm_box(a, w.seq, a.grid[3 * p + c], c), sign, t.copies_log2 + 2);
}
// coordinates of the other side's rows j and j + 1
template <int CH>
__device__ __forceinline__ void pm_coords(const int* gs, int j, int2 (&o)[3])
{
#pragma unroll
    for (int c = 0; c < 3; ++c) o[c] = *(const int2*)(gs + c * CH + j);
}
// places of the entries of four pairs (rows g[0], g[1] of this lane and two of the other side); SIGN: the lane's point is
// the query (+1) or the key
template <int SIGN, bool CLAMP>
__device__ __forceinline__ void pm_places(const PmBias& b, const int (&g)[2][3], const int2 (&o)[3], uint32_t (&at)[4][3])
{
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        auto place = [&](int mine, int other) {
            return (uint32_t)(CLAMP ? min(__viaddmax_s32(mine, -SIGN * other, b.lo[c]), b.hi[c]) : mine - SIGN * other);
        };
        at[0][c] = place(g[0][c], o[c].x);
        at[1][c] = place(g[0][c], o[c].y);
        at[2][c] = place(g[1][c], o[c].x);
        at[3][c] = place(g[1][c], o[c].y);
    }
}
// scores and biases of four pairs, in powers of two
__device__ __forceinline__ void pm_bias(const uint32_t (&at)[4][3], float scale2, float (&s)[4])
{
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
        uint64_t t[3];
#pragma unroll
        for (int c = 0; c < 3; ++c) t[c] = pack2(pm_lds(at[r][c]), pm_lds(at[r + 1][c]));
        unpack2(add2(fma2(pack2(s[r], s[r + 1]), pack2(scale2, scale2), t[0]), add2(t[1], t[2])), s[r], s[r + 1]);
    }
}

__device__ __forceinline__ float pm_max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x of both
__device__ __forceinline__ uint64_t pm_exp2(uint64_t x)
{
    float a, b;
    unpack2(x, a, b);
    return pack2(fast_exp2(a), fast_exp2(b));
}
__device__ __forceinline__ uint64_t pm_both(float v) { return pack2(v, v); }

// this lane's rows of the RT tiles of its warp: row g + 8 r of tile x
template <int RT>
struct PmOwn {
    int row[RT][2], e[RT][2];      // e: of the row list, -1 for rows that are not there
    bool any;                      // whether one of the warp's answers for a point
    __device__ __forceinline__ void load(const PatchArgs& a, const PmPlace& w, int first)
    {
        any = false;
#pragma unroll
        for (int x = 0; x < RT; ++x)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                row[x][r] = first + (int)(threadIdx.x / 32) * 16 * RT + 16 * x + ((threadIdx.x & 31) >> 2) + 8 * r;
                e[x][r] = row[x][r] < w.L ? a.rows[w.start + row[x][r]] : -1;
                any |= e[x][r] >= 0;
            }
        any = __any_sync(0xffffffffu, any);
    }
};
// fragments of a matrix's rows (this head's W values from `base` on), zeros for rows that answer for no point
template <int W, int RT>
__device__ __forceinline__ void pm_own_rows(const PmOwn<RT>& own, const __nv_bfloat16* base, int64_t stride, uint32_t flip,
                                            uint32_t (&f)[RT][W / 16][4])
{
#pragma unroll
    for (int x = 0; x < RT; ++x)
        pm_rows<W>(own.e[x][0] >= 0 ? base + own.e[x][0] * stride : nullptr,
                   own.e[x][1] >= 0 ? base + own.e[x][1] * stride : nullptr, flip, f[x]);
}

// ------------------------------------------------------------------------------------------------- forward
template <int W, int MAPS, bool BIAS, bool KEEP, int RT, int NT>
__global__ void __launch_bounds__(NT, (W == 64 && (MAPS == 2 || RT == 2) ? 256 : 512) / NT) patch_mma_fwd_kernel(const PatchArgs a)
{
    pdl_wait();
    constexpr int CH = PmChunk<W, BIAS, NT>::N;
    using S = PmStage<W, CH>;
    extern __shared__ __align__(128) unsigned char smem[];
    const PmPlace w = pm_place(a);
    const int q0 = w.tile * (NT / 2) * RT, L = w.L;
    if (q0 >= L) return;
    if (w.h == 0 && a.status) pa_check_owners(a.rows, a.owner, a.status, w.start + q0, w.start + min(q0 + NT / 2 * RT, L));
    const int t = threadIdx.x & 3;
    PmOwn<RT> own;
    own.load(a, w, q0);
    if (!__syncthreads_or(own.any)) return;         // (a scene's last patch may end in borrowed rows alone)
    const int64_t stride = 3 * (int64_t)a.C;
    const __nv_bfloat16* base = (const __nv_bfloat16*)a.qkv + w.h * W;
    PatchTable table = {};
    if (BIAS) table = pa_table(a, w.seq, PmTableBytes<NT>::TABLE, false);
    PmStream<W, MAPS, false, BIAS, false, NT> in = {a, base + a.C, base + 2 * a.C, stride, stride, w.seq, w.start, L, w.h, false,
                                         table.copies_log2 + 2, 0.f, nullptr, smem};
    in.begin();
    PmBias bias;
    int point[RT][2][3];
    if (BIAS) {
        float* tab = (float*)(smem + PM_STAGES * S::BYTES);
        pa_load_table(a, table, w.h, tab, threadIdx.x, NT);      // (the first chunk's barrier stands behind it)
        pm_bias_setup(table, smem_u32(tab), bias);
#pragma unroll
        for (int x = 0; x < RT; ++x)
#pragma unroll
            for (int r = 0; r < 2; ++r) pm_bias_point(a, table, bias, w, own.row[x][r], 1, point[x][r]);
    }
    uint32_t q[RT][W / 16][4];
    // (of a negative scale the sign goes to the queries, so that larger products are larger scores)
    pm_own_rows<W, RT>(own, base, stride, a.scale < 0.f ? 0x80008000u : 0u, q);
    const float scale2 = fabsf(a.scale) * PA_LOG2E;
    float o[MAPS][RT][W / 8][4], sum[MAPS][RT][4], m[MAPS][RT][2];
    uint64_t l[MAPS][RT][2];
#pragma unroll
    for (int k = 0; k < MAPS; ++k)
#pragma unroll
        for (int x = 0; x < RT; ++x) {
            m[k][x][0] = m[k][x][1] = PA_LOWEST;
            l[k][x][0] = l[k][x][1] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sum[k][x][j] = 0.f;
#pragma unroll
                for (int i = 0; i < W / 8; ++i) o[k][x][i][j] = 0.f;
            }
        }
    constexpr uint32_t ONES = 0x3f803f80u;
    constexpr int KG = 32 / RT;      // keys whose scores are held at a time
    auto walk = [&](auto clamp) {
        constexpr bool CLAMP = decltype(clamp)::value;
        for (int i = 0; i * CH < L; ++i) {
            const unsigned char* st = in.next(i);
            if (!own.any) continue;
            const uint32_t ks = smem_u32(st), vs = ks + S::TILE;
            const int* gs = (const int*)(st + S::GRID);
            const int nk = L - i * CH;
#pragma unroll 2
            for (int j0 = 0; j0 < CH; j0 += KG) {
                if (j0 >= nk) break;
                float s[KG / 16][RT][MAPS][2][4];
#pragma unroll
                for (int u = 0; u < KG / 16; ++u) {
                    pm_products<W, MAPS, RT>(q, ks, j0 + 16 * u, s[u]);
                    if (BIAS)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            int2 g[3];
                            pm_coords<CH>(gs, j0 + 16 * u + 8 * n + 2 * t, g);
#pragma unroll
                            for (int x = 0; x < RT; ++x) {
                                uint32_t at[4][3];
                                pm_places<1, CLAMP>(bias, point[x], g, at);
                                pm_bias(at, scale2, s[u][x][0][n]);
                            }
                        }
                    if (j0 + KG > nk)
#pragma unroll
                        for (int x = 0; x < RT; ++x)
#pragma unroll
                            for (int k = 0; k < MAPS; ++k)
#pragma unroll
                                for (int n = 0; n < 2; ++n)
#pragma unroll
                                    for (int c = 0; c < 4; ++c)
                                        if (j0 + 16 * u + 8 * n + 2 * t + (c & 1) >= nk) s[u][x][k][n][c] = -INFINITY;
                }
#pragma unroll
                for (int k = 0; k < MAPS; ++k) {
#pragma unroll
                    for (int x = 0; x < RT; ++x) {
                        float top[2];
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            top[r] = fmaxf(s[0][x][k][0][2 * r], s[0][x][k][0][2 * r + 1]);
#pragma unroll
                            for (int u = 0; u < KG / 16; ++u)
#pragma unroll
                                for (int n = 0; n < 2; ++n)
                                    if (u + n) top[r] = pm_max3(top[r], s[u][x][k][n][2 * r], s[u][x][k][n][2 * r + 1]);
                            if (!BIAS) top[r] *= scale2;
                        }
                        if (__any_sync(0xffffffffu, top[0] > m[k][x][0] + PM_LAZY || top[1] > m[k][x][1] + PM_LAZY)) {
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                                top[r] = fmaxf(m[k][x][r], fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2)));
                                const float fix = fast_exp2(m[k][x][r] - top[r]);
                                m[k][x][r] = top[r];
                                l[k][x][r] = mul2(l[k][x][r], pm_both(fix));
                                sum[k][x][2 * r] *= fix;
#pragma unroll
                                for (int n = 0; n < W / 8; ++n) {
                                    o[k][x][n][2 * r] *= fix;
                                    o[k][x][n][2 * r + 1] *= fix;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int u = 0; u < KG / 16; ++u) {
                        uint32_t p[RT][1][4];
#pragma unroll
                        for (int x = 0; x < RT; ++x) {
#pragma unroll
                            for (int n = 0; n < 2; ++n)
#pragma unroll
                                for (int r = 0; r < 2; ++r) {
                                    const uint64_t v = pack2(s[u][x][k][n][2 * r], s[u][x][k][n][2 * r + 1]);
                                    const uint64_t e = pm_exp2(BIAS ? add2(v, pm_both(-m[k][x][r]))
                                                                    : fma2(v, pm_both(scale2), pm_both(-m[k][x][r])));
                                    if (KEEP) l[k][x][r] = add2(l[k][x][r], e);
                                    float y, z;
                                    unpack2(e, y, z);
                                    p[x][0][2 * n + r] = pack_bf16(y, z);
                                }
                            // the sum that the result is divided by is that of the rounded probabilities
                            mma_bf16(sum[k][x], p[x][0], ONES, ONES);
                        }
                        pm_accumulate<W, 1, RT>(p, vs, j0 + 16 * u, o[k], p, o[k]);
                    }
                }
            }
        }
    };
    if (BIAS && table.clamps) walk(PmYes());
    else walk(PmNo());
    in.end();
    if (!own.any) return;
    const float lam = MAPS == 2 ? pa_param(a.lam, w.h, a.lam_bf16) : 0.f;
#pragma unroll
    for (int x = 0; x < RT; ++x)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int e = own.e[x][r];
            if (KEEP)
#pragma unroll
                for (int k = 0; k < MAPS; ++k) {
                    float v = hsum2(l[k][x][r]);
                    v += __shfl_xor_sync(0xffffffffu, v, 1);
                    v += __shfl_xor_sync(0xffffffffu, v, 2);
                    if (t == 0 && e >= 0) {
                        float* to = a.lse + (int64_t)(w.h * MAPS + k) * a.n_pad + w.start + own.row[x][r];
                        *to = m[k][x][r];
                        to[(int64_t)a.H * MAPS * a.n_pad] = 1.f / v;
                    }
                }
            if (e < 0) continue;
            const float w0 = 1.f / sum[0][x][2 * r], w2 = 1.f / sum[MAPS - 1][x][2 * r], w1 = lam * w2;
            const int64_t at = (int64_t)e * a.C + w.h * W;
#pragma unroll
            for (int n = 0; n < W / 8; ++n) {
                float y = o[0][x][n][2 * r] * w0, z = o[0][x][n][2 * r + 1] * w0;
                if (MAPS == 2) {
                    y -= o[MAPS - 1][x][n][2 * r] * w1;
                    z -= o[MAPS - 1][x][n][2 * r + 1] * w1;
                }
                ((uint32_t*)((__nv_bfloat16*)a.out + at))[4 * n + t] = pack_bf16(y, z);
                if (MAPS == 2 && KEEP)
                    ((uint32_t*)((__nv_bfloat16*)a.second + at))[4 * n + t] =
                        pack_bf16(o[MAPS - 1][x][n][2 * r] * w2, o[MAPS - 1][x][n][2 * r + 1] * w2);
            }
        }
}

// ------------------------------------------------------------------------- backward, a warp's own queries
// row g and row g + 8 of two fragments: sums of products over the four lanes that hold them
template <int W>
__device__ __forceinline__ void pm_row_dots(const uint32_t (&x)[W / 16][4], const uint32_t (&y)[W / 16][4], float (&d)[2])
{
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < W / 16; ++k)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float x0, x1, y0, y1;
                unpack2(unpack_bf16x2(x[k][2 * half + r]), x0, x1);
                unpack2(unpack_bf16x2(y[k][2 * half + r]), y0, y1);
                v = fmaf(x0, y0, fmaf(x1, y1, v));
            }
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        d[r] = v + __shfl_xor_sync(0xffffffffu, v, 2);
    }
}

template <int W, int MAPS, bool BIAS, int RT, int NT>
__global__ void __launch_bounds__(NT, (W == 64 ? 256 : 512) / NT) patch_mma_rows_kernel(const PatchArgs a)
{
    pdl_wait();
    constexpr int CH = PmChunk<W, BIAS, NT>::N;
    using S = PmStage<W, CH>;
    extern __shared__ __align__(128) unsigned char smem[];
    const PmPlace w = pm_place(a);
    const int q0 = w.tile * (NT / 2) * RT, L = w.L;
    if (q0 >= L) return;
    const int t = threadIdx.x & 3;
    PmOwn<RT> own;
    own.load(a, w, q0);
    const int64_t stride = 3 * (int64_t)a.C;
    const __nv_bfloat16* base = (const __nv_bfloat16*)a.qkv + w.h * W;
    PatchTable table = {};
    if (BIAS) table = pa_table(a, w.seq, PmTableBytes<NT>::TABLE, false);
    PmStream<W, MAPS, false, BIAS, W == 16, NT> in = {a, base + a.C, base + 2 * a.C, stride, stride, w.seq, w.start, L, w.h, false,
                                         table.copies_log2 + 2, 0.f, nullptr, smem};
    in.begin();
    PmBias bias;
    int point[RT][2][3];
    if (BIAS) {
        float* tab = (float*)(smem + PM_STAGES * S::BYTES);
        pa_load_table(a, table, w.h, tab, threadIdx.x, NT);
        pm_bias_setup(table, smem_u32(tab), bias);
#pragma unroll
        for (int x = 0; x < RT; ++x)
#pragma unroll
            for (int r = 0; r < 2; ++r) pm_bias_point(a, table, bias, w, own.row[x][r], 1, point[x][r]);
    }
    uint32_t q[RT][W / 16][4], go[RT][W / 16][4];
    float ref[MAPS][RT][2], shift[MAPS][RT][2], most[RT][2];
    uint64_t E[MAPS][RT][2], total[MAPS][RT][2];
    const float lam = MAPS == 2 ? pa_param(a.lam, w.h, a.lam_bf16) : 0.f;
    pm_own_rows<W, RT>(own, (const __nv_bfloat16*)a.dout + w.h * W, a.C, 0u, go);
    pm_own_rows<W, RT>(own, (const __nv_bfloat16*)a.out + w.h * W, a.C, 0u, q);
#pragma unroll
    for (int x = 0; x < RT; ++x) pm_row_dots<W>(go[x], q[x], shift[0][x]);
    if (MAPS == 2) {
        pm_own_rows<W, RT>(own, (const __nv_bfloat16*)a.second + w.h * W, a.C, 0u, q);
#pragma unroll
        for (int x = 0; x < RT; ++x) {
            pm_row_dots<W>(go[x], q[x], shift[MAPS - 1][x]);
            shift[0][x][0] += lam * shift[MAPS - 1][x][0];
            shift[0][x][1] += lam * shift[MAPS - 1][x][1];
        }
    }
    pm_own_rows<W, RT>(own, base, stride, 0u, q);
    const float scale2 = a.scale * PA_LOG2E;
    float dq[RT][W / 8][4], pk[RT][W / 8][4];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
        most[x][0] = most[x][1] = 0.f;
#pragma unroll
        for (int n = 0; n < W / 8; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) dq[x][n][c] = pk[x][n][c] = 0.f;
#pragma unroll
        for (int k = 0; k < MAPS; ++k)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                ref[k][x][r] = own.e[x][r] >= 0 ? a.lse[(int64_t)(w.h * MAPS + k) * a.n_pad + w.start + own.row[x][r]]
                                                : INFINITY;
                E[k][x][r] = total[k][x][r] = 0;
            }
    }

    auto walk = [&](auto clamp) {
        constexpr bool CLAMP = decltype(clamp)::value;
        for (int i = 0; i * CH < L; ++i) {
            const unsigned char* st = in.next(i);
            if (!own.any) continue;
            const uint32_t ks = smem_u32(st), vs = ks + S::TILE;
            const int* gs = (const int*)(st + S::GRID);
            const int nk = L - i * CH;
#pragma unroll (2 / RT)
            for (int j0 = 0; j0 < CH; j0 += 16) {
                if (j0 >= nk) break;
                float s[RT][MAPS][2][4], G[RT][1][2][4];
                pm_products<W, MAPS, RT>(q, ks, j0, s);
                pm_products<W, 1, RT>(go, vs, j0, G);
                if (BIAS)
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        int2 g[3];
                        pm_coords<CH>(gs, j0 + 8 * n + 2 * t, g);
#pragma unroll
                        for (int x = 0; x < RT; ++x) {
                            uint32_t at[4][3];
                            pm_places<1, CLAMP>(bias, point[x], g, at);
                            pm_bias(at, scale2, s[x][0][n]);
                        }
                    }
                if (j0 + 16 > nk)
#pragma unroll
                    for (int x = 0; x < RT; ++x)
#pragma unroll
                        for (int k = 0; k < MAPS; ++k)
#pragma unroll
                            for (int n = 0; n < 2; ++n)
#pragma unroll
                                for (int c = 0; c < 4; ++c)
                                    if (j0 + 8 * n + 2 * t + (c & 1) >= nk)
                                        s[x][k][n][c] = BIAS || a.scale > 0.f ? -INFINITY : INFINITY;
                uint32_t p[RT][MAPS][4], d[RT][MAPS][4];
#pragma unroll
                for (int x = 0; x < RT; ++x)
#pragma unroll
                    for (int k = 0; k < MAPS; ++k)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const uint64_t v = pack2(s[x][k][n][2 * r], s[x][k][n][2 * r + 1]);
                                const uint64_t pr = pm_exp2(BIAS ? add2(v, pm_both(-ref[k][x][r]))
                                                                 : fma2(v, pm_both(scale2), pm_both(-ref[k][x][r])));
                                total[k][x][r] = add2(total[k][x][r], pr);
                                const uint64_t ds = mul2(pr, add2(pack2(G[x][0][n][2 * r], G[x][0][n][2 * r + 1]),
                                                                  pm_both(-shift[k][x][r])));
                                E[k][x][r] = add2(E[k][x][r], ds);
                                float y, z;
                                unpack2(pr, y, z);
                                p[x][k][2 * n + r] = pack_bf16(y, z);
                                unpack2(ds, y, z);
                                d[x][k][2 * n + r] = pack_bf16(y, z);
                                if (BIAS) most[x][r] += fabsf(y) + fabsf(z);
                            }
                pm_accumulate<W, MAPS, RT, true>(d, ks, j0, dq, p, pk);
            }
        }
    };
    if (BIAS && table.clamps) walk(PmYes());
    else walk(PmNo());
    in.end();
    auto quad = [](float v) {
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        return v + __shfl_xor_sync(0xffffffffu, v, 2);
    };
#pragma unroll
    for (int x = 0; x < RT; ++x)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int e = own.e[x][r], row = own.row[x][r];
            float by[MAPS], eps[MAPS];
#pragma unroll
            for (int k = 0; k < MAPS; ++k) {
                // (probabilities so far are times their row's sum)
                const float sum = quad(hsum2(total[k][x][r])), inv = e >= 0 ? 1.f / sum : 0.f;
                eps[k] = quad(hsum2(E[k][x][r])) * inv;
                by[k] = inv * a.scale * (k == 1 ? -lam : 1.f);
                if (t == 0 && row < L)
                    a.delta[(int64_t)(w.h * MAPS + k) * a.n_pad + w.start + row] = e >= 0 ? shift[k][x][r] + eps[k] : 0.f;
                if (BIAS && a.reach) {
                    const float reach = quad(most[x][r]) * inv + fabsf(eps[0]);
                    if (t == 0 && row < L) a.reach[(int64_t)w.h * a.n_pad + w.start + row] = e >= 0 ? reach : 0.f;
                }
            }
            if (e < 0) continue;
            uint32_t* dst = (uint32_t*)((__nv_bfloat16*)a.dqkv + e * stride + w.h * W);
#pragma unroll
            for (int n = 0; n < W / 8; ++n) {
                const int k = n * 8 / (W / MAPS);
                dst[4 * n + t] = pack_bf16((dq[x][n][2 * r] - eps[k] * pk[x][n][2 * r]) * by[k],
                                           (dq[x][n][2 * r + 1] - eps[k] * pk[x][n][2 * r + 1]) * by[k]);
            }
        }
}

// --------------------------------------------------------------------------- backward, a warp's own keys
template <int W, int MAPS, bool BIAS, int RT, int NT>
__global__ void __launch_bounds__(NT, (W == 64 || (W == 32 && RT == 2 && BIAS) ? 256 : W == 32 && RT == 2 ? 384 : 512) / NT) patch_mma_cols_kernel(const PatchArgs a)
{
    pdl_wait();
    constexpr int CH = PmChunk<W, BIAS, NT>::N;
    using S = PmStage<W, CH>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float part[4 * NT / 32];
    __shared__ int marks[PM_STAGES];       // (as they come: a chunk taken for marked is as right, and slower)
    const PmPlace w = pm_place(a);
    const int k0 = w.tile * (NT / 2) * RT, L = w.L;
    const bool learns = BIAS && a.bins;
    float* bins = learns ? pa_bins<NT / 2 * RT>(a, w.seq, w.tile, w.h, w.start, L, NT) : nullptr;
    if (k0 >= L) return;
    const int t = threadIdx.x & 3, warp0 = k0 + (int)(threadIdx.x / 32) * 16 * RT;
    PmOwn<RT> own;
    own.load(a, w, k0);
    const int64_t stride = 3 * (int64_t)a.C;
    const __nv_bfloat16* base = (const __nv_bfloat16*)a.qkv + w.h * W;
    PatchTable table = {};
    if (BIAS) table = pa_table(a, w.seq, PmTableBytes<NT>::BINS, true);
    const float minus_lam = MAPS == 2 ? -pa_param(a.lam, w.h, a.lam_bf16) : 0.f;
    PmStream<W, MAPS, true, BIAS, false, NT> in = {a, base, (const __nv_bfloat16*)a.dout + w.h * W, stride, a.C, w.seq, w.start, L, w.h, true,
                                        table.copies_log2 + 2, minus_lam, marks, smem};
    in.begin();
    float* tab = (float*)(smem + PM_STAGES * S::BYTES);
    int* hist = (int*)(tab + (BIAS ? table.entries << table.copies_log2 : 0));
    float* sums = (float*)hist + (BIAS ? table.entries << table.bins_log2 : 0);
    // from an entry's place to its bin's, in copies of this lane's number
    const int fewer = table.copies_log2 - table.bins_log2, lane = threadIdx.x & 31;
    const uint32_t to_hist = smem_u32(hist) + 4 * (lane & ((1 << table.bins_log2) - 1)) -
                             ((smem_u32(tab) + 4 * (lane & ((1 << table.copies_log2) - 1))) >> fewer);
    PmBias bias;
    int point[RT][2][3];
    float unit = 0.f, per_unit = 0.f;
    if (BIAS) {
        pa_load_table(a, table, w.h, tab, threadIdx.x, NT);
        pm_bias_setup(table, smem_u32(tab), bias);
#pragma unroll
        for (int x = 0; x < RT; ++x)
#pragma unroll
            for (int r = 0; r < 2; ++r) pm_bias_point(a, table, bias, w, own.row[x][r], -1, point[x][r]);
        if (learns) {
            for (int i = threadIdx.x; i < table.entries << table.bins_log2; i += NT) hist[i] = 0;
            for (int i = threadIdx.x; i < table.entries; i += NT) sums[i] = 0.f;
        }
    }
    uint32_t kf[RT][W / 16][4], vf[RT][W / 16][4];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
        const __nv_bfloat16* p[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int e = own.e[x][r];
            p[r] = own.row[x][r] < L ? base + a.C + (e >= 0 ? e : -(e + 1)) * stride : nullptr;
        }
        pm_rows<W>(p[0], p[1], 0u, kf[x]);
        pm_rows<W>(p[0] ? p[0] + a.C : nullptr, p[1] ? p[1] + a.C : nullptr, 0u, vf[x]);
    }
    const float scale2 = a.scale * PA_LOG2E;
    float dk[RT][W / 8][4], dv[RT][W / 8][4];
#pragma unroll
    for (int x = 0; x < RT; ++x)
#pragma unroll
        for (int n = 0; n < W / 8; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) dk[x][n][c] = dv[x][n][c] = 0.f;

    auto chunk = [&](int i, const unsigned char* st, auto clamp, auto far) {
        constexpr bool CLAMP = decltype(clamp)::value, FAR = decltype(far)::value;
        const uint32_t qs = smem_u32(st), os = qs + S::TILE;
        const float* aux = (const float*)(st + S::AUX);
        const int* gs = (const int*)(st + S::GRID);
        const int nq = L - i * CH;
#pragma unroll (2 / RT)
        for (int j0 = 0; j0 < CH; j0 += 16) {
            if (j0 >= nq) break;
            uint32_t p[RT][MAPS][4], pm[RT][1][4];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int j = j0 + 8 * n + 2 * t;
                float s[RT][MAPS][4], G[RT][1][4];
                pm_products8<W, MAPS, RT>(kf, qs, j0 + 8 * n, s);
                pm_products8<W, 1, RT>(vf, os, j0 + 8 * n, G);
                int2 g[3];
                if (BIAS) pm_coords<CH>(gs, j, g);
                uint64_t ref[MAPS], coef[MAPS], delta[MAPS];
#pragma unroll
                for (int k = 0; k < MAPS; ++k) {
                    ref[k] = *(const uint64_t*)(aux + k * CH + j);
                    if (FAR) coef[k] = *(const uint64_t*)(aux + (MAPS + k) * CH + j);
                    delta[k] = *(const uint64_t*)(aux + (2 * MAPS + k) * CH + j);
                }
#pragma unroll
                for (int x = 0; x < RT; ++x) {
                    uint32_t at[4][3];
                    if (BIAS) {
                        pm_places<-1, CLAMP>(bias, point[x], g, at);
                        pm_bias(at, scale2, s[x][0]);
                    }
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        uint64_t mix = 0;
#pragma unroll
                        for (int k = 0; k < MAPS; ++k) {
                            const uint64_t v = pack2(s[x][k][2 * r], s[x][k][2 * r + 1]);
                            uint64_t pr = pm_exp2(BIAS ? add2(v, ref[k]) : fma2(v, pm_both(scale2), ref[k]));
                            if (FAR) pr = mul2(pr, coef[k]);
                            else if (k == 1) pr = mul2(pr, pm_both(minus_lam));
                            mix = k == 0 ? pr : add2(mix, pr);
                            const uint64_t ds = mul2(pr, add2(pack2(G[x][0][2 * r], G[x][0][2 * r + 1]), delta[k]));
                            float y, z;
                            unpack2(ds, y, z);
                            p[x][k][2 * n + r] = pack_bf16(y, z);
                            // (rows beyond the patch have no key: their lanes add nothing)
                            if (learns && own.row[x][r] < L) {
                                const int vy = __float2int_rn(y * per_unit), vz = __float2int_rn(z * per_unit);
#pragma unroll
                                for (int c = 0; c < 3; ++c) {
                                    pm_add_shared((at[2 * r][c] >> fewer) + to_hist, vy);
                                    pm_add_shared((at[2 * r + 1][c] >> fewer) + to_hist, vz);
                                }
                            }
                        }
                        float y, z;
                        unpack2(mix, y, z);
                        pm[x][0][2 * n + r] = pack_bf16(y, z);
                    }
                }
            }
            pm_accumulate<W, 1, RT>(pm, os, j0, dv, pm, dv);
            pm_accumulate<W, MAPS, RT>(p, qs, j0, dk, p, dk);
        }
    };
    auto walk = [&](auto clamp) {
        for (int i = 0; i * CH < L; ++i) {
            if (learns && i % (PM_WINDOW / CH) == 0) {
                if (i) {
                    __syncthreads();
                    pa_flush(table, hist, sums, unit, NT);
                }
                unit = pa_unit<NT / 32, PM_WINDOW>(a, table, w.h, w.start, L, i * CH, part);
                per_unit = pa_per_unit(unit);
            }
            const unsigned char* st = in.next(i);
            if (warp0 >= L) continue;
            if (BIAS || marks[i % PM_STAGES] == i + 1) chunk(i, st, clamp, PmYes());
            else chunk(i, st, clamp, PmNo());
        }
    };
    if (BIAS && table.clamps) walk(PmYes());
    else walk(PmNo());
    in.end();
    if (learns) {
        pa_flush(table, hist, sums, unit, NT);
        __syncthreads();
        pa_store_bins(a, table, sums, bins, NT);
    }
#pragma unroll
    for (int x = 0; x < RT; ++x)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (own.row[x][r] >= L) continue;
            const int e = own.e[x][r], slot = a.slot ? a.slot[w.start + own.row[x][r]] : -1;
            if (slot >= 0) {             // this point's other row is some other patch's: added up later
                float2* dst = (float2*)(a.shared + (int64_t)slot * 2 * a.C + w.h * W);
#pragma unroll
                for (int n = 0; n < W / 8; ++n) {
                    dst[4 * n + t] = make_float2(dk[x][n][2 * r] * a.scale, dk[x][n][2 * r + 1] * a.scale);
                    dst[a.C / 2 + 4 * n + t] = make_float2(dv[x][n][2 * r], dv[x][n][2 * r + 1]);
                }
            } else if (e >= 0) {
                uint32_t* dst = (uint32_t*)((__nv_bfloat16*)a.dqkv + e * stride + a.C + w.h * W);
#pragma unroll
                for (int n = 0; n < W / 8; ++n) {
                    dst[4 * n + t] = pack_bf16(dk[x][n][2 * r] * a.scale, dk[x][n][2 * r + 1] * a.scale);
                    dst[a.C / 2 + 4 * n + t] = pack_bf16(dv[x][n][2 * r], dv[x][n][2 * r + 1]);
                }
            }
        }
}

template <int NT, typename K>
static int launch(K kern, const PatchArgs& a, size_t smem, cudaStream_t stream)
{
    const cudaError_t err = allow_smem(kern);
    PTV3_REQUIRE(err == cudaSuccess, PTV3_ERR_CUDA, "ptv3_patch_attention: %s", cudaGetErrorString(err));
    launch_dependent(kern, dim3((unsigned)((int64_t)a.n_seq * a.tiles * a.H)), dim3(NT), smem, stream, a);
    count_launches(1);
    return check_launch("ptv3_patch_attention");
}

// What a block is.  Eight warps of a row tile each; two tiles to a warp, so that what it reads of the other side serves twice the
// rows, where registers allow it, patches fill such blocks and launches are long.  us with one and with two, heads of 16:
// forward with a bias, 120 000 x 64, 489 and 392; 100 000 x 64, rows with a bias 462 and 432, columns 886 and 804, columns of
// two maps 356 and 319; not so forward and rows without a bias (312 and 326, 341 and 465).  Heads of 32, 100 000 x 64: columns with a
// bias, a CTA to an SM, 667 and 543 (10 000 x 64: 108 and 87), of two maps in blocks of four warps, three to an SM, 252 and 233
// (20 000 x 64: 75 and 67; 10 000 x 64 42 and 42); forward and rows are slower or as fast (with a bias 238 and 281, 289 and 300).  Heads
// of 64, a CTA to an SM: forward with a bias 238 and 178 (20 000 x 64: 76 and 58); columns with a bias 410 and 383, of two maps 261 and
// 228, but 202 and 247, 122 and 149 at 40 000 x 64, whose 160 blocks are two rounds: one tile.  Four warps where patches are short
// (60 000 x 64 in patches of 48, two maps, the three passes: 62, 70 and 74 us with eight, 34, 38 and 36) or blocks without a bias
// few (1 560 x 256 forward 33 and 27.5; with a bias, 6 760 x 128, 68 and 72).
struct PmForm {
    int threads, tiles;      // tiles of a warp
    int rows() const { return threads / 2 * tiles; }
};
static PmForm block_form(int64_t n_seq, int64_t longest, int heads, int width, int maps, bool bias, int pass)
{
    auto blocks = [&](int rows) { return n_seq * heads * ((longest + rows - 1) / rows); };
    if (longest <= 64 || (!bias && blocks(128) < 2 * SMS)) return PmForm{128, 1};
    const int least = width == 16 ? 2 * SMS : bias ? SMS / 2 : SMS;
    const bool suits = width == 16   ? bias || (maps == 2 && pass == PA_COLS)
                       : width == 32 ? pass == PA_COLS && (bias || maps == 2)
                                     : pass == PA_FWD && bias;
    const bool two = suits && longest >= 256 && blocks(256) >= least;
    return PmForm{two && width == 32 && !bias ? 128 : 256, two ? 2 : 1};
}
int patch_mma_cols_rows(int64_t n_seq, int64_t longest, int heads, int width)
{
    return block_form(n_seq, longest, heads, width, 1, true, PA_COLS).rows();
}

template <int W, int MAPS, bool BIAS, int RT, int NT>
static int launch_block(const PatchArgs& a, int pass, cudaStream_t stream)
{
    const size_t stages = PM_STAGES * PmStage<W, PmChunk<W, BIAS, NT>::N>::BYTES;
    const size_t smem = stages + (BIAS ? PmTableBytes<NT>::TABLE : 0);
    // (block_form has what takes two tiles)
    constexpr int ROWS2 = BIAS && W == 16 ? RT : 1, FWD2 = BIAS && W != 32 ? RT : 1, COLS2 = W == 64 ? 1 : RT;
    if (pass == PA_ROWS) return launch<NT>(patch_mma_rows_kernel<W, MAPS, BIAS, ROWS2, NT>, a, smem, stream);
    if (pass == PA_COLS)      // the table, its bins, and their sums
        return launch<NT>(patch_mma_cols_kernel<W, MAPS, BIAS, COLS2, NT>, a,
                          stages + (BIAS ? PmTableBytes<NT>::BINS + pm_sums_bytes(a.bnd, PmTableBytes<NT>::BINS) : 0), stream);
    return a.lse ? launch<NT>(patch_mma_fwd_kernel<W, MAPS, BIAS, true, FWD2, NT>, a, smem, stream)
                 : launch<NT>(patch_mma_fwd_kernel<W, MAPS, BIAS, false, FWD2, NT>, a, smem, stream);
}

template <int W, int MAPS, bool BIAS>
static int launch_pass(const PatchArgs& args, int pass, cudaStream_t stream)
{
    PatchArgs a = args;
    const int longest = a.max_seqlen < a.n_pad ? a.max_seqlen : a.n_pad;
    const PmForm form = block_form(a.n_seq, longest, a.H, W, MAPS, BIAS, pass);
    a.tiles = ceil_div(longest, form.rows());
    constexpr int RT = BIAS || (W == 16 && MAPS == 2) ? 2 : 1, RT4 = W == 32 && MAPS == 2 ? 2 : 1;
    if (form.threads == 128)
        return form.tiles == 2 ? launch_block<W, MAPS, BIAS, RT4, 128>(a, pass, stream)
                               : launch_block<W, MAPS, BIAS, 1, 128>(a, pass, stream);
    return form.tiles == 2 ? launch_block<W, MAPS, BIAS, RT, 256>(a, pass, stream)
                           : launch_block<W, MAPS, BIAS, 1, 256>(a, pass, stream);
}

template <int W>
static int launch_form(const PatchArgs& a, int maps, int pass, cudaStream_t stream)
{
    if (maps == 2) return launch_pass<W, 2, false>(a, pass, stream);
    return a.grid ? launch_pass<W, 1, true>(a, pass, stream) : launch_pass<W, 1, false>(a, pass, stream);
}

int launch_patch_mma(const PatchArgs& a, int width, int maps, int pass, cudaStream_t stream)
{
    switch (width) {
        case 16: return launch_form<16>(a, maps, pass, stream);
        case 32: return launch_form<32>(a, maps, pass, stream);
        default: return launch_form<64>(a, maps, pass, stream);
    }
}

}  // namespace ptv3
