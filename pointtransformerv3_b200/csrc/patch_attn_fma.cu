// Patch attention with bias or of two maps, forward and backward, in fp32 arithmetic on CUDA cores (patch_attn.cuh
// has the mathematics): a thread owns a query (or, in the pass over columns, a key), the other side comes through shared memory
// in chunks that all threads read at the same address.  Heads of 64 are shared by two neighbouring threads, so that
// accumulators stay in registers.
#include "patch_attn.cuh"
#include "mma_util.cuh"

namespace ptv3 {

constexpr int PF_THREADS = 128;
constexpr int PF_CHUNK = 64;      // rows of the other side in shared memory
constexpr int PF_STEP = 8;        // of which scores are held at a time
constexpr int PF_WINDOW = 8;      // queries between two clearings of the bins: the unit is that much finer (gradient of a
                                  // table, patches of 1 024, off by 4e-6 of its norm with 32, 6e-7 with 8)
constexpr int PF_BINS_LOG2 = 4;   // 16 copies of them, so that clearing costs little
constexpr int PF_TABLE_BYTES = 32 * 1024, PF_BINS_BYTES = 48 * 1024;      // for the table; for the table and its bins

template <int W, int MAPS>
struct PfShape {
    static constexpr int SPLIT = W == 64 ? 2 : 1;      // threads to a row
    static constexpr int ROWS = PF_THREADS / SPLIT;
    static constexpr int D = W / MAPS;                 // of a map's queries and keys
    static constexpr int DP = D / SPLIT, WP = W / SPLIT;
};

// value i of this thread's share of a row of queries or keys: map-major, the share of a map contiguous
template <int W, int MAPS>
__device__ __forceinline__ constexpr int pf_dim(int i, int part)
{
    using S = PfShape<W, MAPS>;
    return (i / S::DP) * S::D + part * S::DP + i % S::DP;
}

// A chunk of rows in shared memory: x (queries or keys) and y (values or gradients of the result), grid coordinates
template <int W>
__device__ __forceinline__ void pf_stage(const PatchArgs& a, const float* x, int64_t x_stride, const float* y, int64_t y_stride,
                                         bool owners, int start, int nk, float (*xs)[W], float (*ys)[W], int (*gs)[4])
{
    for (int i = threadIdx.x; i < nk * W; i += PF_THREADS) {
        const int j = i / W, d = i % W;
        const int e = a.rows[start + j];
        const int64_t p = e >= 0 ? e : -(e + 1);
        xs[j][d] = (x[p * x_stride + d]);
        ys[j][d] = owners && e < 0 ? 0.f : (y[p * y_stride + d]);
    }
    if (gs)
        for (int i = threadIdx.x; i < nk * 3; i += PF_THREADS) {
            const int j = i / 3, e = a.rows[start + j];
            gs[j][i % 3] = pa_coord(a, e >= 0 ? e : -(e + 1), i % 3);
        }
}

// places of the three look-ups of a pair (d: coordinates of the query minus those of the key)
__device__ __forceinline__ void pf_places(const PatchTable& t, int dx, int dy, int dz, int copy, int (&at)[3])
{
    const int d[3] = {dx, dy, dz};
#pragma unroll
    for (int c = 0; c < 3; ++c)
        at[c] = ((min(max(d[c], -t.reach[c]), t.reach[c]) + t.reach[c] + t.first[c]) << t.copies_log2) + copy;
}

// A thread's share of a row as packed pairs: half the multiply-adds to issue (20 011 x 64, differential, fp32: forward 127 us with
// single ones, rows 133, columns 205; 111, 112 and 169 so).
template <int N>
__device__ __forceinline__ uint64_t pf_sum(const uint64_t (&x)[N], int first, const float* y, int n)
{
    uint64_t v = 0;
    const ulonglong2* y2 = (const ulonglong2*)y;
#pragma unroll
    for (int i = 0; i < n / 4; ++i) {
        const ulonglong2 p = y2[i];
        v = fma2(x[first + 2 * i], p.x, fma2(x[first + 2 * i + 1], p.y, v));
    }
    return v;
}
template <int W, int MAPS>
__device__ __forceinline__ void pf_scores(const uint64_t (&q)[PfShape<W, MAPS>::WP / 2], const float* k, int part,
                                          float (&s)[MAPS])
{
    using S = PfShape<W, MAPS>;
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
        float v = hsum2(pf_sum(q, m * S::DP / 2, k + m * S::D + part * S::DP, S::DP));
        if (S::SPLIT == 2) v += __shfl_xor_sync(0xffffffffu, v, 1);
        s[m] = v;
    }
}
template <int W, int MAPS>
__device__ __forceinline__ float pf_dot(const uint64_t (&x)[PfShape<W, MAPS>::WP / 2], const float* y, int part)
{
    using S = PfShape<W, MAPS>;
    float v = hsum2(pf_sum(x, 0, y + part * S::WP, S::WP));
    if (S::SPLIT == 2) v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v;
}
// acc[first ..] += f y over n values
template <int N>
__device__ __forceinline__ void pf_add(uint64_t (&acc)[N], int first, float f, const float* y, int n)
{
    const uint64_t f2 = pack2(f, f);
    const ulonglong2* y2 = (const ulonglong2*)y;
#pragma unroll
    for (int i = 0; i < n / 4; ++i) {
        const ulonglong2 p = y2[i];
        acc[first + 2 * i] = fma2(f2, p.x, acc[first + 2 * i]);
        acc[first + 2 * i + 1] = fma2(f2, p.y, acc[first + 2 * i + 1]);
    }
}
// pair i of a share of a row of queries or keys, and that of a contiguous share
template <int W, int MAPS>
__device__ __forceinline__ uint64_t pf_pair(const float* row, int i, int part)
{
    const float2 v = *(const float2*)(row + pf_dim<W, MAPS>(2 * i, part));
    return pack2(v.x, v.y);
}
__device__ __forceinline__ uint64_t pf_pair(const float* share, int i)
{
    const float2 v = ((const float2*)share)[i];
    return pack2(v.x, v.y);
}
__device__ __forceinline__ void pf_put(float* to, uint64_t v, float f)
{
    float x, y;
    unpack2(v, x, y);
    *(float2*)to = make_float2(x * f, y * f);
}

// ------------------------------------------------------------------------------------------------- forward
template <int W, int MAPS, bool BIAS>
__global__ void __launch_bounds__(PF_THREADS) patch_fma_fwd_kernel(const PatchArgs a)
{
    pdl_wait();
    using S = PfShape<W, MAPS>;
    __shared__ __align__(16) float Ks[PF_CHUNK][W], Vs[PF_CHUNK][W];
    __shared__ int Gs[BIAS ? PF_CHUNK : 1][4];
    extern __shared__ float tab[];
    const int h = blockIdx.x % a.H, tile = blockIdx.x / a.H % a.tiles, seq = blockIdx.x / a.H / a.tiles;
    const int part = threadIdx.x % S::SPLIT;
    int start;
    const int L = pa_sequence(a, seq, start);
    const int q0 = tile * S::ROWS, qi = q0 + threadIdx.x / S::SPLIT;
    if (q0 >= L) return;
    PatchTable table = {};
    if (BIAS) {
        table = pa_table(a, seq, PF_TABLE_BYTES, false, false);
        pa_load_table(a, table, h, tab, threadIdx.x, PF_THREADS);
    }
    const int copy = threadIdx.x & ((1 << table.copies_log2) - 1);
    const int e = qi < L ? a.rows[start + qi] : -1;
    const int64_t p = e >= 0 ? e : -(e + 1), stride = 3 * (int64_t)a.C;
    const float* base = (const float*)a.qkv + h * W;
    constexpr int NP = S::WP / 2;
    uint64_t q[NP], acc[MAPS][NP];
    float m[MAPS], l[MAPS];
    int g[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < NP; ++i) q[i] = pf_pair<W, MAPS>(base + p * stride, i, part);
    if (BIAS)
        for (int c = 0; c < 3; ++c) g[c] = pa_coord(a, p, c);
#pragma unroll
    for (int k = 0; k < MAPS; ++k) {
        m[k] = -1e30f;          // (finite: scores may all be -inf)
        l[k] = 0.f;
#pragma unroll
        for (int i = 0; i < NP; ++i) acc[k][i] = 0;
    }
    const float scale2 = a.scale * PA_LOG2E;
    for (int c0 = 0; c0 < L; c0 += PF_CHUNK) {
        const int nk = min(PF_CHUNK, L - c0);
        __syncthreads();
        pf_stage<W>(a, base + a.C, stride, base + 2 * a.C, stride, false, start + c0, nk, Ks, Vs, BIAS ? Gs : nullptr);
        __syncthreads();
        for (int j0 = 0; j0 < nk; j0 += PF_STEP) {
            float s[PF_STEP][MAPS], top[MAPS];
#pragma unroll
            for (int k = 0; k < MAPS; ++k) top[k] = m[k];
#pragma unroll
            for (int j = 0; j < PF_STEP; ++j) {
                const int jj = min(j0 + j, nk - 1);
                pf_scores<W, MAPS>(q, Ks[jj], part, s[j]);
                if (BIAS) {
                    int at[3];
                    pf_places(table, g[0] - Gs[jj][0], g[1] - Gs[jj][1], g[2] - Gs[jj][2], copy, at);
                    s[j][0] = fmaf(s[j][0], scale2, tab[at[0]]) + (tab[at[1]] + tab[at[2]]);
                }
#pragma unroll
                for (int k = 0; k < MAPS; ++k) {
                    if (j0 + j >= nk) s[j][k] = BIAS || scale2 > 0.f ? -INFINITY : INFINITY;
                    top[k] = fmaxf(top[k], BIAS ? s[j][k] : s[j][k] * scale2);
                }
            }
#pragma unroll
            for (int k = 0; k < MAPS; ++k) {
                const float fix = fast_exp2(m[k] - top[k]);
                m[k] = top[k];
                l[k] *= fix;
#pragma unroll
                for (int i = 0; i < NP; ++i) acc[k][i] = mul2(acc[k][i], pack2(fix, fix));
            }
            float sum[MAPS] = {};      // of a step's, so that rounding does not grow with every key
#pragma unroll
            for (int j = 0; j < PF_STEP; ++j) {
                const int jj = min(j0 + j, nk - 1);
#pragma unroll
                for (int k = 0; k < MAPS; ++k) {
                    const float pr = fast_exp2(BIAS ? s[j][k] - m[k] : fmaf(s[j][k], scale2, -m[k]));
                    sum[k] += pr;
                    pf_add(acc[k], 0, pr, &Vs[jj][part * S::WP], S::WP);
                }
            }
#pragma unroll
            for (int k = 0; k < MAPS; ++k) l[k] += sum[k];
        }
    }
    if (e < 0) return;
    if (a.lse && part == 0)
#pragma unroll
        for (int k = 0; k < MAPS; ++k) {
            float* to = a.lse + (int64_t)(h * MAPS + k) * a.n_pad + start + qi;
            *to = m[k];
            to[(int64_t)a.H * MAPS * a.n_pad] = 1.f / l[k];
        }
    const float lam = MAPS == 2 ? pa_param(a.lam, h, a.lam_bf16) : 0.f;
    const float w0 = 1.f / l[0], w1 = MAPS == 2 ? lam / l[MAPS - 1] : 0.f;
    float* op = (float*)a.out + p * a.C + h * W + part * S::WP;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const uint64_t v = mul2(acc[0][i], pack2(w0, w0));
        pf_put(op + 2 * i, MAPS == 2 ? fma2(acc[MAPS - 1][i], pack2(-w1, -w1), v) : v, 1.f);
    }
    if (MAPS == 2 && a.lse) {
        const float w2 = 1.f / l[MAPS - 1];
        float* o2 = (float*)a.second + p * a.C + h * W + part * S::WP;
#pragma unroll
        for (int i = 0; i < NP; ++i) pf_put(o2 + 2 * i, acc[MAPS - 1][i], w2);
    }
}

// ------------------------------------------------------------------------- backward, a thread's own query
// (in fp32 the stored results give delta as close as dQ needs it, and the softmax's sum is kept as such.  What is left, the
// sum of P (G - delta), goes into the delta that the columns read: the same error for all of a row's keys adds up
// in the table's gradient, 2e-6 of its norm with patches of 1 024 without this.)
template <int W, int MAPS, bool BIAS>
__global__ void __launch_bounds__(PF_THREADS) patch_fma_rows_kernel(const PatchArgs a)
{
    pdl_wait();
    using S = PfShape<W, MAPS>;
    __shared__ __align__(16) float Ks[PF_CHUNK][W], Vs[PF_CHUNK][W];
    __shared__ int Gs[BIAS ? PF_CHUNK : 1][4];
    extern __shared__ float tab[];
    const int h = blockIdx.x % a.H, tile = blockIdx.x / a.H % a.tiles, seq = blockIdx.x / a.H / a.tiles;
    const int part = threadIdx.x % S::SPLIT;
    int start;
    const int L = pa_sequence(a, seq, start);
    const int q0 = tile * S::ROWS, qi = q0 + threadIdx.x / S::SPLIT;
    if (q0 >= L) return;
    PatchTable table = {};
    if (BIAS) {
        table = pa_table(a, seq, PF_TABLE_BYTES, false, false);
        pa_load_table(a, table, h, tab, threadIdx.x, PF_THREADS);
    }
    const int copy = threadIdx.x & ((1 << table.copies_log2) - 1);
    const int e = qi < L ? a.rows[start + qi] : -1;
    const int64_t p = e >= 0 ? e : -(e + 1), stride = 3 * (int64_t)a.C, all = (int64_t)a.H * MAPS * a.n_pad;
    const float* base = (const float*)a.qkv + h * W;
    const int64_t own = p * a.C + h * W + part * S::WP;        // this thread's share of a row of C
    constexpr int NP = S::WP / 2;
    uint64_t q[NP], go[NP], dq[NP], sum1 = 0, sum2 = 0;
    float ref[MAPS], by[MAPS], delta[MAPS], left[MAPS] = {}, reach = 0.f;
    int g[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        q[i] = pf_pair<W, MAPS>(base + p * stride, i, part);
        go[i] = e >= 0 ? pf_pair((const float*)a.dout + own, i) : 0;
        sum1 = fma2(go[i], e >= 0 ? pf_pair((const float*)a.out + own, i) : 0, sum1);
        if (MAPS == 2) sum2 = fma2(go[i], e >= 0 ? pf_pair((const float*)a.second + own, i) : 0, sum2);
        dq[i] = 0;
    }
    float d1 = hsum2(sum1), d2 = hsum2(sum2);
    if (S::SPLIT == 2) {
        d1 += __shfl_xor_sync(0xffffffffu, d1, 1);
        d2 += __shfl_xor_sync(0xffffffffu, d2, 1);
    }
    if (BIAS)
        for (int c = 0; c < 3; ++c) g[c] = pa_coord(a, p, c);
    const float lam = MAPS == 2 ? pa_param(a.lam, h, a.lam_bf16) : 0.f;
    delta[0] = MAPS == 2 ? fmaf(lam, d2, d1) : d1;
    if (MAPS == 2) delta[MAPS - 1] = d2;
#pragma unroll
    for (int k = 0; k < MAPS; ++k) {
        const int64_t at = (int64_t)(h * MAPS + k) * a.n_pad + start + qi;
        // a row that answers for no point has no gradient: its probabilities are taken as nothing
        ref[k] = e >= 0 ? a.lse[at] : INFINITY;
        by[k] = e >= 0 ? a.lse[at + all] : 0.f;
    }
    const float scale2 = a.scale * PA_LOG2E;
    for (int c0 = 0; c0 < L; c0 += PF_CHUNK) {
        const int nk = min(PF_CHUNK, L - c0);
        __syncthreads();
        pf_stage<W>(a, base + a.C, stride, base + 2 * a.C, stride, false, start + c0, nk, Ks, Vs, BIAS ? Gs : nullptr);
        __syncthreads();
#pragma unroll 4
        for (int j = 0; j < nk; ++j) {
            float s[MAPS];
            pf_scores<W, MAPS>(q, Ks[j], part, s);
            if (BIAS) {
                int at[3];
                pf_places(table, g[0] - Gs[j][0], g[1] - Gs[j][1], g[2] - Gs[j][2], copy, at);
                s[0] = fmaf(s[0], scale2, tab[at[0]]) + (tab[at[1]] + tab[at[2]]);
            }
            const float G = pf_dot<W, MAPS>(go, Vs[j], part);
#pragma unroll
            for (int k = 0; k < MAPS; ++k) {
                const float ds = fast_exp2(BIAS ? s[k] - ref[k] : fmaf(s[k], scale2, -ref[k])) * (G - delta[k]);
                left[k] += ds;
                if (BIAS) reach += fabsf(ds);
                pf_add(dq, k * S::DP / 2, ds, &Ks[j][k * S::D + part * S::DP], S::DP);
            }
        }
    }
    if (qi < L && part == 0) {
#pragma unroll
        for (int k = 0; k < MAPS; ++k)
            a.delta[(int64_t)(h * MAPS + k) * a.n_pad + start + qi] = fmaf(left[k], by[k], delta[k]);
        if (BIAS && a.reach) a.reach[(int64_t)h * a.n_pad + start + qi] = (reach + fabsf(left[0])) * by[0];
    }
    if (e < 0) return;
    by[0] *= a.scale;
    if (MAPS == 2) by[MAPS - 1] *= -lam * a.scale;
    float* dst = (float*)a.dqkv + p * stride + h * W;
#pragma unroll
    for (int i = 0; i < NP; ++i) pf_put(dst + pf_dim<W, MAPS>(2 * i, part), dq[i], by[2 * i / S::DP]);
}

// --------------------------------------------------------------------------- backward, a thread's own key
template <int W, int MAPS, bool BIAS>
__global__ void __launch_bounds__(PF_THREADS) patch_fma_cols_kernel(const PatchArgs a)
{
    pdl_wait();
    using S = PfShape<W, MAPS>;
    __shared__ __align__(16) float Qs[PF_CHUNK][W], Os[PF_CHUNK][W];
    __shared__ int Gs[BIAS ? PF_CHUNK : 1][4];
    // reference value, (-lam) / sum and delta of every query
    __shared__ float Ms[MAPS][PF_CHUNK], Is[MAPS][PF_CHUNK], Ds[MAPS][PF_CHUNK], units[PF_CHUNK / PF_WINDOW];
    extern __shared__ float tab[];
    const int h = blockIdx.x % a.H, tile = blockIdx.x / a.H % a.tiles, seq = blockIdx.x / a.H / a.tiles;
    const int part = threadIdx.x % S::SPLIT;
    int start;
    const int L = pa_sequence(a, seq, start);
    const int k0 = tile * S::ROWS, kj = k0 + threadIdx.x / S::SPLIT;
    const bool learns = BIAS && a.bins;
    float* bins = learns ? a.bins + ((int64_t)(seq * a.tiles + tile) * a.H + h) * 3 * (2 * a.bnd + 1) : nullptr;
    if (k0 >= L) {
        if (learns)
            for (int i = threadIdx.x; i < 3 * (2 * a.bnd + 1); i += PF_THREADS) bins[i] = 0.f;
        return;
    }
    PatchTable table = {};
    if (BIAS) {
        table = pa_table(a, seq, PF_BINS_BYTES, true, false, PF_BINS_LOG2);
        pa_load_table(a, table, h, tab, threadIdx.x, PF_THREADS);
    }
    const int copy = threadIdx.x & ((1 << table.copies_log2) - 1);
    const int fewer = table.copies_log2 - table.bins_log2;      // (0 or 1) copies of the bins than of the table
    int* hist = (int*)tab + (BIAS ? table.entries << table.copies_log2 : 0);
    float* sums = (float*)hist + (BIAS ? table.entries << table.bins_log2 : 0);
    if (learns) {
        for (int i = threadIdx.x; i < table.entries << table.bins_log2; i += PF_THREADS) hist[i] = 0;
        for (int i = threadIdx.x; i < table.entries; i += PF_THREADS) sums[i] = 0.f;
    }
    float unit = 0.f, per_unit = 0.f;
    const int e = kj < L ? a.rows[start + kj] : -1;
    const int64_t p = e >= 0 ? e : -(e + 1), stride = 3 * (int64_t)a.C;
    const float* base = (const float*)a.qkv + h * W;
    constexpr int NP = S::WP / 2;
    uint64_t k[NP], v[NP], dk[NP], dv[NP];
    float coef[MAPS];
    int g[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        k[i] = pf_pair<W, MAPS>(base + p * stride + a.C, i, part);
        v[i] = pf_pair(base + p * stride + 2 * a.C + part * S::WP, i);
        dk[i] = dv[i] = 0;
    }
    if (BIAS)
        for (int c = 0; c < 3; ++c) g[c] = pa_coord(a, p, c);
    coef[0] = 1.f;
    if (MAPS == 2) coef[MAPS - 1] = -pa_param(a.lam, h, a.lam_bf16);
    const float scale2 = a.scale * PA_LOG2E;
    for (int c0 = 0; c0 < L; c0 += PF_CHUNK) {
        const int nq = min(PF_CHUNK, L - c0);
        __syncthreads();
        pf_stage<W>(a, base, stride, (const float*)a.dout + h * W, a.C, true, start + c0, nq, Qs, Os, BIAS ? Gs : nullptr);
        for (int i = threadIdx.x; i < nq * MAPS; i += PF_THREADS) {
            const int m = i / nq, j = i % nq;
            const int64_t at = (int64_t)(h * MAPS + m) * a.n_pad + start + c0 + j;
            const bool own = a.rows[start + c0 + j] >= 0;
            Ms[m][j] = own ? a.lse[at] : INFINITY;
            Is[m][j] = own ? a.lse[at + (int64_t)a.H * MAPS * a.n_pad] * coef[m] : 0.f;
            Ds[m][j] = a.delta[at];
        }
        if (learns && threadIdx.x < PF_CHUNK) {
            // what the queries of a window can add to a bin at most is 2^31 units, less what rounding may add
            float r = threadIdx.x < nq ? a.reach[(int64_t)h * a.n_pad + start + c0 + threadIdx.x] : 0.f;
#pragma unroll
            for (int d = 1; d < PF_WINDOW; d <<= 1) r += __shfl_xor_sync(0xffffffffu, r, d);
            if (threadIdx.x % PF_WINDOW == 0) units[threadIdx.x / PF_WINDOW] = r * (1.f / 2147000000.f);
        }
        __syncthreads();
        for (int j0 = 0; j0 < nq; j0 += PF_WINDOW) {
            if (learns) {
                if (c0 + j0) {
                    __syncthreads();
                    pa_flush(table, hist, sums, unit, PF_THREADS);
                    __syncthreads();
                }
                unit = units[j0 / PF_WINDOW];
                per_unit = pa_per_unit(unit);
            }
#pragma unroll 4
            for (int j = j0; j < min(j0 + PF_WINDOW, nq); ++j) {
                float s[MAPS];
                int at[3];
                pf_scores<W, MAPS>(k, Qs[j], part, s);
                if (BIAS) {
                    pf_places(table, Gs[j][0] - g[0], Gs[j][1] - g[1], Gs[j][2] - g[2], copy, at);
                    s[0] = fmaf(s[0], scale2, tab[at[0]]) + (tab[at[1]] + tab[at[2]]);
                }
                const float G = pf_dot<W, MAPS>(v, Os[j], part);
                float mix = 0.f;
#pragma unroll
                for (int m = 0; m < MAPS; ++m) {
                    const float pr = Is[m][j] * fast_exp2(BIAS ? s[m] - Ms[m][j] : fmaf(s[m], scale2, -Ms[m][j]));
                    const float ds = pr * (G - Ds[m][j]);
                    mix += pr;
                    if (learns && part == 0 && kj < L) {
                        const int v = __float2int_rn(ds * per_unit);
#pragma unroll
                        for (int c = 0; c < 3; ++c) atomicAdd(hist + (at[c] >> fewer), v);
                    }
                    pf_add(dk, m * S::DP / 2, ds, &Qs[j][m * S::D + part * S::DP], S::DP);
                }
                pf_add(dv, 0, mix, &Os[j][part * S::WP], S::WP);
            }
        }
    }
    if (learns) {
        __syncthreads();
        pa_flush(table, hist, sums, unit, PF_THREADS);
        __syncthreads();
        pa_store_bins(a, table, sums, bins, PF_THREADS);
    }
    if (kj >= L) return;
    const int slot = a.slot ? a.slot[start + kj] : -1;
    if (slot >= 0) {             // this point's other row is some other patch's: added up later
        float* dst = a.shared + (int64_t)slot * 2 * a.C + h * W;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            pf_put(dst + pf_dim<W, MAPS>(2 * i, part), dk[i], a.scale);
            pf_put(dst + a.C + part * S::WP + 2 * i, dv[i], 1.f);
        }
    } else if (e >= 0) {
        float* dst = (float*)a.dqkv + p * stride + a.C + h * W;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            pf_put(dst + pf_dim<W, MAPS>(2 * i, part), dk[i], a.scale);
            pf_put(dst + a.C + part * S::WP + 2 * i, dv[i], 1.f);
        }
    }
}

template <int W, int MAPS, bool BIAS>
static int launch_pass(const PatchArgs& args, int pass, cudaStream_t stream)
{
    PatchArgs a = args;
    // the table; in the pass over columns the table, its bins and their sums
    const size_t entries = BIAS ? 3 * (2 * a.bnd + 1) : 0, full = entries * 32 * 4, both = full + full / 2;
    const size_t table = full < PF_TABLE_BYTES ? full : PF_TABLE_BYTES;
    const size_t cols = (both < PF_BINS_BYTES ? both : PF_BINS_BYTES) + entries * 4;
    a.tiles = ceil_div(a.max_seqlen < a.n_pad ? a.max_seqlen : a.n_pad, PfShape<W, MAPS>::ROWS);
    const unsigned grid = (unsigned)((int64_t)a.n_seq * a.tiles * a.H);
    auto go = [&](auto kern, size_t smem) {
        const cudaError_t e = BIAS ? allow_smem(kern) : cudaSuccess;
        return e == cudaSuccess ? launch_dependent(kern, dim3(grid), dim3(PF_THREADS), smem, stream, a) : e;
    };
    const cudaError_t err = pass == PA_FWD    ? go(patch_fma_fwd_kernel<W, MAPS, BIAS>, table)
                            : pass == PA_ROWS ? go(patch_fma_rows_kernel<W, MAPS, BIAS>, table)
                                              : go(patch_fma_cols_kernel<W, MAPS, BIAS>, cols);
    PTV3_REQUIRE(err == cudaSuccess, PTV3_ERR_CUDA, "ptv3_patch_attention: %s", cudaGetErrorString(err));
    count_launches(1);
    return check_launch("ptv3_patch_attention");
}

template <int W>
static int launch_form(const PatchArgs& a, int maps, int pass, cudaStream_t stream)
{
    if (maps == 2) return launch_pass<W, 2, false>(a, pass, stream);
    return a.grid ? launch_pass<W, 1, true>(a, pass, stream) : launch_pass<W, 1, false>(a, pass, stream);
}

int launch_patch_fma(const PatchArgs& a, int width, int maps, int pass, cudaStream_t stream)
{
    switch (width) {
        case 16: return launch_form<16>(a, maps, pass, stream);
        case 32: return launch_form<32>(a, maps, pass, stream);
        default: return launch_form<64>(a, maps, pass, stream);
    }
}

int patch_fma_rows(int width) { return width == 64 ? PF_THREADS / 2 : PF_THREADS; }

int patch_fma_cols_rows(int width) { return width == 64 ? PF_THREADS / 2 : PF_THREADS; }

}  // namespace ptv3
