// Patch attention with bias or of two maps, forward and backward, in fp32 arithmetic on CUDA cores (patch_attn.cuh
// has the mathematics): a thread owns a query (or, in the pass over columns, a key), the other side streams through shared
// memory in chunks that all threads read at the same address, gathered by cp.async a chunk ahead.  Heads of 64 are shared by two
// neighbouring threads, so that accumulators stay in registers.
#include <type_traits>

#include "patch_attn.cuh"
#include "mma_util.cuh"

namespace ptv3 {

constexpr int PF_STEP = 8;        // keys whose scores are held at a time
constexpr int PF_PART = 64;       // keys whose share of a result is summed by itself
constexpr int PF_WINDOW = 8;      // queries between two clearings of the bins: the unit is that much finer (gradient of a
                                  // table, patches of 1 024, off by 4e-6 of its norm with 32, 6e-7 with 8)
constexpr int PF_BINS_LOG2 = 4;   // 16 copies of them, so that clearing costs little
constexpr int PF_TABLE_BYTES = 32 * 1024, PF_BINS_BYTES = 48 * 1024;      // for the table; for the table and its bins

constexpr int PF_THREADS = 128;

// SPLIT threads have a row: two of 64 values, one or two of fewer (pf_split).  (Two rows to a thread halve its reads of shared memory
// and leave too few threads: 20 000 x 64 in heads of 16, forward, rows and columns 320, 298 and 400 us instead of 268, 265 and 334.)
template <int W, int MAPS, int SPLIT>
struct PfShape {
    static constexpr int ROWS = PF_THREADS / SPLIT;
    static constexpr int D = W / MAPS;                 // of a map's queries and keys
    static constexpr int DP = D / SPLIT, NP = W / SPLIT / 2;
};

// value i of this thread's share of a row of queries or keys: map-major, of a map every SPLIT-th four values
template <int W, int MAPS, int SPLIT>
__device__ __forceinline__ constexpr int pf_dim(int i, int part)
{
    using S = PfShape<W, MAPS, SPLIT>;
    const int m = i / S::DP, k = i % S::DP;
    return m * S::D + (k / 4 * SPLIT + part) * 4 + k % 4;
}

// Two stages of the other side: x (queries or keys) and y (values or gradients of the result), grid coordinates, and of every
// query and map its reference value, its coefficient over the sum, and delta
template <int W, int MAPS, bool BIAS, bool COLS>
struct PfStages {
    static constexpr int N = W == 16 ? 64 : 32;        // rows of a stage
    float x[2][N][W], y[2][N][W];
    int4 g[2][BIAS ? N : 1];
    float4 aux[2][COLS ? MAPS : 1][COLS ? N : 1];
    float unit[2][COLS && BIAS ? N / PF_WINDOW : 1];
};

// rows [c0, c0 + nk) of a sequence into a stage; matrices arrive behind cp_async_wait
template <int W, int MAPS, bool BIAS, bool COLS>
__device__ __forceinline__ void pf_stage(const PatchArgs& a, PfStages<W, MAPS, BIAS, COLS>& st, int k, const float* x, int64_t xs,
                                         const float* y, int64_t ys, int start, int c0, int L, int h, const float (&coef)[MAPS])
{
    const int nk = min(st.N, L - c0);
    constexpr int C4 = W / 4;
    for (int i = threadIdx.x; i < nk * C4; i += PF_THREADS) {
        const int j = i / C4, d = i % C4 * 4;
        const int e = a.rows[start + c0 + j];
        const int64_t p = e >= 0 ? e : -(e + 1);
        cp_async16(smem_u32(&st.x[k][j][d]), x + p * xs + d);
        cp_async16_zfill(smem_u32(&st.y[k][j][d]), y + p * ys + d, !COLS || e >= 0);
    }
    cp_async_commit();
    if (BIAS)
        for (int j = threadIdx.x; j < nk; j += PF_THREADS) {
            const int e = a.rows[start + c0 + j];
            const int64_t p = e >= 0 ? e : -(e + 1);
            st.g[k][j] = make_int4(pa_coord(a, p, 0), pa_coord(a, p, 1), pa_coord(a, p, 2), 0);
        }
    if (COLS) {
        for (int i = threadIdx.x; i < nk * MAPS; i += PF_THREADS) {
            const int m = i / nk, j = i % nk;
            const int64_t at = (int64_t)(h * MAPS + m) * a.n_pad + start + c0 + j;
            // a row that answers for no point has no gradient: its probabilities are taken as nothing
            const bool own = a.rows[start + c0 + j] >= 0;
            st.aux[k][m][j] = make_float4(own ? a.lse[at] : INFINITY,
                                          own ? a.lse[at + (int64_t)a.H * MAPS * a.n_pad] * coef[m] : 0.f, a.delta[at], 0.f);
        }
        if (BIAS && a.bins && threadIdx.x < st.N) {
            // what the queries of a window can add to a bin at most is 2^31 units, less what rounding may add
            float r = threadIdx.x < nk ? a.reach[(int64_t)h * a.n_pad + start + c0 + threadIdx.x] : 0.f;
#pragma unroll
            for (int d = 1; d < PF_WINDOW; d <<= 1) r += __shfl_xor_sync(0xffffffffu, r, d);
            if (threadIdx.x % PF_WINDOW == 0) st.unit[k][threadIdx.x / PF_WINDOW] = r * (1.f / 2147000000.f);
        }
    }
}

// This thread's look-ups: places in shared memory and clamped reach of its axes, coordinates of its rows along them
template <int SPLIT>
struct PfBias {
    // two threads of a row share the axes, their sums meet in the score's
    static constexpr int AXES = SPLIT == 1 ? 3 : 2;
    int axis[AXES], reach[AXES], base[AXES], g[AXES], log2;
    bool idle;          // the last axis is none: of two threads the second has one axis
    __device__ __forceinline__ void set(const PatchTable& t, int part)
    {
        log2 = t.copies_log2;
        idle = part == 1;
#pragma unroll
        for (int i = 0; i < AXES; ++i) {
            const int c = part ? 2 : i;
            axis[i] = c;
            reach[i] = c == 0 ? t.reach[0] : c == 1 ? t.reach[1] : t.reach[2];
            const int first = c == 0 ? t.first[0] : c == 1 ? t.first[1] : t.first[2];
            base[i] = ((reach[i] + first) << log2) + (threadIdx.x & ((1 << log2) - 1));
        }
    }
    // places for the pair of this thread's row and a row of the other side; s: 1 where the own row is the query, or -1
    __device__ __forceinline__ void places(const int4& other, int s, int (&at)[AXES]) const
    {
#pragma unroll
        for (int i = 0; i < AXES; ++i) {
            const int o = SPLIT == 1 ? (i == 0 ? other.x : i == 1 ? other.y : other.z) : ((const int*)&other)[axis[i]];
            const int d = s * (g[i] - o);
            at[i] = (min(max(d, -reach[i]), reach[i]) << log2) + base[i];
        }
    }
    __device__ __forceinline__ float look(const float* tab, const int (&at)[AXES]) const
    {
        if (AXES == 3) return tab[at[0]] + (tab[at[1]] + tab[at[2]]);
        return tab[at[0]] + (idle ? 0.f : tab[at[1]]);
    }
};

// A thread's share of a row as packed pairs: half the multiply-adds to issue.
template <int SPLIT, int N>
__device__ __forceinline__ void pf_load(uint64_t (&v)[N], const float* row, int part)
{
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const ulonglong2 p = *(const ulonglong2*)(row + (i * SPLIT + part) * 4);
        v[2 * i] = p.x;
        v[2 * i + 1] = p.y;
    }
}
template <int N>
__device__ __forceinline__ float pf_dot(const uint64_t (&x)[N], const uint64_t (&y)[N], int first, int n)
{
    uint64_t v = 0;
#pragma unroll
    for (int i = 0; i < n; ++i) v = fma2(x[first + i], y[first + i], v);
    return hsum2(v);
}
template <int SPLIT>
__device__ __forceinline__ float pf_meet(float v)      // sum over the threads of a row
{
#pragma unroll
    for (int d = 1; d < SPLIT; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// acc[first ..] += f y[first ..] over n pairs
template <int N>
__device__ __forceinline__ void pf_add(uint64_t (&acc)[N], int first, float f, const uint64_t (&y)[N], int n)
{
    const uint64_t f2 = pack2(f, f);
#pragma unroll
    for (int i = 0; i < n; ++i) acc[first + i] = fma2(f2, y[first + i], acc[first + i]);
}
// acc[k] = fix[k] acc[k] + sum of f[j][k] times row j over a step: in a sum of its own first, so that rounding grows with the number of
// steps and not of rows.  (The difference of two maps leaves a fifth of them at lambda = 0.8, and their rounding: by a model of it
// and patches of 1 024, 3.6e-6 of the result's norm without, 1.4e-6 so, and 5e-7 where every 64 keys have a sum as well and
// the softmax's sum keeps what it loses; in heads of 32, 20 000 x 64, 323 us instead of 297.)
template <int SPLIT, int MAPS, int N>
__device__ __forceinline__ void pf_step_add(uint64_t (&acc)[MAPS][N], const float (&fix)[MAPS], const float (&f)[PF_STEP][MAPS],
                                            const float* const (&rows)[PF_STEP], int part)
{
    constexpr int AT = MAPS == 1 ? 4 : 2;          // pairs at a time: registers
#pragma unroll
    for (int c = 0; c < N; c += AT) {
        uint64_t t[MAPS][AT];
#pragma unroll
        for (int j = 0; j < PF_STEP; ++j)
#pragma unroll
            for (int i = 0; i < AT; i += 2) {
                const ulonglong2 y = *(const ulonglong2*)(rows[j] + ((c + i) / 2 * SPLIT + part) * 4);
#pragma unroll
                for (int k = 0; k < MAPS; ++k) {
                    const uint64_t f2 = pack2(f[j][k], f[j][k]);
                    t[k][i] = j ? fma2(f2, y.x, t[k][i]) : mul2(f2, y.x);
                    t[k][i + 1] = j ? fma2(f2, y.y, t[k][i + 1]) : mul2(f2, y.y);
                }
            }
#pragma unroll
        for (int k = 0; k < MAPS; ++k)
#pragma unroll
            for (int i = 0; i < AT; ++i) acc[k][c + i] = fma2(acc[k][c + i], pack2(fix[k], fix[k]), t[k][i]);
    }
}
__device__ __forceinline__ void pf_put(float* to, uint64_t v, float f)
{
    float x, y;
    unpack2(v, x, y);
    *(float2*)to = make_float2(x * f, y * f);
}

// ------------------------------------------------------------------------------------------------- forward
template <int W, int MAPS, bool BIAS, int SPLIT>
__global__ void __launch_bounds__(PF_THREADS) patch_fma_fwd_kernel(const PatchArgs a)
{
    pdl_wait();
    using S = PfShape<W, MAPS, SPLIT>;
    constexpr int NP = S::NP, HP = S::DP / 2;
    __shared__ __align__(16) PfStages<W, MAPS, BIAS, false> st;
    extern __shared__ __align__(16) float tab[];
    const int h = blockIdx.x % a.H, tile = blockIdx.x / a.H % a.tiles, seq = blockIdx.x / a.H / a.tiles;
    const int part = threadIdx.x % SPLIT;
    int start;
    const int L = pa_sequence(a, seq, start);
    const int q0 = tile * S::ROWS, qi = q0 + threadIdx.x / SPLIT;
    if (q0 >= L) return;
    if (h == 0 && a.status) pa_check_owners(a.rows, a.owner, a.status, start + q0, start + min(q0 + S::ROWS, L));
    const bool busy = q0 + threadIdx.x / 32 * 32 / SPLIT < L;          // (warps with no row at all only gather)
    const int64_t stride = 3 * (int64_t)a.C;
    const float* base = (const float*)a.qkv + h * W;
    const float none[MAPS] = {};
    pf_stage(a, st, 0, base + a.C, stride, base + 2 * a.C, stride, start, 0, L, h, none);
    PfBias<SPLIT> bias;
    if (BIAS) {
        const PatchTable table = pa_table(a, seq, PF_TABLE_BYTES, false, false);
        pa_load_table(a, table, h, tab, threadIdx.x, PF_THREADS);
        bias.set(table, part);
    }
    uint64_t q[NP], acc[MAPS][NP];
    uint64_t* total = (uint64_t*)tab + threadIdx.x;       // two maps: what `acc` held up to the last PF_PART keys, times `since`
    float m[MAPS], l[MAPS], lost[MAPS] = {}, since[MAPS];
    const int e = qi < L ? a.rows[start + qi] : -1;
    const int64_t p = e >= 0 ? e : -(e + 1);
    pf_load<SPLIT>(q, base + p * stride, part);
    if (BIAS)
#pragma unroll
        for (int i = 0; i < bias.AXES; ++i) bias.g[i] = pa_coord(a, p, bias.axis[i]);
#pragma unroll
    for (int k = 0; k < MAPS; ++k) {
        m[k] = PA_LOWEST;       // (finite: scores may all be -inf)
        l[k] = 0.f;
        since[k] = 1.f;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            acc[k][i] = 0;
            if (MAPS == 2) total[(k * NP + i) * PF_THREADS] = 0;
        }
    }
    const float scale2 = a.scale * PA_LOG2E;
    for (int c0 = 0, cur = 0; c0 < L; c0 += st.N, cur ^= 1) {
        const int nk = min(st.N, L - c0);
        cp_async_wait<0>();
        __syncthreads();
        if (c0 + st.N < L)
            pf_stage(a, st, cur ^ 1, base + a.C, stride, base + 2 * a.C, stride, start, c0 + st.N, L, h, none);
        if (!busy) continue;
        auto step = [&](int j0, auto whole) {
            constexpr bool full = decltype(whole)::value;
            float s[PF_STEP][MAPS], top[MAPS], sum[MAPS] = {}, fix[MAPS];
#pragma unroll
            for (int k = 0; k < MAPS; ++k) top[k] = m[k];
#pragma unroll
            for (int j = 0; j < PF_STEP; ++j) {
                const int jj = full ? j0 + j : min(j0 + j, nk - 1);
                uint64_t key[NP];
                pf_load<SPLIT>(key, st.x[cur][jj], part);
#pragma unroll
                for (int k = 0; k < MAPS; ++k) {
                    float v = pf_dot(q, key, k * HP, HP);
                    if (BIAS) {
                        int at[bias.AXES];
                        bias.places(st.g[cur][jj], 1, at);
                        v = fmaf(v, scale2, bias.look(tab, at));
                    }
                    s[j][k] = pf_meet<SPLIT>(v);
                    top[k] = fmaxf(top[k], BIAS ? s[j][k] : s[j][k] * scale2);
                }
            }
            const float* rows[PF_STEP];
#pragma unroll
            for (int j = 0; j < PF_STEP; ++j) rows[j] = st.y[cur][full ? j0 + j : min(j0 + j, nk - 1)];
#pragma unroll
            for (int k = 0; k < MAPS; ++k) {
                fix[k] = fast_exp2(m[k] - top[k]);
                m[k] = top[k];
#pragma unroll
                for (int j = 0; j < PF_STEP; ++j) {
                    s[j][k] = fast_exp2(BIAS ? s[j][k] - m[k] : fmaf(s[j][k], scale2, -m[k]));
                    if (!full && j0 + j >= nk) s[j][k] = 0.f;
                    sum[k] += s[j][k];
                }
                const float now = fmaf(l[k], fix[k], sum[k]);
                lost[k] = fmaf(lost[k], fix[k], fmaf(l[k], fix[k], -now) + sum[k]);
                l[k] = now;
                since[k] *= fix[k];
            }
            pf_step_add<SPLIT>(acc, fix, s, rows, part);
        };
        int j0 = 0;
        for (; j0 + PF_STEP <= nk; j0 += PF_STEP) step(j0, std::true_type());
        if (j0 < nk) step(j0, std::false_type());
        if (MAPS == 2 && (c0 + st.N) % PF_PART == 0)
#pragma unroll
            for (int k = 0; k < MAPS; ++k) {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    uint64_t* at = total + (k * NP + i) * PF_THREADS;
                    *at = fma2(*at, pack2(since[k], since[k]), acc[k][i]);
                    acc[k][i] = 0;
                }
                since[k] = 1.f;
            }
    }
    if (MAPS == 2)
#pragma unroll
        for (int k = 0; k < MAPS; ++k)
#pragma unroll
            for (int i = 0; i < NP; ++i) acc[k][i] = fma2(total[(k * NP + i) * PF_THREADS], pack2(since[k], since[k]), acc[k][i]);
#pragma unroll
    for (int k = 0; k < MAPS; ++k) l[k] += lost[k];
    if (e < 0) return;
    const float lam = MAPS == 2 ? pa_param(a.lam, h, a.lam_bf16) : 0.f;
    if (a.lse && part == 0)
#pragma unroll
        for (int k = 0; k < MAPS; ++k) {
            float* to = a.lse + (int64_t)(h * MAPS + k) * a.n_pad + start + qi;
            *to = m[k];
            to[(int64_t)a.H * MAPS * a.n_pad] = 1.f / l[k];
        }
    const float w0 = 1.f / l[0], w2 = 1.f / l[MAPS - 1], w1 = MAPS == 2 ? lam / l[MAPS - 1] : 0.f;
    const int64_t own = (int64_t)e * a.C + h * W;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int d = pf_dim<W, 1, SPLIT>(2 * i, part);
        const uint64_t v = mul2(acc[0][i], pack2(w0, w0));
        pf_put((float*)a.out + own + d, MAPS == 2 ? fma2(acc[MAPS - 1][i], pack2(-w1, -w1), v) : v, 1.f);
        if (MAPS == 2 && a.lse) pf_put((float*)a.second + own + d, acc[MAPS - 1][i], w2);
    }
}

// ------------------------------------------------------------------------- backward, a thread's own queries
// (in fp32 the stored results give delta as close as dQ needs it, and the softmax's sum is kept as such.  What is left, the
// sum of P (G - delta), goes into the delta that the columns read: the same error for all of a row's keys adds up
// in the table's gradient, 2e-6 of its norm with patches of 1 024 without this.)
template <int W, int MAPS, bool BIAS, int SPLIT>
__global__ void __launch_bounds__(PF_THREADS) patch_fma_rows_kernel(const PatchArgs a)
{
    pdl_wait();
    using S = PfShape<W, MAPS, SPLIT>;
    constexpr int NP = S::NP, HP = S::DP / 2;
    __shared__ __align__(16) PfStages<W, MAPS, BIAS, false> st;
    extern __shared__ __align__(16) float tab[];
    const int h = blockIdx.x % a.H, tile = blockIdx.x / a.H % a.tiles, seq = blockIdx.x / a.H / a.tiles;
    const int part = threadIdx.x % SPLIT;
    int start;
    const int L = pa_sequence(a, seq, start);
    const int q0 = tile * S::ROWS, qi = q0 + threadIdx.x / SPLIT;
    if (q0 >= L) return;
    const bool busy = q0 + threadIdx.x / 32 * 32 / SPLIT < L;
    const int64_t stride = 3 * (int64_t)a.C, all = (int64_t)a.H * MAPS * a.n_pad;
    const float* base = (const float*)a.qkv + h * W;
    const float none[MAPS] = {};
    pf_stage(a, st, 0, base + a.C, stride, base + 2 * a.C, stride, start, 0, L, h, none);
    PfBias<SPLIT> bias;
    if (BIAS) {
        const PatchTable table = pa_table(a, seq, PF_TABLE_BYTES, false, false);
        pa_load_table(a, table, h, tab, threadIdx.x, PF_THREADS);
        bias.set(table, part);
    }
    const float lam = MAPS == 2 ? pa_param(a.lam, h, a.lam_bf16) : 0.f;
    uint64_t q[NP], go[NP], dq[NP];
    float ref[MAPS], delta[MAPS], left[MAPS] = {}, total_left[MAPS] = {}, reach = 0.f;
    int e = qi < L ? a.rows[start + qi] : -1;
    const int64_t p = e >= 0 ? e : -(e + 1);
    pf_load<SPLIT>(q, base + p * stride, part);
    float d1 = 0.f, d2 = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) go[i] = dq[i] = 0;
    if (e >= 0) {
        uint64_t o[NP];
        pf_load<SPLIT>(go, (const float*)a.dout + p * a.C + h * W, part);
        pf_load<SPLIT>(o, (const float*)a.out + p * a.C + h * W, part);
        d1 = pf_dot(go, o, 0, NP);
        if (MAPS == 2) {
            pf_load<SPLIT>(o, (const float*)a.second + p * a.C + h * W, part);
            d2 = pf_dot(go, o, 0, NP);
        }
    }
    d1 = pf_meet<SPLIT>(d1);
    if (MAPS == 2) d2 = pf_meet<SPLIT>(d2);
    delta[0] = MAPS == 2 ? fmaf(lam, d2, d1) : d1;
    if (MAPS == 2) delta[MAPS - 1] = d2;
    if (BIAS)
#pragma unroll
        for (int i = 0; i < bias.AXES; ++i) bias.g[i] = pa_coord(a, p, bias.axis[i]);
#pragma unroll
    for (int k = 0; k < MAPS; ++k)
        // a row that answers for no point has no gradient: its probabilities are taken as nothing
        ref[k] = e >= 0 ? a.lse[(int64_t)(h * MAPS + k) * a.n_pad + start + qi] : INFINITY;
    const float scale2 = a.scale * PA_LOG2E;
    for (int c0 = 0, cur = 0; c0 < L; c0 += st.N, cur ^= 1) {
        const int nk = min(st.N, L - c0);
        cp_async_wait<0>();
        __syncthreads();
        if (c0 + st.N < L)
            pf_stage(a, st, cur ^ 1, base + a.C, stride, base + 2 * a.C, stride, start, c0 + st.N, L, h, none);
        if (!busy) continue;
#pragma unroll (MAPS == 2 ? (W == 64 ? 1 : 4) : (W == 16 ? 2 : 1))
        for (int j = 0; j < nk; ++j) {
            uint64_t key[NP], val[NP];
            pf_load<SPLIT>(key, st.x[cur][j], part);
            pf_load<SPLIT>(val, st.y[cur][j], part);
            const float G = pf_meet<SPLIT>(pf_dot(go, val, 0, NP));
#pragma unroll
            for (int k = 0; k < MAPS; ++k) {
                float s = pf_dot(q, key, k * HP, HP);
                if (BIAS) {
                    int at[bias.AXES];
                    bias.places(st.g[cur][j], 1, at);
                    s = fmaf(s, scale2, bias.look(tab, at));
                }
                s = pf_meet<SPLIT>(s);
                const float ds = fast_exp2(BIAS ? s - ref[k] : fmaf(s, scale2, -ref[k])) * (G - delta[k]);
                left[k] += ds;
                if (BIAS) reach += fabsf(ds);
                pf_add(dq, k * HP, ds, key, HP);
            }
        }
        if (MAPS == 2)             // (lambda's gradient is a sum of these: a stage's first)
#pragma unroll
            for (int k = 0; k < MAPS; ++k) {
                total_left[k] += left[k];
                left[k] = 0.f;
            }
    }
    if (qi >= L) return;
    // (read again where registers decide how many CTAs an SM holds: 20 000 x 64 with a bias 358 -> 315 us)
    if (W == 16) e = a.rows[start + qi];
    float by[MAPS];
#pragma unroll
    for (int k = 0; k < MAPS; ++k) {
        left[k] += total_left[k];
        const int64_t at = (int64_t)(h * MAPS + k) * a.n_pad + start + qi;
        by[k] = e >= 0 ? a.lse[at + all] : 0.f;
        if (part == 0) a.delta[at] = fmaf(left[k], by[k], delta[k]);
    }
    if (BIAS && a.reach && part == 0)
        a.reach[(int64_t)h * a.n_pad + start + qi] = (reach + fabsf(left[0])) * by[0];
    if (e < 0) return;
    by[0] *= a.scale;
    if (MAPS == 2) by[MAPS - 1] *= -lam * a.scale;
    float* dst = (float*)a.dqkv + (int64_t)e * stride + h * W;
#pragma unroll
    for (int i = 0; i < NP; ++i) pf_put(dst + pf_dim<W, MAPS, SPLIT>(2 * i, part), dq[i], by[2 * i / S::DP]);
}

// --------------------------------------------------------------------------- backward, a thread's own keys
template <int W, int MAPS, bool BIAS, int SPLIT>
__global__ void __launch_bounds__(PF_THREADS) patch_fma_cols_kernel(const PatchArgs a)
{
    pdl_wait();
    using S = PfShape<W, MAPS, SPLIT>;
    constexpr int NP = S::NP, HP = S::DP / 2;
    __shared__ __align__(16) PfStages<W, MAPS, BIAS, true> st;
    extern __shared__ __align__(16) float tab[];
    const int h = blockIdx.x % a.H, tile = blockIdx.x / a.H % a.tiles, seq = blockIdx.x / a.H / a.tiles;
    const int part = threadIdx.x % SPLIT;
    int start;
    const int L = pa_sequence(a, seq, start);
    const int k0 = tile * S::ROWS, kj = k0 + threadIdx.x / SPLIT;
    const bool learns = BIAS && a.bins;
    float* bins = learns ? pa_bins<S::ROWS>(a, seq, tile, h, start, L, PF_THREADS) : nullptr;
    if (k0 >= L) return;
    const bool busy = k0 + threadIdx.x / 32 * 32 / SPLIT < L;
    const int64_t stride = 3 * (int64_t)a.C;
    const float* base = (const float*)a.qkv + h * W;
    const float* dout = (const float*)a.dout + h * W;
    float coef[MAPS];
    coef[0] = 1.f;
    if (MAPS == 2) coef[MAPS - 1] = -pa_param(a.lam, h, a.lam_bf16);
    pf_stage(a, st, 0, base, stride, dout, a.C, start, 0, L, h, coef);
    PatchTable table = {};
    PfBias<SPLIT> bias;
    if (BIAS) {
        table = pa_table(a, seq, PF_BINS_BYTES, true, false, PF_BINS_LOG2);
        pa_load_table(a, table, h, tab, threadIdx.x, PF_THREADS);
        bias.set(table, part);
    }
    const int fewer = table.copies_log2 - table.bins_log2;      // (0 or 1) copies of the bins than of the table
    int* hist = (int*)tab + (BIAS ? table.entries << table.copies_log2 : 0);
    float* sums = (float*)hist + (BIAS ? table.entries << table.bins_log2 : 0);
    if (learns) {
        for (int i = threadIdx.x; i < table.entries << table.bins_log2; i += PF_THREADS) hist[i] = 0;
        for (int i = threadIdx.x; i < table.entries; i += PF_THREADS) sums[i] = 0.f;
    }
    float unit = 0.f, per_unit = 0.f;
    uint64_t k[NP], v[NP], dk[NP], dv[NP];
    const int e = kj < L ? a.rows[start + kj] : -1;
    const int64_t p = e >= 0 ? e : -(e + 1);
    pf_load<SPLIT>(k, base + p * stride + a.C, part);
    pf_load<SPLIT>(v, base + p * stride + 2 * a.C, part);
#pragma unroll
    for (int i = 0; i < NP; ++i) dk[i] = dv[i] = 0;
    if (BIAS)
#pragma unroll
        for (int i = 0; i < bias.AXES; ++i) bias.g[i] = pa_coord(a, p, bias.axis[i]);
    const float scale2 = a.scale * PA_LOG2E;
    for (int c0 = 0, cur = 0; c0 < L; c0 += st.N, cur ^= 1) {
        const int nq = min(st.N, L - c0);
        cp_async_wait<0>();
        __syncthreads();
        if (c0 + st.N < L) pf_stage(a, st, cur ^ 1, base, stride, dout, a.C, start, c0 + st.N, L, h, coef);
        for (int j0 = 0; j0 < nq; j0 += PF_WINDOW) {
            if (learns) {
                if (c0 + j0) {
                    __syncthreads();
                    pa_flush(table, hist, sums, unit, PF_THREADS);
                    __syncthreads();
                }
                unit = st.unit[cur][j0 / PF_WINDOW];
                per_unit = pa_per_unit(unit);
            }
            if (!busy) continue;
#pragma unroll 4
            for (int j = j0; j < min(j0 + PF_WINDOW, nq); ++j) {
                uint64_t qs[NP], os[NP];
                pf_load<SPLIT>(qs, st.x[cur][j], part);
                pf_load<SPLIT>(os, st.y[cur][j], part);
                const float G = pf_meet<SPLIT>(pf_dot(v, os, 0, NP));
                float mix = 0.f;
#pragma unroll
                for (int m = 0; m < MAPS; ++m) {
                    const float4 x = st.aux[cur][m][j];
                    int at[bias.AXES];
                    float s = pf_dot(k, qs, m * HP, HP);
                    if (BIAS) {
                        bias.places(st.g[cur][j], -1, at);
                        s = fmaf(s, scale2, bias.look(tab, at));
                    }
                    s = pf_meet<SPLIT>(s);
                    const float pr = x.y * fast_exp2(BIAS ? s - x.x : fmaf(s, scale2, -x.x));
                    const float ds = pr * (G - x.z);
                    mix += pr;
                    if (learns && kj < L) {
                        const int add = __float2int_rn(ds * per_unit);
#pragma unroll
                        for (int i = 0; i < bias.AXES; ++i)
                            if (!(bias.idle && i == 1)) atomicAdd(hist + (at[i] >> fewer), add);
                    }
                    pf_add(dk, m * HP, ds, qs, HP);
                }
                pf_add(dv, 0, mix, os, NP);
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
    if (slot < 0 && e < 0) return;
    // where a point's other row is some other patch's, both are added up later
    float* dst = slot >= 0 ? a.shared + (int64_t)slot * 2 * a.C + h * W : (float*)a.dqkv + (int64_t)e * stride + a.C + h * W;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        pf_put(dst + pf_dim<W, MAPS, SPLIT>(2 * i, part), dk[i], a.scale);
        pf_put(dst + a.C + pf_dim<W, 1, SPLIT>(2 * i, part), dv[i], 1.f);
    }
}

// Threads to a row.  Rows of 16 or 32 values get two where a block's rows are not filled by the patch (60 000 x 64 in patches of 48 and
// heads of 32, differential: forward, rows and columns 42, 52 and 56 us, 69, 67 and 93 with one), and where blocks are fewer than half the
// SMs (4 096 x 64, patches of 1 024: 82, 139 and 126 us instead of 123, 147 and 165; 8 192 x 64: 121, 170 and 171, 120, 148 and 164
// with one).  Behind a bias the backward pass has one in the latter case (rows 178 us, 168 so).
static int pf_split(int width, int longest, int64_t rows_and_heads, bool learns)
{
    if (width == 64 || longest <= PF_THREADS / 2) return 2;
    return rows_and_heads * ceil_div(longest, PF_THREADS) <= SMS / 2 && !learns ? 2 : 1;
}

template <int W, int MAPS, bool BIAS, int SPLIT>
static int launch_split(const PatchArgs& args, int longest, int pass, cudaStream_t stream)
{
    PatchArgs a = args;
    // the table; in the pass over columns the table, its bins and their sums
    const size_t entries = BIAS ? 3 * (2 * a.bnd + 1) : 0, full = entries * 32 * 4, both = full + full / 2;
    const size_t table = full < PF_TABLE_BYTES ? full : PF_TABLE_BYTES;
    const size_t cols = (both < PF_BINS_BYTES ? both : PF_BINS_BYTES) + entries * 4;
    const size_t totals = MAPS == 2 ? PF_THREADS * MAPS * PfShape<W, MAPS, SPLIT>::NP * 8 : 0;
    a.tiles = ceil_div(longest, PfShape<W, MAPS, SPLIT>::ROWS);
    const unsigned grid = (unsigned)((int64_t)a.n_seq * a.tiles * a.H);
    auto go = [&](auto kern, size_t smem) {
        const cudaError_t e = smem ? allow_smem(kern) : cudaSuccess;
        return e == cudaSuccess ? launch_dependent(kern, dim3(grid), dim3(PF_THREADS), smem, stream, a) : e;
    };
    const cudaError_t err = pass == PA_FWD    ? go(patch_fma_fwd_kernel<W, MAPS, BIAS, SPLIT>, table + totals)
                            : pass == PA_ROWS ? go(patch_fma_rows_kernel<W, MAPS, BIAS, SPLIT>, table)
                                              : go(patch_fma_cols_kernel<W, MAPS, BIAS, SPLIT>, cols);
    PTV3_REQUIRE(err == cudaSuccess, PTV3_ERR_CUDA, "ptv3_patch_attention: %s", cudaGetErrorString(err));
    count_launches(1);
    return check_launch("ptv3_patch_attention");
}

template <int W, int MAPS, bool BIAS>
static int launch_pass(const PatchArgs& a, int pass, cudaStream_t stream)
{
    const int longest = a.max_seqlen < a.n_pad ? a.max_seqlen : a.n_pad;
    if (pf_split(W, longest, (int64_t)a.n_seq * a.H, BIAS && pass != PA_FWD) == 2)
        return launch_split<W, MAPS, BIAS, 2>(a, longest, pass, stream);
    return launch_split<W, MAPS, BIAS, W == 64 ? 2 : 1>(a, longest, pass, stream);
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

int patch_fma_cols_rows(int64_t longest, int width) { return PF_THREADS / pf_split(width, (int)longest, 0, true); }

}  // namespace ptv3
