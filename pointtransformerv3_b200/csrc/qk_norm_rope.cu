// Norms of queries and keys for each head with their rotation by grid coordinates, forward and backward, in one pass over the rows
// of a QKV projection (values are copied, so that the result is a QKV matrix again).
//
//   y = x r w,  r = rsqrt(mean(x^2) + eps);   (z_2i, z_2i+1) = R(angle_i) (y_2i, y_2i+1)
//   backward:  dy = R(-angle) dz,  dw = sum over rows and heads of dy x r,  dx = r (dy w - x r mean(dy w x r))
//
// Bound by memory: a thread owns 16 bytes of a row, a head's sum of squares is a shuffle over the neighbouring lanes that
// hold it.  The angles of a row serve all its heads and both of q and k, so a block computes them once, into shared
// memory.  An angle is a coordinate times a frequency, up to 65 535 radians and more, of which only the fraction of a turn counts:
// the frequency is held in turns as a 64-bit fraction, the product modulo 2^64 is exact, and its upper half is the
// angle to 2^-32 of a turn (a float product would be off by 65 535 2^-24 = 0.004 radians).
#include <math.h>

#include "common.cuh"
#include "convert.cuh"
#include "vec.cuh"

namespace ptv3 {

constexpr int QK_THREADS = 256;
constexpr int QK_UNROLL = 4;          // vectors of a thread per block of rows
constexpr int QK_MAX_FREQ = 21;       // frequencies of an axis, D = 128

struct QkArgs {
    const void *qkv, *qw, *kw;
    const int32_t* grid;
    const void* dout;
    void* out;
    float* partial;        // blocks x 2 D
    int64_t n;
    int vec_row, vec_c;    // 16-byte vectors of a row, of a third of it
    int rows;              // of a block
    int D, p, w_bf16;
    float eps;
    uint64_t freq[QK_MAX_FREQ];     // in turns, times 2^64
};

// cos and sin of every pair's angle for the rows of a block
__device__ __forceinline__ void qk_angles(const QkArgs& a, int64_t row0, int rows, float2* cs)
{
    const int pairs = 3 * a.p;
    for (int i = threadIdx.x; i < rows * pairs; i += QK_THREADS) {
        const int r = i / pairs, j = i - r * pairs, axis = j / a.p;
        const uint64_t turn = (uint64_t)(int64_t)a.grid[3 * (row0 + r) + axis] * a.freq[j - axis * a.p];
        // signed fraction of a turn, of which sincospif wants twice as many half turns
        const float half = (float)(int32_t)(turn >> 32) * (2.f / 4294967296.f);
        sincospif(half, &cs[i].y, &cs[i].x);
    }
}

template <int N>
__device__ __forceinline__ void qk_rotate(float (&y)[N], const float2* cs, int first, int pairs, float sign)
{
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
        if (first + i < pairs) {
            const float2 t = cs[first + i];
            const float u = y[2 * i], v = y[2 * i + 1], s = t.y * sign;
            y[2 * i] = u * t.x - v * s;
            y[2 * i + 1] = u * s + v * t.x;
        }
}

// sum over the lanes that hold a head
__device__ __forceinline__ float qk_head_sum(float v, int lanes)
{
    for (int d = 1; d < lanes; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

template <typename T, bool NORM, bool BACK>
__global__ void __launch_bounds__(QK_THREADS) qk_norm_rope_kernel(const QkArgs a)
{
    using V = Vec<T>;
    using Raw = typename V::Raw;
    extern __shared__ float2 cs[];
    const int lanes = a.D / V::N;                       // of a head: a power of two that divides a warp
    const int at = threadIdx.x % lanes * V::N;          // this thread's place in a head, always the same one
    const int pairs = a.grid ? 3 * a.p : 0;
    float w[2][V::N], dw[2][V::N];
    if (NORM) {
#pragma unroll
        for (int i = 0; i < V::N; ++i) {
            w[0][i] = a.w_bf16 ? __bfloat162float(((const __nv_bfloat16*)a.qw)[at + i]) : ((const float*)a.qw)[at + i];
            w[1][i] = a.w_bf16 ? __bfloat162float(((const __nv_bfloat16*)a.kw)[at + i]) : ((const float*)a.kw)[at + i];
            dw[0][i] = dw[1][i] = 0.f;
        }
    }
    const Raw* in = (const Raw*)a.qkv;
    const Raw* grad = (const Raw*)a.dout;
    Raw* out = (Raw*)a.out;
    for (int64_t row0 = (int64_t)blockIdx.x * a.rows; row0 < a.n; row0 += (int64_t)gridDim.x * a.rows) {
        const int rows = (int)min((int64_t)a.rows, a.n - row0);
        const int count = rows * a.vec_row;
        const int64_t base = row0 * a.vec_row;
        if (pairs) {
            __syncthreads();
            qk_angles(a, row0, rows, cs);
            __syncthreads();
        }
        for (int first = 0; first < count; first += QK_THREADS * QK_UNROLL) {
            Raw x[QK_UNROLL], gx[QK_UNROLL];
#pragma unroll
            for (int u = 0; u < QK_UNROLL; ++u) {
                const int i = first + u * QK_THREADS + threadIdx.x;
                if (i < count) {
                    if (BACK) gx[u] = grad[base + i];
                    if (!BACK || NORM) x[u] = in[base + i];
                }
            }
#pragma unroll
            for (int u = 0; u < QK_UNROLL; ++u) {
                const int i = first + u * QK_THREADS + threadIdx.x;
                const bool live = i < count;
                const int r = live ? i / a.vec_row : 0, c = i - r * a.vec_row;
                // (all lanes of a head are queries, keys or values together, but lanes of a warp need not be)
                const int part = live ? (c < a.vec_c ? 0 : c < 2 * a.vec_c ? 1 : 2) : 2;
                float y[V::N], g[V::N];
                if (!BACK) {
                    V::unpack(x[u], y);
                    if (NORM) {
                        float s = 0.f;
#pragma unroll
                        for (int k = 0; k < V::N; ++k) s = fmaf(y[k], y[k], s);
                        const float inv = rsqrtf(qk_head_sum(s, lanes) / (float)a.D + a.eps);
#pragma unroll
                        for (int k = 0; k < V::N; ++k) y[k] *= inv * (part == 0 ? w[0][k] : w[1][k]);
                    }
                    qk_rotate(y, cs + r * pairs, at / 2, pairs, 1.f);
                    if (live) out[base + i] = part == 2 ? x[u] : V::pack(y);
                } else {
                    V::unpack(gx[u], g);
                    qk_rotate(g, cs + r * pairs, at / 2, pairs, -1.f);
                    if (NORM) {
                        V::unpack(x[u], y);
                        float s = 0.f, m = 0.f;
#pragma unroll
                        for (int k = 0; k < V::N; ++k) s = fmaf(y[k], y[k], s);
                        const float inv = rsqrtf(qk_head_sum(s, lanes) / (float)a.D + a.eps);
#pragma unroll
                        for (int k = 0; k < V::N; ++k) {
                            y[k] *= inv;
                            if (part == 0) dw[0][k] = fmaf(g[k], y[k], dw[0][k]);
                            if (part == 1) dw[1][k] = fmaf(g[k], y[k], dw[1][k]);
                            g[k] *= part == 0 ? w[0][k] : w[1][k];
                            m = fmaf(g[k], y[k], m);
                        }
                        m = qk_head_sum(m, lanes) / (float)a.D;
#pragma unroll
                        for (int k = 0; k < V::N; ++k) g[k] = inv * (g[k] - y[k] * m);
                    }
                    if (live) out[base + i] = part == 2 ? gx[u] : V::pack(g);
                }
            }
        }
    }
    if (NORM && BACK) {
        // sums of a block: lanes of one place in a head, then the warps, in a fixed order
        __shared__ float sums[QK_THREADS / 32][2 * 128];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int k = 0; k < V::N; ++k) {
                float v = dw[q][k];
                for (int d = lanes; d < 32; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
                if ((threadIdx.x & 31) < lanes) sums[threadIdx.x / 32][q * a.D + at + k] = v;
            }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * a.D; i += QK_THREADS) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < QK_THREADS / 32; ++k) v += sums[k][i];
            a.partial[(int64_t)blockIdx.x * 2 * a.D + i] = v;
        }
    }
}

// weights' gradients: a warp per value adds the blocks' sums
__global__ void __launch_bounds__(QK_THREADS) qk_weights_kernel(const float* partial, int blocks, int D, void* dq, void* dk,
                                                                int bf16)
{
    const int i = (blockIdx.x * QK_THREADS + threadIdx.x) / 32, lane = threadIdx.x & 31;
    if (i >= 2 * D) return;
    float v = 0.f;
    for (int b = lane; b < blocks; b += 32) v += partial[(int64_t)b * 2 * D + i];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (lane) return;
    void* to = i < D ? dq : dk;
    if (bf16) ((__nv_bfloat16*)to)[i % D] = __float2bfloat16_rn(v);
    else ((float*)to)[i % D] = v;
}

constexpr int QK_MAX_BLOCKS = SMS * 8;

// rows of a block, and how many blocks: a block's vectors once through its threads, on long inputs a few times over
static int qk_rows(int vec_row) { return vec_row >= QK_THREADS * QK_UNROLL ? 1 : QK_THREADS * QK_UNROLL / vec_row; }
static int qk_blocks(int64_t n, int vec_row)
{
    const int64_t b = (n + qk_rows(vec_row) - 1) / qk_rows(vec_row);
    return (int)(b < QK_MAX_BLOCKS ? b : QK_MAX_BLOCKS);
}

static int qk_check(const char* what, const void* qkv, const void* qw, const void* kw, int weight_dtype,
                    const int32_t* grid, const void* out, int64_t n, int channels, int heads, double base, int dtype)
{
    PTV3_REQUIRE(n >= 0 && channels >= 1 && heads >= 1 && channels % heads == 0, PTV3_ERR_INVALID_ARGUMENT, "%s: bad sizes",
                 what);
    const int D = channels / heads;
    PTV3_REQUIRE(D == 8 || D == 16 || D == 32 || D == 64 || D == 128, PTV3_ERR_UNSUPPORTED,
                 "%s: head dim %d (supported: 8, 16, 32, 64, 128)", what, D);
    PTV3_REQUIRE((dtype == PTV3_DTYPE_F32 || dtype == PTV3_DTYPE_BF16) &&
                     (weight_dtype == PTV3_DTYPE_F32 || weight_dtype == PTV3_DTYPE_BF16),
                 PTV3_ERR_UNSUPPORTED, "%s: dtypes %d, %d", what, dtype, weight_dtype);
    PTV3_REQUIRE(channels <= 1 << 20, PTV3_ERR_UNSUPPORTED, "%s: %d channels", what, channels);
    PTV3_REQUIRE(!qw == !kw && (qw || grid), PTV3_ERR_INVALID_ARGUMENT,
                 "%s: weights of both queries and keys, coordinates, or all three", what);
    PTV3_REQUIRE(!grid || base > 0, PTV3_ERR_INVALID_ARGUMENT, "%s: base %g", what, base);
    PTV3_REQUIRE(n == 0 || (qkv && out && (((uintptr_t)qkv | (uintptr_t)out) & 15) == 0), PTV3_ERR_INVALID_ARGUMENT,
                 "%s: null or unaligned rows", what);
    return PTV3_OK;
}

static QkArgs qk_args(const void* qkv, const void* qw, const void* kw, int weight_dtype, const int32_t* grid, void* out,
                      int64_t n, int channels, int heads, float eps, double base, int dtype)
{
    QkArgs a = {};
    a.qkv = qkv;
    a.qw = qw;
    a.kw = kw;
    a.grid = grid;
    a.out = out;
    a.n = n;
    a.vec_c = channels * (dtype == PTV3_DTYPE_F32 ? 4 : 2) / 16;
    a.vec_row = 3 * a.vec_c;
    a.rows = qk_rows(a.vec_row);
    a.D = channels / heads;
    a.p = a.D / 6;
    a.w_bf16 = weight_dtype == PTV3_DTYPE_BF16;
    a.eps = eps;
    // 2^64 base^(-k/p) / 2 pi; whole turns of frequencies above one turn a cell fall away
    for (int k = 0; grid && k < a.p; ++k) {
        const double turns = pow(base, -(double)k / a.p) * 0.15915494309189533577;
        a.freq[k] = (uint64_t)((turns - floor(turns)) * 18446744073709551616.0);
    }
    return a;
}

template <typename T, bool BACK>
static int launch_qk(const QkArgs& a, const char* what, cudaStream_t stream)
{
    const int blocks = qk_blocks(a.n, a.vec_row);
    const size_t smem = a.grid ? (size_t)a.rows * 3 * a.p * sizeof(float2) : 0;
    if (a.qw) qk_norm_rope_kernel<T, true, BACK><<<blocks, QK_THREADS, smem, stream>>>(a);
    else qk_norm_rope_kernel<T, false, BACK><<<blocks, QK_THREADS, smem, stream>>>(a);
    count_launches(1);
    return check_launch(what);
}

}  // namespace ptv3

using namespace ptv3;

extern "C" int ptv3_qk_norm_rope_fwd(const void* qkv, const void* q_weight, const void* k_weight, int weight_dtype,
                                     const int32_t* grid_coord, void* out, int64_t n, int channels, int heads, float eps,
                                     double base, int dtype, void* stream)
{
    const char* what = "ptv3_qk_norm_rope_fwd";
    const int rc = qk_check(what, qkv, q_weight, k_weight, weight_dtype, grid_coord, out, n, channels, heads, base, dtype);
    if (rc != PTV3_OK || n == 0) return rc;
    const QkArgs a = qk_args(qkv, q_weight, k_weight, weight_dtype, grid_coord, out, n, channels, heads, eps, base, dtype);
    return dtype == PTV3_DTYPE_F32 ? launch_qk<float, false>(a, what, (cudaStream_t)stream)
                                   : launch_qk<__nv_bfloat16, false>(a, what, (cudaStream_t)stream);
}

extern "C" size_t ptv3_qk_norm_rope_workspace_bytes(int64_t n, int channels, int heads)
{
    if (n <= 0 || channels < 1 || heads < 1) return 0;
    return (size_t)QK_MAX_BLOCKS * 2 * (channels / heads) * sizeof(float);
}

extern "C" int ptv3_qk_norm_rope_bwd(const void* qkv, const void* q_weight, const void* k_weight, int weight_dtype,
                                     const int32_t* grid_coord, const void* dout, void* dqkv, void* dq_weight,
                                     void* dk_weight, int64_t n, int channels, int heads, float eps, double base, int dtype,
                                     void* workspace, size_t workspace_bytes, void* stream)
{
    const char* what = "ptv3_qk_norm_rope_bwd";
    // (without weights the rows themselves are not read)
    int rc = qk_check(what, q_weight ? qkv : dout, q_weight, k_weight, weight_dtype, grid_coord, dqkv, n, channels, heads,
                      base, dtype);
    if (rc != PTV3_OK) return rc;
    PTV3_REQUIRE(n == 0 || (dout && ((uintptr_t)dout & 15) == 0), PTV3_ERR_INVALID_ARGUMENT, "%s: null or unaligned rows",
                 what);
    PTV3_REQUIRE(!q_weight || (dq_weight && dk_weight), PTV3_ERR_INVALID_ARGUMENT, "%s: weights without gradients", what);
    PTV3_REQUIRE(!q_weight || n == 0 ||
                     (workspace && workspace_bytes >= ptv3_qk_norm_rope_workspace_bytes(n, channels, heads)),
                 PTV3_ERR_WORKSPACE, "%s: workspace of %zu bytes", what, workspace_bytes);
    cudaStream_t s = (cudaStream_t)stream;
    QkArgs a = qk_args(qkv, q_weight, k_weight, weight_dtype, grid_coord, dqkv, n, channels, heads, eps, base, dtype);
    a.dout = dout;
    a.partial = (float*)workspace;
    if (n > 0) {
        rc = dtype == PTV3_DTYPE_F32 ? launch_qk<float, true>(a, what, s) : launch_qk<__nv_bfloat16, true>(a, what, s);
        if (rc != PTV3_OK) return rc;
    }
    if (q_weight) {
        qk_weights_kernel<<<ceil_div(2 * a.D * 32, QK_THREADS), QK_THREADS, 0, s>>>(
            a.partial, n > 0 ? qk_blocks(n, a.vec_row) : 0, a.D, dq_weight, dk_weight, a.w_bf16);
        count_launches(1);
    }
    return check_launch(what);
}
