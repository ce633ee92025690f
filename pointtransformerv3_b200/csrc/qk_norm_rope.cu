// Norms of queries and keys for each head with their rotation by grid coordinates, forward and backward, in one pass over the rows
// of a QKV projection (values are copied, so that the result is a QKV matrix again).
//
//   y = x r w,  r = rsqrt(mean(x^2) + eps);   (z_2i, z_2i+1) = R(angle_i) (y_2i, y_2i+1)
//   backward:  dy = R(-angle) dz,  dw = sum over rows and heads of dy x r,  dx = r (dy w - x r mean(dy w x r))
//
// Bound by memory and, in 16 bits, as much by instructions: a thread keeps one 16-byte column of the rows that it visits,
// so that its head's place, its weights and its part (query, key, value) are settled once, and works on packed pairs of floats; a head's sum of
// squares is a shuffle over the neighbouring lanes that hold it.  The angles of a row serve all its heads and both of q and k, so a block
// computes them once, into shared memory.  An angle is a coordinate times a frequency, up to 65 535 radians and more, of which
// only the fraction of a turn counts: the frequency is held in turns as a 64-bit fraction, the product modulo 2^64 is exact,
// and its upper half is the angle to 2^-32 of a turn (a float product would be off by 65 535 2^-24 = 0.004 radians).
// 407 678 x 64 forward, bf16: 81 us with threads that walked vectors of a row in order (176 instructions a vector), 59
// here; 105 505 x 128 backward 96 (318), 64 here.
#include <math.h>

#include "common.cuh"
#include "convert.cuh"
#include "vec.cuh"

namespace ptv3 {

constexpr int QK_THREADS = 384;       // a multiple of the vectors of most rows (3 channels / 8 or / 4)
constexpr int QK_PASSES = 4;          // rows of a thread per round
constexpr int QK_MAX_FREQ = 21;       // frequencies of an axis, D = 128

// floor(i / d) for i d < 2^32 as a product
struct QkDiv {
    uint32_t d, m;
    __host__ QkDiv(uint32_t d = 1) : d(d), m(d == 1 ? 0 : (uint32_t)((0xffffffffull + d) / d)) {}
    __device__ int operator()(int i) const { return d == 1 ? i : (int)__umulhi((uint32_t)i, m); }
};

struct QkArgs {
    const void *qkv, *qw, *kw;
    const int32_t* grid;
    const void* dout;
    void* out;
    float* partial;        // (blocks, 2 D)
    int64_t n;
    int vec_row, vec_c;    // 16-byte vectors of a row, of a third of it
    int columns, rows;     // of a block at a time: vectors, rows
    int D, p, w_bf16;
    float eps;
    QkDiv by_pairs, by_p;
    uint64_t freq[QK_MAX_FREQ];     // in turns, times 2^64
};

// cos and sin of every pair's angle for `rows` rows
__device__ __forceinline__ void qk_angles(const QkArgs& a, int64_t row0, int rows, float2* cs)
{
    const int pairs = 3 * a.p;
    for (int i = threadIdx.x; i < rows * pairs; i += QK_THREADS) {
        const int r = a.by_pairs(i), j = i - r * pairs, axis = a.by_p(j);
        const uint64_t turn = (uint64_t)(int64_t)a.grid[3 * (row0 + r) + axis] * a.freq[j - axis * a.p];
        // signed fraction of a turn, of which sincospif wants twice as many half turns
        const float half = (float)(int32_t)(turn >> 32) * (2.f / 4294967296.f);
        sincospif(half, &cs[i].y, &cs[i].x);
    }
}

// 16 bytes as packed pairs of floats
template <typename T> struct QkPairs;
template <> struct QkPairs<float> {
    static constexpr int N = 2;
    __device__ static void load(const uint4& r, uint64_t* p)
    {
        p[0] = pack2u(r.x, r.y);
        p[1] = pack2u(r.z, r.w);
    }
    __device__ static uint4 store(const uint64_t* p)
    {
        return make_uint4((uint32_t)p[0], (uint32_t)(p[0] >> 32), (uint32_t)p[1], (uint32_t)(p[1] >> 32));
    }
};
template <> struct QkPairs<__nv_bfloat16> {
    static constexpr int N = 4;
    __device__ static void load(const uint4& r, uint64_t* p)
    {
        p[0] = unpack_bf16x2(r.x);
        p[1] = unpack_bf16x2(r.y);
        p[2] = unpack_bf16x2(r.z);
        p[3] = unpack_bf16x2(r.w);
    }
    __device__ static uint32_t one(uint64_t p)
    {
        float x, y;
        unpack2(p, x, y);
        return pack_bf16(x, y);
    }
    __device__ static uint4 store(const uint64_t* p) { return make_uint4(one(p[0]), one(p[1]), one(p[2]), one(p[3])); }
};

// Weights i and i + 1 as a pair.  A vector of weights is wherever its caller has it (a slice of a buffer of all parameters), so it
// is read value by value: 16-bit weights start on 2 bytes.  A thread does this once.
__device__ __forceinline__ uint64_t qk_weights(const void* weights, int i, int bf16)
{
    if (!bf16) return pack2(((const float*)weights)[i], ((const float*)weights)[i + 1]);
    const __nv_bfloat16* w = (const __nv_bfloat16*)weights;
    return pack2(__bfloat162float(w[i]), __bfloat162float(w[i + 1]));
}

// the first `turned` pairs rotated
template <int N>
__device__ __forceinline__ void qk_rotate(uint64_t (&y)[N], const float2* cs, int turned, bool back)
{
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < turned) {
            const float2 t = cs[i];
            const float s = back ? -t.y : t.y;
            float u, v;
            unpack2(y[i], u, v);
            y[i] = pack2(fmaf(u, t.x, -v * s), fmaf(u, s, v * t.x));
        }
}

// sum over the lanes that hold a head
__device__ __forceinline__ float qk_head_sum(float v, int lanes)
{
    for (int d = 1; d < lanes; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

template <typename T, bool NORM, bool BACK>
__global__ void __launch_bounds__(QK_THREADS, NORM && BACK ? 2 : 3) qk_norm_rope_kernel(const QkArgs a)
{
    using P = QkPairs<T>;
    constexpr int N = P::N;
    extern __shared__ float2 angles[];
    __shared__ float sums[NORM && BACK ? QK_THREADS : 1][2 * N + 1];
    const int lanes = a.D / (2 * N);                    // of a head: a power of two that divides a warp
    const int pairs = a.grid ? 3 * a.p : 0;
    // this thread's column, and its row among those of a pass (threads beyond the last have none)
    const int c = blockIdx.y * QK_THREADS + threadIdx.x % a.columns, r0 = threadIdx.x / a.columns;
    const bool have = c < a.vec_row && r0 < a.rows;
    const int part = !have ? 2 : c < a.vec_c ? 0 : c < 2 * a.vec_c ? 1 : 2;
    const int first = threadIdx.x % lanes * N;          // pair of its head (all threads of a head have such neighbours)
    const int turned = part == 2 ? 0 : pairs - first;
    uint64_t w[N], dw[N];
    if (NORM) {
        const void* weights = part == 0 ? a.qw : a.kw;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[i] = qk_weights(weights, 2 * (first + i), a.w_bf16);
            dw[i] = 0;
        }
    }
    const uint4* in = (const uint4*)a.qkv;
    const uint4* grad = (const uint4*)a.dout;
    uint4* out = (uint4*)a.out;
    const int rows = a.rows * QK_PASSES;
    int turn = 0;
    for (int64_t row0 = (int64_t)blockIdx.x * rows; row0 < a.n; row0 += (int64_t)gridDim.x * rows, turn ^= 1) {
        const int left = (int)min((int64_t)rows, a.n - row0);
        // two sets of angles in turn: nobody is still reading the one before the last
        float2* cs = angles + turn * rows * pairs;
        uint4 x[QK_PASSES], g[QK_PASSES];
        const int64_t base = (row0 + r0) * a.vec_row + c, step = (int64_t)a.rows * a.vec_row;
        // (rows are asked for ahead of their angles, so that one latency hides the other)
#pragma unroll
        for (int u = 0; u < QK_PASSES; ++u)
            if (have && r0 + u * a.rows < left) {
                if (BACK) g[u] = grad[base + u * step];
                if (!BACK || (NORM && part != 2)) x[u] = in[base + u * step];
            }
        if (pairs) {
            qk_angles(a, row0, left, cs);
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < QK_PASSES; ++u) {
            const int r = r0 + u * a.rows;
            const bool live = have && r < left;
            const float2* turns = cs + (live ? r * pairs + first : 0);
            uint64_t y[N], z[N];
            float inv = 0.f;
            if (!BACK || NORM) P::load(x[u], y);
            if (NORM) {
                uint64_t s = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) s = fma2(y[i], y[i], s);
                inv = rsqrtf(qk_head_sum(hsum2(s), lanes) / (float)a.D + a.eps);
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = mul2(y[i], pack2(inv, inv));
            }
            if (!BACK) {
                if (NORM)
#pragma unroll
                    for (int i = 0; i < N; ++i) y[i] = mul2(y[i], w[i]);
                qk_rotate(y, turns, turned, false);
                if (live) out[base + u * step] = part == 2 ? x[u] : P::store(y);
            } else {
                P::load(g[u], z);
                qk_rotate(z, turns, turned, true);
                if (NORM) {
                    uint64_t m = 0;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        if (live) dw[i] = fma2(z[i], y[i], dw[i]);
                        z[i] = mul2(z[i], w[i]);
                        m = fma2(z[i], y[i], m);
                    }
                    const float mean = -qk_head_sum(hsum2(m), lanes) / (float)a.D;
#pragma unroll
                    for (int i = 0; i < N; ++i) z[i] = mul2(fma2(y[i], pack2(mean, mean), z[i]), pack2(inv, inv));
                }
                if (live) out[base + u * step] = part == 2 ? g[u] : P::store(z);
            }
        }
    }
    if (NORM && BACK) {
        // a block's sums: its threads of one part and place, in their order
#pragma unroll
        for (int i = 0; i < N; ++i) unpack2(dw[i], sums[threadIdx.x][2 * i], sums[threadIdx.x][2 * i + 1]);
        __syncthreads();
        const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
        for (int i = threadIdx.x; i < 2 * a.D; i += QK_THREADS) {
            const int key = i >= a.D, d = i - key * a.D;
            const int lo = max(key * a.vec_c - (int)blockIdx.y * QK_THREADS, 0);
            const int hi = min((key + 1) * a.vec_c - (int)blockIdx.y * QK_THREADS, a.columns);
            float v = 0.f;
            for (int r = 0; r < a.rows; ++r)
                for (int k = lo + d / (2 * N); k < hi; k += lanes) v += sums[r * a.columns + k][d % (2 * N)];
            a.partial[block * 2 * a.D + i] = v;
        }
    }
}

// weights' gradients: a warp per value adds the blocks' sums
__global__ void __launch_bounds__(256) qk_weights_kernel(const float* partial, int blocks, int D, void* dq, void* dk,
                                                                int bf16)
{
    const int i = (blockIdx.x * 256 + threadIdx.x) / 32, lane = threadIdx.x & 31;
    if (i >= 2 * D) return;
    float v = 0.f;
#pragma unroll 8
    for (int b = lane; b < blocks; b += 32) v += partial[(int64_t)b * 2 * D + i];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (lane) return;
    void* to = i < D ? dq : dk;
    if (bf16) ((__nv_bfloat16*)to)[i % D] = __float2bfloat16_rn(v);
    else ((float*)to)[i % D] = v;
}

// Blocks of rows: as many as are resident; and of columns, for rows of more vectors than a block has threads
constexpr int QK_MAX_BLOCKS = SMS * 3;
static dim3 qk_grid(int64_t n, int vec_row)
{
    const int rows = (vec_row < QK_THREADS ? QK_THREADS / vec_row : 1) * QK_PASSES, wide = ceil_div(vec_row, QK_THREADS);
    const int64_t b = (n + rows - 1) / rows, most = ceil_div(QK_MAX_BLOCKS, wide);
    return dim3((unsigned)(b < most ? b : most), wide);
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
    PTV3_REQUIRE(channels <= 1 << 16, PTV3_ERR_UNSUPPORTED, "%s: %d channels", what, channels);
    PTV3_REQUIRE(!qw == !kw && (qw || grid), PTV3_ERR_INVALID_ARGUMENT,
                 "%s: weights of both queries and keys, coordinates, or all three", what);
    PTV3_REQUIRE((((uintptr_t)qw | (uintptr_t)kw) & (weight_dtype == PTV3_DTYPE_BF16 ? 1 : 3)) == 0,
                 PTV3_ERR_INVALID_ARGUMENT, "%s: unaligned weights", what);
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
    a.columns = a.vec_row < QK_THREADS ? a.vec_row : QK_THREADS;
    a.rows = QK_THREADS / a.columns;
    a.D = channels / heads;
    a.p = a.D / 6;
    a.w_bf16 = weight_dtype == PTV3_DTYPE_BF16;
    a.eps = eps;
    a.by_pairs = QkDiv(3 * a.p);
    a.by_p = QkDiv(a.p);
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
    const dim3 grid = qk_grid(a.n, a.vec_row);
    const size_t smem = a.grid ? (size_t)a.rows * QK_PASSES * 3 * a.p * 2 * sizeof(float2) : 0;
    if (a.qw) qk_norm_rope_kernel<T, true, BACK><<<grid, QK_THREADS, smem, stream>>>(a);
    else qk_norm_rope_kernel<T, false, BACK><<<grid, QK_THREADS, smem, stream>>>(a);
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
    const dim3 most = qk_grid(n, 3 * channels * 4 / 16), least = qk_grid(n, 3 * channels * 2 / 16);     // fp32, bf16
    const size_t blocks = (size_t)most.x * most.y > (size_t)least.x * least.y ? (size_t)most.x * most.y
                                                                             : (size_t)least.x * least.y;
    return blocks * 2 * (channels / heads) * sizeof(float);
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
        const dim3 grid = qk_grid(n, a.vec_row);
        qk_weights_kernel<<<ceil_div(2 * a.D * 32, 256), 256, 0, s>>>(a.partial, n > 0 ? (int)(grid.x * grid.y) : 0, a.D,
                                                                      dq_weight, dk_weight, a.w_bf16);
        count_launches(1);
    }
    return check_launch(what);
}
