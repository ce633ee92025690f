// Rows of logits, for the kernels that answer or learn from them (class_scores.cu, distill.cu, seg_head_scores.cu).
//
// z = x / T, m = max x, S = sum exp((x - m) / T), log p_j = (x_j - m) / T - log S.  The maximum is taken out of the
// logits themselves, before the division, so that rows of any height keep their differences; a gradient is made from m and
// log S apart, for the same reason.  Exponentials are 2^(d c), d = x - m, c = log2(e) / T, on the exponential unit
// (relative error 2^-22); log S is log1p(S - 1), the accurate function, once per row: near a certain class log S is small, and
// the fast logarithm has an absolute error there.
//
// Masked classes are minus infinity: d is held at -1e38, whose exponential is zero, so that 0 * d is zero too.  NaN and plus
// infinity pass through max.NaN and make the row's sums NaN.  A row of minus infinities alone has S = 0.
#pragma once
#include "common.cuh"
#include "convert.cuh"
#include "vec.cuh"

namespace ptv3 {

constexpr int CLASSES_MAX = 1 << 18;
constexpr int LIST_MAX = 64;
constexpr float LOG2E = 1.4426950408889634f;
// Of all classes' probability, what a sum of some of them may be before it is taken again from their own maximum: values
// beside it are then lost below the smallest fp32, not before.
constexpr float REST_TOO_SMALL = 1e-20f;

__device__ __forceinline__ float below_max(float x, float m) { return max_nan(x - m, -1e38f); }
// what is taken out of the logits of a row whose largest is m
__device__ __forceinline__ float row_origin(float m) { return m == -INFINITY ? 0.f : m; }

// Order of logits as unsigned integers: NaN above all, both zeros alike; 0 is below every logit.
__device__ __forceinline__ uint32_t order_key(float x)
{
    uint32_t u = __float_as_uint(x);
    if (u == 0x80000000u) u = 0;
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t key)
{
    return __uint_as_float(key ^ ((uint32_t)((int32_t)~key >> 31) | 0x80000000u));
}

__device__ __forceinline__ int64_t load_index(const void* p, int bytes, int64_t i)
{
    return bytes == 8 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}
__device__ __forceinline__ float load_value(const void* p, bool bf16, int64_t i)
{
    return bf16 ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : ((const float*)p)[i];
}

// ---- G threads to a row: a warp (of several in a block) or a whole block --------------------------------------------
template <int G>
struct Group {
    static constexpr int WARPS = G / 32;
    // scratch: 3 * WARPS floats of shared memory for a block, unused by a warp
    float* scratch;
    __device__ __forceinline__ int rank() const { return G == 32 ? (threadIdx.x & 31) : threadIdx.x; }
    __device__ __forceinline__ void sync() const
    {
        if (G == 32)
            __syncwarp();
        else
            __syncthreads();
    }
    __device__ __forceinline__ float max(float v) const
    {
#pragma unroll
        for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(~0u, v, o));
        if (G > 32) {
            __syncthreads();
            if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
            __syncthreads();
            v = scratch[0];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) v = max_nan(v, scratch[w]);
        }
        return v;
    }
    // sums in an order that depends on G alone
    template <int N>
    __device__ __forceinline__ void sum(float (&v)[N]) const
    {
#pragma unroll
        for (int o = 16; o; o >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(~0u, v[i], o);
        if (G > 32) {
            __syncthreads();
            if ((threadIdx.x & 31) == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) scratch[N * (threadIdx.x >> 5) + i] = v[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = scratch[i];
#pragma unroll
            for (int w = 1; w < WARPS; ++w)
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] += scratch[N * w + i];
        }
    }
};

// A row of K logits spread over G threads, in pieces of V values: piece p belongs to thread p % G.  V is what 16 bytes
// hold where rows start on 16 bytes and end there, else 1.
template <typename T, int V>
__device__ __forceinline__ void load_piece(const T* row, int piece, int K, float (&v)[V])
{
    if (V == 1) {
        v[0] = piece < K ? to_f<T>(row[piece]) : -INFINITY;
    } else {
        if (piece * V < K) {
            typename Vec<T>::Raw raw = *reinterpret_cast<const typename Vec<T>::Raw*>(row + (int64_t)piece * V);
            Vec<T>::unpack(raw, v);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = -INFINITY;
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_piece(T* row, int piece, int K, const float (&v)[V])
{
    if (V == 1) {
        if (piece < K) row[piece] = from_f<T>(v[0]);
    } else if (piece * V < K) {
        *reinterpret_cast<typename Vec<T>::Raw*>(row + (int64_t)piece * V) = Vec<T>::pack(v);
    }
}

static inline bool rows_aligned(const void* p, int64_t ld, int K, int size)
{
    return ((uintptr_t)p & 15) == 0 && (ld * size) % 16 == 0 && (K * (int64_t)size) % 16 == 0;
}

// ---- a tile of rows in shared memory, one thread to a row -----------------------------------------------------------
// Rows of up to SMALL_CLASSES logits, as fp32, an odd number of words apart: a thread reads its row without conflicts.
constexpr int SMALL_CLASSES = 64;
constexpr int TILE_ROWS = 128;

__host__ __device__ __forceinline__ int tile_pitch(int K) { return K | 1; }

// Walks the elements idx = first, first + step, ... of rows of K as (row, column) without dividing again.
struct RowWalk {
    int row, col, rows_step, cols_step, K;
    __device__ __forceinline__ RowWalk(int first, int step, int k) : row(first / k), col(first % k), rows_step(step / k), cols_step(step % k), K(k) {}
    __device__ __forceinline__ void next()
    {
        row += rows_step;
        col += cols_step;
        if (col >= K) {
            col -= K;
            ++row;
        }
    }
};

template <typename T>
__device__ __forceinline__ void load_tile(float* tile, const T* logits, int64_t ld, int64_t row0, int rows, int K)
{
    const int pitch = tile_pitch(K);
    const T* src = logits + row0 * ld;
    RowWalk w(threadIdx.x, TILE_ROWS, K);
#pragma unroll 8
    for (int idx = threadIdx.x; idx < rows * K; idx += TILE_ROWS) {
        tile[w.row * pitch + w.col] = to_f<T>(src[w.row * ld + w.col]);
        w.next();
    }
}
template <typename T>
__device__ __forceinline__ void store_tile(const float* tile, T* out, int64_t row0, int rows, int K)
{
    const int pitch = tile_pitch(K);
    T* dst = out + row0 * K;
    RowWalk w(threadIdx.x, TILE_ROWS, K);
#pragma unroll 4
    for (int idx = threadIdx.x; idx < rows * K; idx += TILE_ROWS) {
        dst[idx] = from_f<T>(tile[w.row * pitch + w.col]);
        w.next();
    }
}

}  // namespace ptv3
