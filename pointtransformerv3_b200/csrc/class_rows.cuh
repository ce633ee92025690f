// Rows of logits, for the kernels that answer or learn from them (class_scores.cu, distill.cu, seg_head_scores.cu).
//
// z = x / T, m = max x, S = sum exp((x - m) / T), log p_j = (x_j - m) / T - log S.  The maximum is taken out of the
// logits themselves, before the division, so that rows of any height keep their differences; a gradient is made from m and
// log S apart, for the same reason.  Exponentials are 2^t, t = (x - m) c, c = log2(e) / T, on the exponential unit
// (relative error 2^-22); log S is log1p(S - 1), the accurate function, once per row: near a certain class log S is small, and
// the fast logarithm has an absolute error there.
//
// Masked classes are minus infinity: t is held at -200, whose power is zero in fp32, so that 0 * t is zero too.  NaN and plus
// infinity pass through max.NaN and make the row's sums NaN.  A row of minus infinities alone has S = 0.
#pragma once
#include "common.cuh"
#include "convert.cuh"
#include "mma_util.cuh"
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

// ---- 8 neighbouring logits of a row ---------------------------------------------------------------------------------
template <typename T> struct Eight;
template <> struct Eight<__nv_bfloat16> {
    static constexpr int WORDS = 4;
    uint32_t w[4];
    __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
    __device__ __forceinline__ uint64_t pair(int q) const { return unpack_bf16x2(w[q]); }
    __device__ __forceinline__ void keep_first(int count)       // the others become minus infinity
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i >= count) w[i >> 1] = i & 1 ? (w[i >> 1] & 0xffffu) | 0xff800000u : (w[i >> 1] & 0xffff0000u) | 0xff80u;
    }
    __device__ __forceinline__ float largest() const            // NaN if one is
    {
        __nv_bfloat162 a = __hmax2_nan(h(0), h(1)), b = __hmax2_nan(h(2), h(3));
        a = __hmax2_nan(a, b);
        return max_nan(__low2float(a), __high2float(a));
    }
    __device__ __forceinline__ __nv_bfloat162 h(int q) const { return *reinterpret_cast<const __nv_bfloat162*>(&w[q]); }
    __device__ __forceinline__ void set(int q, float lo, float hi) { w[q] = pack_bf16(lo, hi); }
};
template <> struct Eight<float> {
    static constexpr int WORDS = 8;
    uint32_t w[8];
    __device__ __forceinline__ float at(int i) const { return __uint_as_float(w[i]); }
    __device__ __forceinline__ uint64_t pair(int q) const { return pack2u(w[2 * q], w[2 * q + 1]); }
    __device__ __forceinline__ void keep_first(int count)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i >= count) w[i] = 0xff800000u;
    }
    __device__ __forceinline__ float largest() const
    {
        return max_nan(max_nan(max_nan(at(0), at(1)), max_nan(at(2), at(3))), max_nan(max_nan(at(4), at(5)), max_nan(at(6), at(7))));
    }
    __device__ __forceinline__ void set(int q, float lo, float hi)
    {
        w[2 * q] = __float_as_uint(lo);
        w[2 * q + 1] = __float_as_uint(hi);
    }
};

constexpr float NO_POWER = -200.f;
// S and, where they are wanted (U), sum e t of a row, in packed pairs.  Eight are added to one another first: a row's sum is rounded an eighth as often.
template <bool U>
struct RowSum {
    uint64_t s, u;
    __device__ __forceinline__ void clear() { s = u = 0; }
    template <typename T>
    __device__ __forceinline__ void add(const Eight<T>& x, uint64_t minus_origin, uint64_t c)
    {
        uint64_t e[4], v = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float lo, hi;
            unpack2(mul2(add2(x.pair(q), minus_origin), c), lo, hi);
            if (U) {
                lo = max_nan(lo, NO_POWER);
                hi = max_nan(hi, NO_POWER);
            }
            e[q] = pack2(fast_exp2(lo), fast_exp2(hi));
            if (U) v = q ? fma2(e[q], pack2(lo, hi), v) : mul2(e[q], pack2(lo, hi));
        }
        s = add2(s, add2(add2(e[0], e[1]), add2(e[2], e[3])));
        if (U) u = add2(u, v);
    }
};
// Eight of a gradient: p (A + B t) with p = 2^t, t = (x - m) c + shift = log2 p; without LOG, p A
template <bool LOG, typename T>
__device__ __forceinline__ void row_gradient(Eight<T>& x, uint64_t minus_m, uint64_t c, uint64_t shift, uint64_t A, uint64_t B)
{
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float lo, hi;
        unpack2(fma2(add2(x.pair(q), minus_m), c, shift), lo, hi);
        if (LOG) {
            lo = max_nan(lo, NO_POWER);
            hi = max_nan(hi, NO_POWER);
        }
        unpack2(mul2(pack2(fast_exp2(lo), fast_exp2(hi)), LOG ? fma2(pack2(lo, hi), B, A) : A), lo, hi);
        x.set(q, lo, hi);
    }
}

// ---- the largest of a row, kept sorted in a thread's registers ------------------------------------------------------------
// Keys say value and class: the larger value first, then the lower class, so that no two are equal and the order in which they
// come does not matter.  bf16: 16 bits of each (rows of up to 2^16 classes); fp32: 32 and 32.  0: no class.
template <typename T> struct TopKey;
template <> struct TopKey<__nv_bfloat16> {
    using Key = uint32_t;
    // of eight classes from j on
    __device__ static __forceinline__ void keys(const Eight<__nv_bfloat16>& x, int j, Key* k)
    {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            // (adding zero: one zero, one NaN)
            const __nv_bfloat162 one = __hadd2_rn(x.h(q), __nv_bfloat162(__ushort_as_bfloat16(0), __ushort_as_bfloat16(0)));
            const uint32_t w = *reinterpret_cast<const uint32_t*>(&one);
            const uint32_t o = w ^ (((w >> 15) & 0x00010001u) * 0x7fffu | 0x80008000u);
            const uint32_t at = 0xffffu - (j + 2 * q);
            k[2 * q] = __byte_perm(at, o, 0x5410);
            k[2 * q + 1] = __byte_perm(at - 1, o, 0x7610);
        }
    }
    __device__ static __forceinline__ int cls(Key k) { return k ? (int)(0xffffu - (k & 0xffffu)) : -1; }
    __device__ static __forceinline__ float value(Key k) { return order_value((k & 0xffff0000u) | (k >> 31 ? 0 : 0xffffu)); }
};
template <> struct TopKey<float> {
    using Key = unsigned long long;
    __device__ static __forceinline__ void keys(const Eight<float>& x, int j, Key* k)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = (unsigned long long)order_key(x.at(i)) << 32 | (0xffffffffu - (j + i));
    }
    __device__ static __forceinline__ int cls(Key k) { return k ? (int)(0xffffffffu - (uint32_t)k) : -1; }
    __device__ static __forceinline__ float value(Key k) { return order_value((uint32_t)(k >> 32)); }
};

__device__ __forceinline__ void larger_first(int& a, int& b)
{
    const int hi = ::max(a, b), lo = ::min(a, b);
    a = hi;
    b = lo;
}
__device__ __forceinline__ void larger_first(uint32_t& a, uint32_t& b)
{
    const uint32_t hi = ::max(a, b), lo = ::min(a, b);
    a = hi;
    b = lo;
}
template <typename K>
__device__ __forceinline__ void larger_first(K& a, K& b)
{
    const K hi = a > b ? a : b, lo = a > b ? b : a;
    a = hi;
    b = lo;
}
// B keys in falling order: odd-even merge sort, about B log^2 B / 4 exchanges (recursion, so that every index is a constant)
template <int LO, int N, int R, typename K>
__device__ __forceinline__ void merge_halves(K* k)
{
    if constexpr (2 * R < N) {
        merge_halves<LO, N, 2 * R>(k);
        merge_halves<LO + R, N, 2 * R>(k);
#pragma unroll
        for (int i = LO + R; i + R < LO + N; i += 2 * R) larger_first(k[i], k[i + R]);
    } else {
        larger_first(k[LO], k[LO + R]);
    }
}
template <int N, int LO = 0, typename K>
__device__ __forceinline__ void sort_keys(K* k)
{
    if constexpr (N > 1) {
        sort_keys<N / 2, LO>(k);
        sort_keys<N / 2, LO + N / 2>(k);
        merge_halves<LO, N, 1>(k);
    }
}
// best, in falling order, becomes the best of itself and k, both in falling order: the larger of each with its opposite is a
// bitonic row of the best B, which log B half-cleaners sort
template <int B, typename K>
__device__ __forceinline__ void merge_keys(K* best, const K* k)
{
#pragma unroll
    for (int i = 0; i < B; ++i) best[i] = best[i] > k[B - 1 - i] ? best[i] : k[B - 1 - i];
#pragma unroll
    for (int d = B / 2; d >= 1; d /= 2)
#pragma unroll
        for (int i = 0; i < B; ++i)
            if ((i & d) == 0) larger_first(best[i], best[i + d]);
}

// ---- G threads to a row: part of a warp, a warp, or a block ----------------------------------------------------------
template <int G>
struct Group {
    static constexpr int WARPS = G <= 32 ? 1 : G / 32;
    static constexpr int BLOCK = G <= 32 ? 128 : G;           // threads of a block
    static constexpr int ROWS = G <= 32 ? 128 / G : 1;        // rows of a block
    // scratch: 4 * WARPS floats of shared memory for a block, unused by a warp
    float* scratch;
    __device__ __forceinline__ int rank() const { return threadIdx.x & (G - 1); }
    __device__ __forceinline__ int slot() const { return G <= 32 ? threadIdx.x / G : 0; }
    __device__ __forceinline__ int64_t row() const { return blockIdx.x * (int64_t)ROWS + slot(); }
    __device__ __forceinline__ void sync() const
    {
        if (G <= 32)
            __syncwarp();
        else
            __syncthreads();
    }
    // whether it holds for any of the row's threads, which meet here
    __device__ __forceinline__ bool any(bool v) const
    {
        if (G > 32) return __syncthreads_or(v);
        const uint32_t all = __ballot_sync(~0u, v);
        return ((G < 32 ? all >> (threadIdx.x & (32 - G) & 31) & ((1u << (G & 31)) - 1) : all)) != 0;
    }
    __device__ __forceinline__ float max(float v) const
    {
#pragma unroll
        for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(~0u, v, o));
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
        for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1)
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
    static unsigned blocks(int64_t n) { return (unsigned)((n + ROWS - 1) / ROWS); }
};

// A row as its pieces of eight logits that start on 16 bytes (32 bytes of fp32: two loads) and, wherever the row starts and ends, the
// values before the first and behind the last of these, its edges: 14 at most, read one by one, so that nothing beside the row is read.
// (With whole pieces whose foreign values are masked, lists of 50 021 x 1 201 took 58 us forward instead of 46, backward 73 instead of 68.)
constexpr int EDGES = 14;
template <typename T>
struct RowPieces {
    const T* row;
    int K, head, pieces, edges;
    __device__ __forceinline__ RowPieces(const T* r, int k)
    {
        row = r;
        K = k;
        head = min(K, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T));
        pieces = (K - head) / 8;
        edges = K - 8 * pieces;
    }
    // class of the first value of piece p, of edge value e
    __device__ __forceinline__ int first(int p) const { return head + p * 8; }
    __device__ __forceinline__ int edge_class(int e) const { return e < head ? e : e + 8 * pieces; }
    __device__ __forceinline__ Eight<T> load(int p) const
    {
        Eight<T> x;
        const uint4* src = reinterpret_cast<const uint4*>(row + first(p));
        *reinterpret_cast<uint4*>(&x.w[0]) = src[0];
        if (Eight<T>::WORDS == 8) *reinterpret_cast<uint4*>(&x.w[Eight<T>::WORDS - 4]) = src[1];
        return x;
    }
    // eight from class j on into a row of results that lies as this one does with respect to 16 bytes (`alike`), or elsewhere
    __device__ __forceinline__ void store(T* out, bool alike, int j, const Eight<T>& x) const
    {
        if (alike) {
            uint4* dst = reinterpret_cast<uint4*>(out + j);
            dst[0] = *reinterpret_cast<const uint4*>(&x.w[0]);
            if (Eight<T>::WORDS == 8) dst[1] = *reinterpret_cast<const uint4*>(&x.w[Eight<T>::WORDS - 4]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) out[j + i] = from_f<T>(x.at(i));
        }
    }
};
// a row with G threads: P pieces of each in registers, or none, to be read again for every pass; and the edges
template <typename T, int G, int P>
struct RowValues {
    static constexpr int EDGE = (EDGES + G - 1) / G;
    Eight<T> x[P > 0 ? P : 1];
    float edge[EDGE];
    const RowPieces<T>& pieces;
    int rank;
    __device__ __forceinline__ RowValues(const RowPieces<T>& p, int me) : pieces(p), rank(me)
    {
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (i * G + rank < pieces.pieces) x[i] = pieces.load(i * G + rank);
#pragma unroll
        for (int q = 0; q < EDGE; ++q) {
            const int e = q * G + rank;
            edge[q] = e < pieces.edges ? to_f<T>(pieces.row[pieces.edge_class(e)]) : -INFINITY;
        }
    }
    // f(eight logits, class of the first), g(one logit, its class; e: its number among the thread's edge values)
    template <typename F, typename E>
    __device__ __forceinline__ void each(F&& f, E&& g) const
    {
        if (P > 0) {
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (i * G + rank < pieces.pieces) f(x[i], pieces.first(i * G + rank), i);
        } else {
#pragma unroll 2
            for (int p = rank; p < pieces.pieces; p += G) f(pieces.load(p), pieces.first(p), p / G);
        }
        if (pieces.edges) {
#pragma unroll
            for (int q = 0; q < EDGE; ++q)
                if (q * G + rank < pieces.edges) g(edge[q], pieces.edge_class(q * G + rank), q);
        }
    }
};
// one logit's part of a row's sums
struct EdgeSum {
    float s, u;
    __device__ __forceinline__ void add(float x, float origin, float c)
    {
        const float t = max_nan((x - origin) * c, NO_POWER), e = fast_exp2(t);       // (few: both, always)
        s += e;
        u = fmaf(e, t, u);
    }
};

// ---- a tile of rows in shared memory, one thread to a row -----------------------------------------------------------
// No sums or choices across threads: a row costs the fewest instructions so, and short rows are bound by these.  Rows lie as they do in
// memory, so that a tile is copied in pieces of 16 bytes whatever K is; a thread reads eight logits at a time, as wide as rows are aligned:
//   16 bytes  rows of a multiple of 16 bytes; an odd number of such pieces apart, so that eight neighbours' reads fill the banks
//   8, 4      rows of another multiple of 8 or 4 bytes: an odd number of 8-byte pieces apart, or of words: no conflicts either
//   2         rows of an odd number of bf16 values: neighbours share words, which are broadcast
constexpr int TILE_SLACK = 64;      // bytes that the last row's last read may reach beyond it

template <typename T>
struct RowTile {
    unsigned char* smem;
    int K, pitch, width;            // bytes from row to row, bytes of a read
    __host__ __device__ static int row_width(int K)
    {
        const int bytes = K * (int)sizeof(T);
        return bytes % 16 == 0 ? 16 : bytes % 8 == 0 ? 8 : bytes % 4 == 0 ? 4 : 2;
    }
    __host__ __device__ static int row_pitch(int K)
    {
        const int bytes = K * (int)sizeof(T);
        return bytes % 16 == 0 ? (bytes / 16 | 1) * 16 : bytes;
    }
    __device__ __forceinline__ RowTile(unsigned char* s, int k) : smem(s), K(k), pitch(row_pitch(k)), width(row_width(k)) {}
    __device__ __forceinline__ T* row(int r) const { return reinterpret_cast<T*>(smem + r * pitch); }

    // rows of the matrix into the tile (all threads; they are there after `wait`).  wide: they may be read in pieces of 16 bytes, which is where
    // they lie one behind the other, or each on 16 bytes
    __device__ __forceinline__ void fetch(const T* logits, int64_t ld, int64_t row0, int rows, bool wide) const
    {
        const int threads = blockDim.x;
        const T* src = logits + row0 * ld;
        int done = 0;                // values
        if (wide && width == 16) {
            const int per_row = K * (int)sizeof(T) / 16;
            int r = threadIdx.x / per_row, c = threadIdx.x % per_row;
            const int dr = threads / per_row, dc = threads % per_row;
            for (int i = threadIdx.x; i < rows * per_row; i += threads) {
                copy16(smem + r * pitch + c * 16, reinterpret_cast<const unsigned char*>(src + r * ld) + c * 16);
                r += dr;
                c += dc;
                if (c >= per_row) {
                    c -= per_row;
                    ++r;
                }
            }
            done = rows * K;
        } else if (wide) {
            const int pieces = rows * K * (int)sizeof(T) / 16;
            for (int i = threadIdx.x; i < pieces; i += threads) copy16(smem + i * 16, reinterpret_cast<const unsigned char*>(src) + i * 16);
            done = pieces * (16 / (int)sizeof(T));
        }
        for (int i = done + threadIdx.x; i < rows * K; i += threads) {
            const int r = i / K, c = i - r * K;
            row(r)[c] = src[r * ld + c];
        }
    }
    __device__ __forceinline__ void wait() const
    {
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
    }
    // the tile's rows out to rows one behind the other (after a barrier of the caller's)
    __device__ __forceinline__ void store(T* out, int64_t row0, int rows, bool wide) const
    {
        const int threads = blockDim.x;
        T* dst = out + row0 * K;
        int done = 0;
        if (wide && width == 16) {
            const int per_row = K * (int)sizeof(T) / 16;
            int r = threadIdx.x / per_row, c = threadIdx.x % per_row;
            const int dr = threads / per_row, dc = threads % per_row;
            for (int i = threadIdx.x; i < rows * per_row; i += threads) {
                reinterpret_cast<uint4*>(dst)[i] = *reinterpret_cast<const uint4*>(smem + r * pitch + c * 16);
                r += dr;
                c += dc;
                if (c >= per_row) {
                    c -= per_row;
                    ++r;
                }
            }
            done = rows * K;
        } else if (wide) {
            const int pieces = rows * K * (int)sizeof(T) / 16;
            for (int i = threadIdx.x; i < pieces; i += threads) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(smem)[i];
            done = pieces * (16 / (int)sizeof(T));
        }
        for (int i = done + threadIdx.x; i < rows * K; i += threads) {
            const int r = i / K;
            dst[i] = row(r)[i - r * K];
        }
    }
    static __device__ __forceinline__ void copy16(void* to, const void* from)
    {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
    }

    // W: the tile's width, known to the compiler.  Values beyond the row are minus infinity.
    template <int W>
    __device__ __forceinline__ Eight<T> read(const T* r, int j) const
    {
        Eight<T> x;
        const unsigned char* p = reinterpret_cast<const unsigned char*>(r + j);
        if (W == 16) {
#pragma unroll
            for (int i = 0; i < Eight<T>::WORDS / 4; ++i) *reinterpret_cast<uint4*>(&x.w[4 * i]) = reinterpret_cast<const uint4*>(p)[i];
        } else if (W == 8) {
#pragma unroll
            for (int i = 0; i < Eight<T>::WORDS / 2; ++i) *reinterpret_cast<uint2*>(&x.w[2 * i]) = reinterpret_cast<const uint2*>(p)[i];
        } else if (W == 4) {
#pragma unroll
            for (int i = 0; i < Eight<T>::WORDS; ++i) x.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < Eight<T>::WORDS; ++i) {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + 2 * i;
                x.w[i] = (uint32_t)h[0] | (uint32_t)h[1] << 16;
            }
        }
        if (j + 8 > K) x.keep_first(K - j);
        return x;
    }
    template <int W>
    __device__ __forceinline__ void write(T* r, int j, const Eight<T>& x) const
    {
        unsigned char* p = reinterpret_cast<unsigned char*>(r + j);
        if (j + 8 > K) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i < K) r[j + i] = from_f<T>(x.at(i));
        } else if (W == 16) {
#pragma unroll
            for (int i = 0; i < Eight<T>::WORDS / 4; ++i) reinterpret_cast<uint4*>(p)[i] = *reinterpret_cast<const uint4*>(&x.w[4 * i]);
        } else if (W == 8) {
#pragma unroll
            for (int i = 0; i < Eight<T>::WORDS / 2; ++i) reinterpret_cast<uint2*>(p)[i] = *reinterpret_cast<const uint2*>(&x.w[2 * i]);
        } else if (W == 4) {
#pragma unroll
            for (int i = 0; i < Eight<T>::WORDS; ++i) reinterpret_cast<uint32_t*>(p)[i] = x.w[i];
        } else {
#pragma unroll
            for (int i = 0; i < Eight<T>::WORDS; ++i) {
                uint16_t* h = reinterpret_cast<uint16_t*>(p) + 2 * i;
                h[0] = (uint16_t)x.w[i];
                h[1] = (uint16_t)(x.w[i] >> 16);
            }
        }
    }
    template <int W>
    __device__ __forceinline__ float largest(const T* r) const
    {
        float m = -INFINITY;
        for (int j = 0; j < K; j += 8) m = max_nan(m, read<W>(r, j).largest());
        return m;
    }
    // whether `load` and `store` may take pieces of 16 bytes
    static bool wide_rows(const void* p, int64_t ld, int K)
    {
        return ((uintptr_t)p & 15) == 0 && (ld == K || (ld * sizeof(T) % 16 == 0 && row_width(K) == 16));
    }
};

// Blocks of these that an SM has at least: 64 registers of a thread for up to 32 words of a row, 102 for 64 (alternatives of 4 099 x 8 192
// fp32: 53 us with the 168 that the compiler would take, 40 so).
template <typename T>
constexpr int row_blocks(int G, int P)
{
    return P * Eight<T>::WORDS <= 32 ? (G <= 128 ? 8 : 1) : (G <= 128 ? 5 : G <= 256 ? 2 : 1);
}
// Threads of a row and pieces of each.  A thread holds up to 128 bf16 or 64 fp32 logits in 64 registers, all of them on the way at once:
// that, not many warps, is what keeps memory busy, and one warp to a row waits for no barrier.  Short rows take part of a warp, so
// that what is done once for a row is done for several at a time.
template <int N> struct Const { static constexpr int value = N; };
template <typename T, typename F>
static inline void for_row_shape(int K, bool warps, bool once, F&& f)
{
    // (once: the row is passed over once, so that the longest need not be held: 1 500 x 20 001 backward 57 us held, 40 read as they are needed)
    constexpr int P = sizeof(T) == 2 ? 8 : 4;
    if (K <= 8 * 8 * P && warps)
        K <= 256 ? f(Const<32>(), Const<1>()) : f(Const<32>(), Const<2>());
    else if (K <= 4 * 8 * P)
        f(Const<4>(), Const<P>());
    else if (K <= 8 * 8 * P)
        f(Const<8>(), Const<P>());
    else if (K <= 16 * 8 * P)
        warps ? f(Const<32>(), Const<P / 2>()) : f(Const<16>(), Const<P>());
    else if (K <= 32 * 8 * P)
        f(Const<32>(), Const<P>());
    else if (K <= 32 * 16 * P)
        f(Const<32>(), Const<2 * P>());
    else if (K <= 128 * 16 * P)
        f(Const<128>(), Const<2 * P>());
    else if (once)
        f(Const<256>(), Const<0>());
    else if (K <= 256 * 16 * P)
        f(Const<256>(), Const<2 * P>());
    else if (K <= 512 * 16 * P)
        f(Const<512>(), Const<2 * P>());
    else
        f(Const<1024>(), Const<0>());
}

// Rows and shared memory of a block with a tile.
struct TileShape {
    int rows;
    size_t smem;
};
// Rows in tiles or spread over threads.  A thread to a row costs the fewest instructions but wants a tile of 128 rows for every SM (many_rows), and
// fewer tiles are resident the longer rows are.  Each operator has the bytes up to which that pays, with both sides measured.
constexpr size_t TILE_BYTES = 128;          // always
constexpr bool many_rows(int64_t n) { return n >= (int64_t)SMS * 128; }
template <typename T>
static inline TileShape tile_shape(int K)
{
    const int pitch = RowTile<T>::row_pitch(K);
    const int rows = pitch <= 272 ? 128 : 64;
    return TileShape{rows, (size_t)rows * pitch + TILE_SLACK};
}

}  // namespace ptv3
