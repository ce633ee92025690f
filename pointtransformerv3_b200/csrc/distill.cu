// A student's logits against the best classes that a teacher kept of each row, and the gradient.  No counterpart in the
// reference (its file ends with the backbone, model.py:966-982).
//
// A row's list has k entries (class c_i, value v_i), absent where c_i = -1.  With p the student's probabilities at T:
//     t = softmax(v / T) over the entries                                       (rest = 0)
//     t_i = exp(v_i), and one outcome more: t_r = max(0, 1 - sum t_i) against p_r, the sum of p outside the list   (rest = 1)
//     L = sum t_i (log t_i - log p_{c_i})  [+ t_r (log t_r - log p_r)],   0 without an entry
//     dx_j = g / T (M p_j - sum_{i: c_i = j} t_i)            M = sum t_i (+ t_r)
//     dx_j = g / T (M p_j - t_r p_j / p_r)                   for j outside the list, rest = 1
// p_j / p_r is taken from the outside's own sum, and t_r from expm1 of the largest entry, so that a row of which the list
// leaves a millionth is as exact as any other.  Where the list leaves no class that the student allows, the outcome for the
// rest is left out.  A class that a list has twice counts as two entries.
#include "class_rows.cuh"

namespace ptv3 {

struct DistillArgs {
    const void* logits;       // n rows of K, ld apart
    int64_t ld, n;
    const void* teacher;      // n x k
    const void* list;         // n x k
    int list_bytes, k, K, rest;
    bool teacher_bf16;
    float* loss;              // n
    float4* stats;            // n x {m, log S, log of the outside's sum or the list's largest, t_r or 1 / the list's sum}, or NULL
    float inv_t;
    uint32_t* status;
    const float* g;           // n, g_step apart
    int64_t g_step;
    void* dlogits;            // n x K
};

constexpr int PLACE_ABSENT = -1, PLACE_BAD = -2;
__device__ __forceinline__ int list_class(const DistillArgs& a, int64_t i)
{
    const int64_t c = load_index(a.list, a.list_bytes, i);
    return c >= 0 && c < a.K ? (int)c : (c == -1 ? PLACE_ABSENT : PLACE_BAD);
}

// what a list says by itself: the largest value, the sum of probabilities, whether there is an entry
struct ListSums {
    float top, sum;
    bool any, bad;
    // probability of an entry
    __device__ __forceinline__ float prob(float v, int rest, float inv_t) const
    {
        return rest ? fast_exp2(v * LOG2E) : fast_exp2(below_max(v, row_origin(top)) * (inv_t * LOG2E));
    }
};
// t log t - t log p of an entry; nothing where t is 0
__device__ __forceinline__ float entry_loss(float t, float log_t, float log_p) { return t == 0.f ? 0.f : t * (log_t - log_p); }

// t_r = 1 - sum t: of one large and other small entries the large one's part is taken by expm1
__device__ __forceinline__ float rest_prob(float top, float others) { return fmaxf(-expm1f(fminf(top, 0.f)) - others, 0.f); }

// ---- up to SMALL_CLASSES classes ------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(TILE_ROWS) distill_tile_kernel(const DistillArgs a)
{
    extern __shared__ __align__(16) float tile[];
    const int64_t row0 = blockIdx.x * (int64_t)TILE_ROWS;
    const int rows = (int)min((int64_t)TILE_ROWS, a.n - row0);
    load_tile(tile, (const T*)a.logits, a.ld, row0, rows, a.K);
    __syncthreads();
    if ((int)threadIdx.x >= rows) return;
    const float* x = tile + threadIdx.x * tile_pitch(a.K);
    const int64_t row = row0 + threadIdx.x, at = row * a.k;

    float m = -INFINITY;
    for (int j = 0; j < a.K; ++j) m = max_nan(m, x[j]);
    const float origin = row_origin(m), c = a.inv_t * LOG2E;
    ListSums l{-INFINITY, 0.f, false, false};
    uint64_t inside = 0;
    int first = 0;
    for (int i = 0; i < a.k; ++i) {
        const int cls = list_class(a, at + i);
        l.bad |= cls == PLACE_BAD;
        if (cls < 0) continue;
        const float v = load_value(a.teacher, a.teacher_bf16, at + i);
        inside |= 1ull << cls;
        if (!l.any || v > l.top || v != v) {
            first = i;
            l.top = v;
        }
        l.any = true;
    }
    float s = 0.f, out = 0.f, out_max = -INFINITY;
    for (int j = 0; j < a.K; ++j) {
        const float e = fast_exp2(below_max(x[j], origin) * c);
        s += e;
        if (a.rest && !(inside >> j & 1)) {
            out += e;
            out_max = max_nan(out_max, x[j]);
        }
    }
    const bool none = s == 0.f;
    const float log_s = none ? -INFINITY : log1pf(s - 1.f);
    float log_out = -INFINITY;
    if (a.rest && out_max != -INFINITY) {
        if (out >= REST_TOO_SMALL || out != out) {
            log_out = logf(out);
        } else {
            out = 0.f;
            for (int j = 0; j < a.K; ++j)
                if (!(inside >> j & 1)) out += fast_exp2(below_max(x[j], out_max) * c);
            log_out = (out_max - origin) * a.inv_t + logf(out);
        }
    }
    // the list's sums, then its part of the loss
    float others = 0.f, loss = 0.f;
    for (int i = 0; i < a.k; ++i) {
        const int cls = list_class(a, at + i);
        if (cls < 0) continue;
        const float t = l.prob(load_value(a.teacher, a.teacher_bf16, at + i), a.rest, a.inv_t);
        l.sum += t;
        if (i != first) others += t;
    }
    const float scale = a.rest ? 1.f : (l.sum > 0.f ? __fdiv_rn(1.f, l.sum) : l.sum);
    const float log_scale = a.rest || !(l.sum > 0.f) ? 0.f : logf(l.sum);
    for (int i = 0; i < a.k; ++i) {
        const int cls = list_class(a, at + i);
        if (cls < 0) continue;
        const float v = load_value(a.teacher, a.teacher_bf16, at + i);
        const float log_t = a.rest ? v : below_max(v, row_origin(l.top)) * a.inv_t - log_scale;
        const float log_p = none ? -INFINITY : (x[cls] - origin) * a.inv_t - log_s;
        loss += entry_loss(l.prob(v, a.rest, a.inv_t) * scale, log_t, log_p);
    }
    float t_r = 0.f;
    if (a.rest && l.any && log_out != -INFINITY) {
        t_r = rest_prob(l.top, others);
        loss += entry_loss(t_r, logf(t_r), log_out - log_s);
    }
    if (l.bad) {
        loss = NAN;
        atomicOr(a.status, PTV3_STATUS_BAD_INDEX);
    }
    a.loss[row] = loss;
    if (a.stats) a.stats[row] = a.rest ? make_float4(origin, log_s, log_out, t_r) : make_float4(origin, log_s, row_origin(l.top), scale);
}

// ---- more classes: G threads to a row -----------------------------------------------------------------------------------
constexpr int WARP_ROWS = 4;

// the list, entry i with thread i % G of the first warp of a row's threads
template <int G>
struct ListPart {
    static constexpr int N = G == 32 ? 2 : 1;        // LIST_MAX entries
    int cls[N];
    float v[N];
    __device__ __forceinline__ void load(const DistillArgs& a, int64_t at, int me)
    {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const int i = me + q * G;
            cls[q] = i < a.k ? list_class(a, at + i) : PLACE_ABSENT;
            v[q] = cls[q] >= 0 ? load_value(a.teacher, a.teacher_bf16, at + i) : -INFINITY;
        }
    }
};

template <typename T, int V, int G>
__global__ void __launch_bounds__(G == 32 ? 32 * WARP_ROWS : G) distill_row_kernel(const DistillArgs a)
{
    __shared__ float scratch_s[G > 32 ? 5 * (G / 32) : 1];
    extern __shared__ uint32_t bits_s[];             // a bit for every class in the list: (K + 31) / 32 words to a row
    const Group<G> group{scratch_s};
    const int64_t row = G == 32 ? blockIdx.x * (int64_t)WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.n) return;
    const int me = group.rank(), words = (a.K + 31) / 32;
    uint32_t* bits = bits_s + (G == 32 ? (threadIdx.x >> 5) * words : 0);
    const T* x = (const T*)a.logits + row * a.ld;
    ListPart<G> list;
    list.load(a, row * a.k, me);
    if (a.rest) {
        for (int w = me; w < words; w += G) bits[w] = 0;
        group.sync();
#pragma unroll
        for (int q = 0; q < ListPart<G>::N; ++q)
            if (list.cls[q] >= 0) atomicOr(&bits[list.cls[q] >> 5], 1u << (list.cls[q] & 31));
        group.sync();
    }
    float m = -INFINITY;
    for (int p = me; p * V < a.K; p += G) {
        float v[V];
        load_piece<T, V>(x, p, a.K, v);
#pragma unroll
        for (int i = 0; i < V; ++i) m = max_nan(m, v[i]);
    }
    m = group.max(m);
    const float origin = row_origin(m), c = a.inv_t * LOG2E;
    float out_max = -INFINITY, sums[2] = {0.f, 0.f};
    for (int p = me; p * V < a.K; p += G) {
        float v[V];
        load_piece<T, V>(x, p, a.K, v);
        const uint32_t in = a.rest ? bits[p * V >> 5] >> (p * V & 31) : 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float e = fast_exp2(below_max(v[i], origin) * c);
            sums[0] += e;
            if (a.rest && !(in >> i & 1)) {
                sums[1] += e;
                out_max = max_nan(out_max, v[i]);
            }
        }
    }
    group.sum(sums);
    const bool none = sums[0] == 0.f;
    const float log_s = none ? -INFINITY : log1pf(sums[0] - 1.f);
    float log_out = -INFINITY;
    if (a.rest) {
        out_max = group.max(out_max);
        if (out_max != -INFINITY) {
            if (sums[1] >= REST_TOO_SMALL || sums[1] != sums[1]) {
                log_out = logf(sums[1]);
            } else {
                float again[1] = {0.f};
                for (int j = me; j < a.K; j += G)
                    if (!(bits[j >> 5] >> (j & 31) & 1)) again[0] += fast_exp2(below_max(to_f<T>(x[j]), out_max) * c);
                group.sum(again);
                log_out = (out_max - origin) * a.inv_t + logf(again[0]);
            }
        }
    }
    // the list
    float top = -INFINITY;
    bool any = false, bad = false;
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q) {
        any |= list.cls[q] >= 0;
        bad |= list.cls[q] == PLACE_BAD;
        top = max_nan(top, list.v[q]);
    }
    top = group.max(top);
    const ListSums l{top, 0.f, false, false};
    // sum of t, entries, bad ones, entries that are as large as the largest
    float ls[4] = {0.f, any ? 1.f : 0.f, bad ? 1.f : 0.f, 0.f};
    float t[ListPart<G>::N];
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q) {
        t[q] = list.cls[q] >= 0 ? l.prob(list.v[q], a.rest, a.inv_t) : 0.f;
        const bool is_top = list.cls[q] >= 0 && list.v[q] == top;
        ls[0] += a.rest && is_top ? 0.f : t[q];
        ls[3] += is_top ? 1.f : 0.f;
    }
    group.sum(ls);
    float scale = 1.f, log_scale = 0.f, t_r = 0.f;
    if (!a.rest) {
        scale = ls[0] > 0.f ? __fdiv_rn(1.f, ls[0]) : ls[0];
        log_scale = ls[0] > 0.f ? logf(ls[0]) : 0.f;
    } else if (ls[1] > 0.f && log_out != -INFINITY) {
        t_r = rest_prob(top, ls[0] + (ls[3] - 1.f) * fast_exp2(top * LOG2E));
    }
    float loss[1] = {0.f};
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q) {
        if (list.cls[q] >= 0) {
            const float log_t = a.rest ? list.v[q] : below_max(list.v[q], row_origin(top)) * a.inv_t - log_scale;
            const float log_p = none ? -INFINITY : (to_f<T>(x[list.cls[q]]) - origin) * a.inv_t - log_s;
            loss[0] += entry_loss(t[q] * scale, log_t, log_p);
        }
    }
    group.sum(loss);
    if (me == 0) {
        if (a.rest) loss[0] += entry_loss(t_r, logf(t_r), log_out - log_s);
        if (ls[2] > 0.f) {
            loss[0] = NAN;
            atomicOr(a.status, PTV3_STATUS_BAD_INDEX);
        }
        a.loss[row] = loss[0];
        if (a.stats) a.stats[row] = a.rest ? make_float4(origin, log_s, log_out, t_r) : make_float4(origin, log_s, row_origin(top), scale);
    }
}

// ---- gradient -------------------------------------------------------------------------------------------------------------
struct DistillGrad {
    float m, c, shift, factor, inside_shift, inside_factor, g;
    bool none;
    // every class as one outside the list
    __device__ __forceinline__ float at(float x) const { return fast_exp2(fmaf(below_max(x, m), c, shift)) * factor; }
    // M p of a class in the list
    __device__ __forceinline__ float in_list(float x) const { return fast_exp2(fmaf(below_max(x, m), c, inside_shift)) * inside_factor; }
};
// mass: sum of the list's t
__device__ __forceinline__ DistillGrad distill_grad(const DistillArgs& a, int64_t row, float4 st, float mass)
{
    DistillGrad r;
    r.m = st.x;
    r.c = a.inv_t * LOG2E;
    r.none = st.y == -INFINITY;
    r.g = r.none ? 0.f : a.g[row * a.g_step] * a.inv_t;
    const float log_s = r.none ? INFINITY : st.y;
    r.inside_shift = r.shift = -log_s * LOG2E;
    r.inside_factor = r.factor = mass * r.g;
    if (a.rest && st.z != -INFINITY) {
        // p_j / p_r (M p_r - t_r)
        const float M = mass + st.w;
        r.inside_factor = M * r.g;
        r.shift = r.none ? -INFINITY : -st.z * LOG2E;
        r.factor = r.g * (M * fast_exp2((st.z - log_s) * LOG2E) - st.w);
    }
    return r;
}
// t of an entry from the row's stats
__device__ __forceinline__ float entry_prob(const DistillArgs& a, float4 st, float v)
{
    return a.rest ? fast_exp2(v * LOG2E) : fast_exp2(below_max(v, st.z) * (a.inv_t * LOG2E)) * st.w;
}

template <typename T>
__global__ void __launch_bounds__(TILE_ROWS) distill_tile_bwd_kernel(const DistillArgs a)
{
    extern __shared__ __align__(16) float tile[];
    const int64_t row0 = blockIdx.x * (int64_t)TILE_ROWS;
    const int rows = (int)min((int64_t)TILE_ROWS, a.n - row0);
    load_tile(tile, (const T*)a.logits, a.ld, row0, rows, a.K);
    __syncthreads();
    if ((int)threadIdx.x < rows) {
        const int64_t row = row0 + threadIdx.x, at = row * a.k;
        float* x = tile + threadIdx.x * tile_pitch(a.K);
        const T* again = (const T*)a.logits + row * a.ld;
        const float4 st = a.stats[row];
        float mass = 0.f;
        for (int i = 0; i < a.k; ++i)
            if (list_class(a, at + i) >= 0) mass += entry_prob(a, st, load_value(a.teacher, a.teacher_bf16, at + i));
        const DistillGrad r = distill_grad(a, row, st, mass);
        for (int j = 0; j < a.K; ++j) x[j] = r.at(x[j]);
        if (a.rest)
            for (int i = 0; i < a.k; ++i) {
                const int cls = list_class(a, at + i);
                if (cls >= 0) x[cls] = r.in_list(to_f<T>(again[cls]));
            }
        for (int i = 0; i < a.k; ++i) {
            const int cls = list_class(a, at + i);
            if (cls >= 0) x[cls] -= r.g * entry_prob(a, st, load_value(a.teacher, a.teacher_bf16, at + i));
        }
    }
    __syncthreads();
    store_tile(tile, (T*)a.dlogits, row0, rows, a.K);
}

template <typename T, int V, int G>
__global__ void __launch_bounds__(G == 32 ? 32 * WARP_ROWS : G) distill_row_bwd_kernel(const DistillArgs a)
{
    __shared__ float scratch[G > 32 ? 3 * (G / 32) : 1];
    __shared__ int list_c[G == 32 ? WARP_ROWS : 1][LIST_MAX];
    __shared__ float list_t[G == 32 ? WARP_ROWS : 1][LIST_MAX];
    const Group<G> group{scratch};
    const int64_t row = G == 32 ? blockIdx.x * (int64_t)WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.n) return;
    const int me = group.rank(), slot = G == 32 ? threadIdx.x >> 5 : 0;
    const T* x = (const T*)a.logits + row * a.ld;
    T* dx = (T*)a.dlogits + row * a.K;
    const float4 st = a.stats[row];
    ListPart<G> list;
    list.load(a, row * a.k, me);
    float mass[1] = {0.f};
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q) {
        const float t = list.cls[q] >= 0 ? entry_prob(a, st, list.v[q]) : 0.f;
        mass[0] += t;
        if (me + q * G < LIST_MAX) {
            list_c[slot][me + q * G] = list.cls[q];
            list_t[slot][me + q * G] = t;
        }
    }
    group.sum(mass);
    const DistillGrad r = distill_grad(a, row, st, mass[0]);
#pragma unroll 4
    for (int p = me; p * V < a.K; p += G) {
        float v[V];
        load_piece<T, V>(x, p, a.K, v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = r.at(v[i]);
        store_piece<T, V>(dx, p, a.K, v);
    }
    // the list's classes once more; one that comes twice is written by its first entry, with the sum of both
    group.sync();
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q) {
        const int mine = me + q * G, cls = list.cls[q];
        if (cls < 0) continue;
        float t = 0.f;
        bool is_first = true;
        for (int i = 0; i < a.k; ++i) {
            if (list_c[slot][i] == cls) {
                t += list_t[slot][i];
                is_first &= i >= mine;
            }
        }
        if (is_first) dx[cls] = from_f<T>(r.in_list(to_f<T>(x[cls])) - r.g * t);
    }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------
template <typename T, int V, int G>
static int launch_distill_rows(const DistillArgs& a, bool backward, cudaStream_t stream)
{
    const unsigned blocks = G == 32 ? (unsigned)((a.n + WARP_ROWS - 1) / WARP_ROWS) : (unsigned)a.n;
    const int threads = G == 32 ? 32 * WARP_ROWS : G;
    if (backward) {
        distill_row_bwd_kernel<T, V, G><<<blocks, threads, 0, stream>>>(a);
    } else {
        const size_t smem = a.rest ? (size_t)((a.K + 31) / 32) * 4 * (G == 32 ? WARP_ROWS : 1) : 0;
        distill_row_kernel<T, V, G><<<blocks, threads, smem, stream>>>(a);
    }
    return 0;
}

template <typename T>
static int launch_distill(const DistillArgs& a, bool backward, cudaStream_t stream)
{
    const bool wide = rows_aligned(a.logits, a.ld, a.K, sizeof(T)) && (!backward || ((uintptr_t)a.dlogits & 15) == 0);
    constexpr int V = Vec<T>::N;
    if (a.K <= SMALL_CLASSES) {
        const unsigned blocks = (unsigned)((a.n + TILE_ROWS - 1) / TILE_ROWS);
        const size_t smem = (size_t)TILE_ROWS * tile_pitch(a.K) * sizeof(float);
        if (backward)
            distill_tile_bwd_kernel<T><<<blocks, TILE_ROWS, smem, stream>>>(a);
        else
            distill_tile_kernel<T><<<blocks, TILE_ROWS, smem, stream>>>(a);
    } else if (a.K <= 1024) {
        wide ? launch_distill_rows<T, V, 32>(a, backward, stream) : launch_distill_rows<T, 1, 32>(a, backward, stream);
    } else {
        wide ? launch_distill_rows<T, V, 256>(a, backward, stream) : launch_distill_rows<T, 1, 256>(a, backward, stream);
    }
    count_launches(1);
    return check_launch(backward ? "ptv3_distill_topk_bwd" : "ptv3_distill_topk_fwd");
}

static int run_distill(const char* what, DistillArgs& a, int teacher_dtype, float temperature, int dtype, bool backward,
                       cudaStream_t stream)
{
    PTV3_REQUIRE(a.n >= 0 && a.n < (1ll << 31), PTV3_ERR_INVALID_ARGUMENT, "%s: n out of range", what);
    PTV3_REQUIRE((dtype == PTV3_DTYPE_F32 || dtype == PTV3_DTYPE_BF16) &&
                     (teacher_dtype == PTV3_DTYPE_F32 || teacher_dtype == PTV3_DTYPE_BF16),
                 PTV3_ERR_UNSUPPORTED, "%s: dtype %d, of the teacher %d", what, dtype, teacher_dtype);
    PTV3_REQUIRE(a.K >= 1 && a.K <= CLASSES_MAX, PTV3_ERR_UNSUPPORTED, "%s: %d classes (1..%d)", what, a.K, CLASSES_MAX);
    PTV3_REQUIRE(a.k >= 1 && a.k <= LIST_MAX, PTV3_ERR_UNSUPPORTED, "%s: lists of %d (1..%d)", what, a.k, LIST_MAX);
    PTV3_REQUIRE(a.ld >= a.K, PTV3_ERR_INVALID_ARGUMENT, "%s: rows of %d that are %lld apart", what, a.K, (long long)a.ld);
    PTV3_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, PTV3_ERR_INVALID_ARGUMENT, "%s: temperature out of range", what);
    PTV3_REQUIRE(a.list_bytes == 4 || a.list_bytes == 8, PTV3_ERR_INVALID_ARGUMENT, "%s: classes of %d bytes", what, a.list_bytes);
    const int size = dtype == PTV3_DTYPE_F32 ? 4 : 2, tsize = teacher_dtype == PTV3_DTYPE_F32 ? 4 : 2;
    PTV3_REQUIRE((uintptr_t)a.logits % size == 0 && (uintptr_t)a.dlogits % size == 0 && (uintptr_t)a.teacher % tsize == 0 &&
                     (uintptr_t)a.list % a.list_bytes == 0 && (uintptr_t)a.stats % 16 == 0,
                 PTV3_ERR_INVALID_ARGUMENT, "%s: unaligned tensor", what);
    a.inv_t = (float)(1.0 / temperature);
    a.teacher_bf16 = teacher_dtype == PTV3_DTYPE_BF16;
    if (a.n == 0) return PTV3_OK;
    PTV3_REQUIRE(a.logits && a.teacher && a.list && (backward ? a.stats && a.g && a.dlogits : a.loss && a.status),
                 PTV3_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    return dtype == PTV3_DTYPE_F32 ? launch_distill<float>(a, backward, stream) : launch_distill<__nv_bfloat16>(a, backward, stream);
}

}  // namespace ptv3

extern "C" int ptv3_distill_topk_fwd(const void* logits, int64_t ld, const void* teacher, int teacher_dtype, const void* list,
                                     int list_bytes, int k, float* loss, float* stats, int64_t n, int classes,
                                     float temperature, int rest, int dtype, uint32_t* status, void* stream)
{
    ptv3::DistillArgs a{};
    a.logits = logits;
    a.ld = ld;
    a.n = n;
    a.teacher = teacher;
    a.list = list;
    a.list_bytes = list_bytes;
    a.k = k;
    a.K = classes;
    a.rest = rest != 0;
    a.loss = loss;
    a.stats = (float4*)stats;
    a.status = status;
    return ptv3::run_distill("ptv3_distill_topk_fwd", a, teacher_dtype, temperature, dtype, false, (cudaStream_t)stream);
}

extern "C" int ptv3_distill_topk_bwd(const void* logits, int64_t ld, const void* teacher, int teacher_dtype, const void* list,
                                     int list_bytes, int k, const float* stats, const float* dloss, int64_t dloss_step,
                                     void* dlogits, int64_t n, int classes, float temperature, int rest, int dtype, void* stream)
{
    ptv3::DistillArgs a{};
    a.logits = logits;
    a.ld = ld;
    a.n = n;
    a.teacher = teacher;
    a.list = list;
    a.list_bytes = list_bytes;
    a.k = k;
    a.K = classes;
    a.rest = rest != 0;
    a.stats = (float4*)stats;
    a.g = dloss;
    a.g_step = dloss_step;
    a.dlogits = dlogits;
    return ptv3::run_distill("ptv3_distill_topk_bwd", a, teacher_dtype, temperature, dtype, true, (cudaStream_t)stream);
}
