// What a row of logits answers: the log probability of a given class, the entropy, the best alternatives, and the gradient
// of all three with respect to the logits.  No counterpart in the reference, whose file ends with the backbone
// (model.py:966-982); the formulas stand in class_rows.cuh and below.
//
//     H = log S - (1/S) sum e_j d_j / T,    e_j = exp(d_j / T), d_j = x_j - m
//     dx_j = 1/T ( p_j (A + B log p_j) + [j = label] g + sum_i [j = t_i] g_i ),   A = -(g + sum g_i) - h H,  B = -h
// with g, h, g_i the gradients of the three.
#include "class_rows.cuh"

namespace ptv3 {

struct ScoresArgs {
    const void* logits;      // n rows of K, ld apart
    int64_t ld, n;
    const void* labels;      // n integers or NULL
    int label_bytes;
    int64_t ignore;
    float *logp, *entropy;   // n
    float* top_logp;         // n x top
    int32_t* top_class;
    float2* stats;           // n x {m, log S} or NULL
    int K, top;
    float inv_t;
    uint32_t* status;
    // backward
    const float *g_logp, *g_entropy;     // steps g_logp_step, g_entropy_step apart (0: one value for all), or NULL
    int64_t g_logp_step, g_entropy_step;
    const float* g_top;                  // n x top or NULL
    void* dlogits;                       // n x K
};

struct RowSums {
    float m, log_s, entropy;   // m: what was taken out; log_s: minus infinity for a row without a class
    bool none;
};
// S, U = sum e d -> log S and the entropy
__device__ __forceinline__ RowSums row_sums(float m, float s, float u, float inv_t)
{
    RowSums r;
    r.m = row_origin(m);
    r.none = s == 0.f;
    r.log_s = r.none ? -INFINITY : log1pf(s - 1.f);
    r.entropy = r.none ? 0.f : r.log_s - __fdiv_rn(u * inv_t, s);
    return r;
}
__device__ __forceinline__ float log_prob_of(const RowSums& r, float x, float inv_t)
{
    return r.none ? -INFINITY : (x - r.m) * inv_t - r.log_s;
}

// The label's log probability: 0 for a row without a label, NaN and a status bit for one that is no class.
template <typename F>
__device__ __forceinline__ void write_row(const ScoresArgs& a, int64_t row, const RowSums& r, F&& logit)
{
    if (a.logp) {
        const int64_t label = load_index(a.labels, a.label_bytes, row);
        float lp = 0.f;
        if (label != a.ignore) {
            const bool is = label >= 0 && label < a.K;
            lp = is ? log_prob_of(r, logit((int)label), a.inv_t) : NAN;
            if (!is) atomicOr(a.status, PTV3_STATUS_BAD_INDEX);
        }
        a.logp[row] = lp;
    }
    if (a.entropy) a.entropy[row] = r.entropy;
    if (a.stats) a.stats[row] = make_float2(r.m, r.log_s);
}

// ---- the best classes, kept sorted in registers while a thread reads its row in order --------------------------------
// bf16 logits and classes below 2^16 share a word, value above (inverted) class: a step of the insertion is a maximum and a
// minimum.  Otherwise the classes move with the keys; equal keys stay in the order they come in, lowest class first.
template <int TOP, bool PACKED>
struct TopList {
    uint32_t key[TOP > 0 ? TOP : 1];
    int cls[TOP > 0 && !PACKED ? TOP : 1];
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < TOP; ++i) {
            key[i] = 0;
            if (!PACKED) cls[i] = -1;
        }
    }
    __device__ __forceinline__ void insert(float x, int j)
    {
        uint32_t k = order_key(x);
        if (PACKED) {
            k = (k & 0xffff0000u) | (0xffffu - j);
#pragma unroll
            for (int i = 0; i < TOP; ++i) {
                const uint32_t hi = ::max(key[i], k);
                k = ::min(key[i], k);
                key[i] = hi;
            }
        } else {
            bool up = false;     // from the first smaller key on, everything moves
#pragma unroll
            for (int i = 0; i < TOP; ++i) {
                up |= k > key[i];
                const uint32_t k2 = up ? key[i] : k;
                const int j2 = up ? cls[i] : j;
                key[i] = up ? k : key[i];
                cls[i] = up ? j : cls[i];
                k = k2;
                j = j2;
            }
        }
    }
    __device__ __forceinline__ int at(int i) const
    {
        if (!PACKED) return cls[i];
        return key[i] ? (int)(0xffffu - (key[i] & 0xffffu)) : -1;
    }
};

// ---- up to SMALL_CLASSES classes: a tile of rows, one thread to a row -------------------------------------------------
template <typename T, int TOP>
__global__ void __launch_bounds__(TILE_ROWS) scores_tile_kernel(const ScoresArgs a)
{
    extern __shared__ __align__(16) float tile[];
    const int64_t row0 = blockIdx.x * (int64_t)TILE_ROWS;
    const int rows = (int)min((int64_t)TILE_ROWS, a.n - row0);
    load_tile(tile, (const T*)a.logits, a.ld, row0, rows, a.K);
    __syncthreads();
    if ((int)threadIdx.x >= rows) return;
    const float* x = tile + threadIdx.x * tile_pitch(a.K);
    const int64_t row = row0 + threadIdx.x;
    TopList<TOP, sizeof(T) == 2> best;
    best.clear();
    float m = -INFINITY;
    for (int j = 0; j < a.K; ++j) {
        m = max_nan(m, x[j]);
        if (TOP) best.insert(x[j], j);
    }
    const float origin = row_origin(m), c = a.inv_t * LOG2E;
    float s = 0.f, u = 0.f;
    for (int j = 0; j < a.K; ++j) {
        const float d = below_max(x[j], origin), e = fast_exp2(d * c);
        s += e;
        u = fmaf(e, d, u);
    }
    const RowSums r = row_sums(m, s, u, a.inv_t);
    write_row(a, row, r, [&](int j) { return x[j]; });
#pragma unroll
    for (int i = 0; i < TOP; ++i) {
        if (i < a.top) {
            const int cls = best.at(i);
            a.top_class[row * a.top + i] = cls;
            a.top_logp[row * a.top + i] = cls < 0 ? -INFINITY : log_prob_of(r, x[cls], a.inv_t);
        }
    }
}

// ---- more classes: G threads to a row -----------------------------------------------------------------------------------
// The row's values stay in registers, E of each thread; rows beyond G x 32 are read again for every sum (E = 0).
constexpr int WARP_ROWS = 4;    // warps of a block where a warp has a row

template <typename T, int V, int G, int E>
struct RowValues {
    static constexpr int P = E / V;
    float v[E > 0 ? P : 1][V];
    const T* row;
    int K, rank;
    __device__ __forceinline__ void load(const T* r, int k, int me)
    {
        row = r;
        K = k;
        rank = me;
        if (E > 0) {
#pragma unroll
            for (int p = 0; p < P; ++p) load_piece<T, V>(row, p * G + rank, K, v[p]);
        }
    }
    // f(value, class), classes ascending; those of no class are minus infinity
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const
    {
        if (E > 0) {
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int i = 0; i < V; ++i) f(v[p][i], (p * G + rank) * V + i);
        } else {
            for (int p = rank; p * V < K; p += G) {
                float w[V];
                load_piece<T, V>(row, p, K, w);
#pragma unroll
                for (int i = 0; i < V; ++i) f(w[i], p * V + i);
            }
        }
    }
};

template <typename T, int V, int G, int E>
__global__ void __launch_bounds__(G == 32 ? 32 * WARP_ROWS : G) scores_row_kernel(const ScoresArgs a)
{
    __shared__ float scratch[G > 32 ? 3 * (G / 32) : 1];
    __shared__ unsigned long long chosen[G > 32 ? G / 32 : 1];
    const Group<G> group{scratch};
    const int64_t row = G == 32 ? blockIdx.x * (int64_t)WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.n) return;
    const int me = group.rank();
    const T* x = (const T*)a.logits + row * a.ld;
    RowValues<T, V, G, E> vals;
    vals.load(x, a.K, me);
    float m = -INFINITY;
    vals.each([&](float v, int) { m = max_nan(m, v); });
    m = group.max(m);
    const float origin = row_origin(m), c = a.inv_t * LOG2E;
    float su[2] = {0.f, 0.f};
    vals.each([&](float v, int) {
        const float d = below_max(v, origin), e = fast_exp2(d * c);
        su[0] += e;
        su[1] = fmaf(e, d, su[1]);
    });
    group.sum(su);
    const RowSums r = row_sums(m, su[0], su[1], a.inv_t);
    if (me == 0) write_row(a, row, r, [&](int j) { return to_f<T>(x[j]); });

    // one alternative after another: the largest of (key, lowest class) behind the last one
    uint32_t last_key = 0xffffffffu;
    int last_class = -1;
    uint32_t key = 0;
    int cls = 0x7fffffff;
    bool again = true;
    for (int i = 0; i < a.top; ++i) {
        if (again) {
            key = 0;
            cls = 0x7fffffff;
            vals.each([&](float v, int j) {
                const uint32_t k = order_key(v);
                const bool left = j < a.K && (k < last_key || (k == last_key && j > last_class));
                if (left && k > key) {
                    key = k;
                    cls = j;
                }
            });
        }
        uint32_t k = __reduce_max_sync(~0u, key);
        int j = (int)__reduce_min_sync(~0u, key == k ? (uint32_t)cls : 0x7fffffffu);
        if (G > 32) {
            __syncthreads();
            if ((threadIdx.x & 31) == 0) chosen[threadIdx.x >> 5] = (unsigned long long)k << 32 | (0x7fffffffu - j);
            __syncthreads();
            unsigned long long best = chosen[0];
#pragma unroll
            for (int w = 1; w < G / 32; ++w) best = best > chosen[w] ? best : chosen[w];
            k = (uint32_t)(best >> 32);
            j = (int)(0x7fffffffu - (uint32_t)best);
        }
        again = j == cls;
        last_key = k;
        last_class = j;
        if (me == 0) {
            a.top_class[row * a.top + i] = k ? j : -1;
            a.top_logp[row * a.top + i] = k ? log_prob_of(r, order_value(k), a.inv_t) : -INFINITY;
        }
    }
}

// ---- gradient -------------------------------------------------------------------------------------------------------------
struct RowGrad {
    float m, log_s, A, B, g, inv_t;
    int label;
    // without the alternatives' own parts
    __device__ __forceinline__ float at(float x, int j) const
    {
        const float d = below_max(x, m);
        const float p = fast_exp2(fmaf(d, inv_t * LOG2E, -log_s * LOG2E));
        float v = p * (B != 0.f && p > 0.f ? fmaf(B, fmaf(d, inv_t, -log_s), A) : A);
        if (j == label) v += g;
        return v * inv_t;
    }
};
__device__ __forceinline__ RowGrad row_grad(const ScoresArgs& a, int64_t row, float g_top_sum, bool& none)
{
    RowGrad r;
    const float2 st = a.stats[row];
    none = st.y == -INFINITY;
    r.m = st.x;
    r.log_s = none ? INFINITY : st.y;
    r.inv_t = a.inv_t;
    r.label = -1;
    r.g = 0.f;
    if (a.g_logp) {
        const int64_t label = load_index(a.labels, a.label_bytes, row);
        if (label != a.ignore && label >= 0 && label < a.K) {
            r.label = (int)label;
            r.g = a.g_logp[row * a.g_logp_step];
        }
    }
    const float h = a.g_entropy ? a.g_entropy[row * a.g_entropy_step] : 0.f;
    r.A = -(r.g + g_top_sum) - (a.g_entropy ? h * a.entropy[row] : 0.f);
    r.B = -h;
    if (none) {
        r.A = r.B = r.g = 0.f;
        r.label = -1;
    }
    return r;
}

template <typename T>
__global__ void __launch_bounds__(TILE_ROWS) scores_tile_bwd_kernel(const ScoresArgs a)
{
    extern __shared__ __align__(16) float tile[];
    const int64_t row0 = blockIdx.x * (int64_t)TILE_ROWS;
    const int rows = (int)min((int64_t)TILE_ROWS, a.n - row0);
    load_tile(tile, (const T*)a.logits, a.ld, row0, rows, a.K);
    __syncthreads();
    if ((int)threadIdx.x < rows) {
        const int64_t row = row0 + threadIdx.x;
        float* x = tile + threadIdx.x * tile_pitch(a.K);
        const float* gt = a.g_top ? a.g_top + row * a.top : nullptr;
        const int32_t* tc = a.g_top ? a.top_class + row * a.top : nullptr;
        float g_sum = 0.f;
        if (gt)
            for (int i = 0; i < a.top; ++i) g_sum += tc[i] >= 0 ? gt[i] : 0.f;
        bool none;
        const RowGrad r = row_grad(a, row, g_sum, none);
        for (int j = 0; j < a.K; ++j) x[j] = r.at(x[j], j);
        if (gt && !none)
            for (int i = 0; i < a.top; ++i)
                if (tc[i] >= 0) x[tc[i]] += gt[i] * a.inv_t;
    }
    __syncthreads();
    store_tile(tile, (T*)a.dlogits, row0, rows, a.K);
}

template <typename T, int V, int G>
__global__ void __launch_bounds__(G == 32 ? 32 * WARP_ROWS : G) scores_row_bwd_kernel(const ScoresArgs a)
{
    __shared__ float scratch[G > 32 ? 3 * (G / 32) : 1];
    const Group<G> group{scratch};
    const int64_t row = G == 32 ? blockIdx.x * (int64_t)WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.n) return;
    const int me = group.rank();
    const T* x = (const T*)a.logits + row * a.ld;
    T* dx = (T*)a.dlogits + row * a.K;
    const float* gt = a.g_top ? a.g_top + row * a.top : nullptr;
    const int32_t* tc = a.g_top ? a.top_class + row * a.top : nullptr;
    float g_sum[1] = {0.f};
    if (gt) {
        for (int i = me; i < a.top; i += G) g_sum[0] += tc[i] >= 0 ? gt[i] : 0.f;
        group.sum(g_sum);
    }
    bool none;
    const RowGrad r = row_grad(a, row, g_sum[0], none);
#pragma unroll 4
    for (int p = me; p * V < a.K; p += G) {
        float v[V];
        load_piece<T, V>(x, p, a.K, v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = r.at(v[i], p * V + i);
        store_piece<T, V>(dx, p, a.K, v);
    }
    if (gt && !none) {
        // the alternatives once more, with their own parts
        group.sync();
        for (int i = me; i < a.top; i += G)
            if (tc[i] >= 0) dx[tc[i]] = from_f<T>(fmaf(gt[i], a.inv_t, r.at(to_f<T>(x[tc[i]]), tc[i])));
    }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------
template <typename T>
static void launch_tile(const ScoresArgs& a, cudaStream_t stream)
{
    const unsigned blocks = (unsigned)((a.n + TILE_ROWS - 1) / TILE_ROWS);
    const size_t smem = (size_t)TILE_ROWS * tile_pitch(a.K) * sizeof(float);
    if (a.top == 0)
        scores_tile_kernel<T, 0><<<blocks, TILE_ROWS, smem, stream>>>(a);
    else if (a.top <= 4)
        scores_tile_kernel<T, 4><<<blocks, TILE_ROWS, smem, stream>>>(a);
    else if (a.top <= 8)
        scores_tile_kernel<T, 8><<<blocks, TILE_ROWS, smem, stream>>>(a);
    else if (a.top <= 16)
        scores_tile_kernel<T, 16><<<blocks, TILE_ROWS, smem, stream>>>(a);
    else if (a.top <= 32)
        scores_tile_kernel<T, 32><<<blocks, TILE_ROWS, smem, stream>>>(a);
    else
        scores_tile_kernel<T, 64><<<blocks, TILE_ROWS, smem, stream>>>(a);
}

template <typename T, int V>
static void launch_rows(const ScoresArgs& a, cudaStream_t stream)
{
    const unsigned warps = (unsigned)((a.n + WARP_ROWS - 1) / WARP_ROWS), rows = (unsigned)a.n;
    if (a.K <= 256)
        scores_row_kernel<T, V, 32, 8><<<warps, 32 * WARP_ROWS, 0, stream>>>(a);
    else if (a.K <= 512)
        scores_row_kernel<T, V, 32, 16><<<warps, 32 * WARP_ROWS, 0, stream>>>(a);
    else if (a.K <= 1024)
        scores_row_kernel<T, V, 32, 32><<<warps, 32 * WARP_ROWS, 0, stream>>>(a);
    else if (a.K <= 2048)
        scores_row_kernel<T, V, 256, 8><<<rows, 256, 0, stream>>>(a);
    else if (a.K <= 4096)
        scores_row_kernel<T, V, 256, 16><<<rows, 256, 0, stream>>>(a);
    else if (a.K <= 8192)
        scores_row_kernel<T, V, 256, 32><<<rows, 256, 0, stream>>>(a);
    else
        scores_row_kernel<T, V, 256, 0><<<rows, 256, 0, stream>>>(a);
}

template <typename T, int V>
static void launch_rows_bwd(const ScoresArgs& a, cudaStream_t stream)
{
    if (a.K <= 1024)
        scores_row_bwd_kernel<T, V, 32><<<(unsigned)((a.n + WARP_ROWS - 1) / WARP_ROWS), 32 * WARP_ROWS, 0, stream>>>(a);
    else
        scores_row_bwd_kernel<T, V, 256><<<(unsigned)a.n, 256, 0, stream>>>(a);
}

template <typename T>
static int launch_scores(const ScoresArgs& a, bool backward, cudaStream_t stream)
{
    const bool wide = rows_aligned(a.logits, a.ld, a.K, sizeof(T)) && (!backward || ((uintptr_t)a.dlogits & 15) == 0);
    if (backward) {
        if (a.K <= SMALL_CLASSES)
            scores_tile_bwd_kernel<T><<<(unsigned)((a.n + TILE_ROWS - 1) / TILE_ROWS), TILE_ROWS,
                                        (size_t)TILE_ROWS * tile_pitch(a.K) * sizeof(float), stream>>>(a);
        else if (wide)
            launch_rows_bwd<T, Vec<T>::N>(a, stream);
        else
            launch_rows_bwd<T, 1>(a, stream);
    } else if (a.K <= SMALL_CLASSES) {
        launch_tile<T>(a, stream);
    } else if (wide) {
        launch_rows<T, Vec<T>::N>(a, stream);
    } else {
        launch_rows<T, 1>(a, stream);
    }
    count_launches(1);
    return check_launch(backward ? "ptv3_class_scores_bwd" : "ptv3_class_scores_fwd");
}

static int check_scores(const char* what, const ScoresArgs& a, float temperature, int dtype)
{
    PTV3_REQUIRE(a.n >= 0 && a.n < (1ll << 31), PTV3_ERR_INVALID_ARGUMENT, "%s: n out of range", what);
    PTV3_REQUIRE(dtype == PTV3_DTYPE_F32 || dtype == PTV3_DTYPE_BF16, PTV3_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
    PTV3_REQUIRE(a.K >= 1 && a.K <= CLASSES_MAX, PTV3_ERR_UNSUPPORTED, "%s: %d classes (1..%d)", what, a.K, CLASSES_MAX);
    PTV3_REQUIRE(a.top >= 0 && a.top <= LIST_MAX, PTV3_ERR_UNSUPPORTED, "%s: %d alternatives (0..%d)", what, a.top, LIST_MAX);
    PTV3_REQUIRE(a.ld >= a.K, PTV3_ERR_INVALID_ARGUMENT, "%s: rows of %d that are %lld apart", what, a.K, (long long)a.ld);
    PTV3_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, PTV3_ERR_INVALID_ARGUMENT, "%s: temperature out of range", what);
    const int size = dtype == PTV3_DTYPE_F32 ? 4 : 2;
    PTV3_REQUIRE((uintptr_t)a.logits % size == 0 && (uintptr_t)a.dlogits % size == 0, PTV3_ERR_INVALID_ARGUMENT, "%s: unaligned logits", what);
    PTV3_REQUIRE(a.label_bytes == 4 || a.label_bytes == 8 || !a.labels, PTV3_ERR_INVALID_ARGUMENT, "%s: labels of %d bytes", what, a.label_bytes);
    return PTV3_OK;
}

}  // namespace ptv3

extern "C" int ptv3_class_scores_fwd(const void* logits, int64_t ld, const void* labels, int label_bytes, int64_t ignore,
                                     float* log_prob, float* entropy, float* top_log_prob, int32_t* top_class, float* stats,
                                     int64_t n, int classes, int top, float temperature, int dtype, uint32_t* status,
                                     void* stream)
{
    using namespace ptv3;
    const char* what = "ptv3_class_scores_fwd";
    ScoresArgs a{};
    a.logits = logits;
    a.ld = ld;
    a.n = n;
    a.labels = labels;
    a.label_bytes = label_bytes;
    a.ignore = ignore;
    a.logp = log_prob;
    a.entropy = entropy;
    a.top_logp = top_log_prob;
    a.top_class = top_class;
    a.stats = (float2*)stats;
    a.K = classes;
    a.top = top;
    a.inv_t = (float)(1.0 / temperature);
    a.status = status;
    const int rc = check_scores(what, a, temperature, dtype);
    if (rc) return rc;
    if (n == 0) return PTV3_OK;
    PTV3_REQUIRE(logits && (status || !log_prob) && (entropy || log_prob || top), PTV3_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    PTV3_REQUIRE(!log_prob || labels, PTV3_ERR_INVALID_ARGUMENT, "%s: log_prob without labels", what);
    PTV3_REQUIRE(top == 0 || (top_log_prob && top_class), PTV3_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    PTV3_REQUIRE(((uintptr_t)stats & 7) == 0, PTV3_ERR_INVALID_ARGUMENT, "%s: unaligned stats", what);
    return dtype == PTV3_DTYPE_F32 ? launch_scores<float>(a, false, (cudaStream_t)stream)
                                   : launch_scores<__nv_bfloat16>(a, false, (cudaStream_t)stream);
}

extern "C" int ptv3_class_scores_bwd(const void* logits, int64_t ld, const void* labels, int label_bytes, int64_t ignore,
                                     const float* entropy, const int32_t* top_class, const float* stats,
                                     const float* dlog_prob, int64_t dlog_prob_step, const float* dentropy,
                                     int64_t dentropy_step, const float* dtop, void* dlogits, int64_t n, int classes,
                                     int top, float temperature, int dtype, void* stream)
{
    using namespace ptv3;
    const char* what = "ptv3_class_scores_bwd";
    ScoresArgs a{};
    a.logits = logits;
    a.ld = ld;
    a.n = n;
    a.labels = labels;
    a.label_bytes = label_bytes;
    a.ignore = ignore;
    a.entropy = const_cast<float*>(entropy);
    a.top_class = const_cast<int32_t*>(top_class);
    a.stats = (float2*)stats;
    a.K = classes;
    a.top = top;
    a.inv_t = (float)(1.0 / temperature);
    a.g_logp = dlog_prob;
    a.g_logp_step = dlog_prob_step;
    a.g_entropy = dentropy;
    a.g_entropy_step = dentropy_step;
    a.g_top = top ? dtop : nullptr;
    a.dlogits = dlogits;
    const int rc = check_scores(what, a, temperature, dtype);
    if (rc) return rc;
    if (n == 0) return PTV3_OK;
    PTV3_REQUIRE(logits && stats && dlogits && (!dentropy || entropy) && (!dlog_prob || labels) && (!a.g_top || top_class),
                 PTV3_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    PTV3_REQUIRE(((uintptr_t)stats & 7) == 0, PTV3_ERR_INVALID_ARGUMENT, "%s: unaligned stats", what);
    return dtype == PTV3_DTYPE_F32 ? launch_scores<float>(a, true, (cudaStream_t)stream)
                                   : launch_scores<__nv_bfloat16>(a, true, (cudaStream_t)stream);
}
