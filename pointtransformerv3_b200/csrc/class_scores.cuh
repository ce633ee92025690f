// What the kernels that answer from logits share: their arguments, a row's answers from its sums.
#pragma once
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
    float4* stats;           // n x {m, log S, entropy, -} or NULL
    int K, top;
    float inv_t;
    bool wide, wide_out;     // logits, gradient: see RowTile::wide_rows
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
constexpr float LN2 = 0.693147180559945309f;
// S, U = sum e t -> log S and the entropy (__fdividef: two units in the last place of a quotient that is as exact as S and U)
__device__ __forceinline__ RowSums row_sums(float m, float s, float u)
{
    RowSums r;
    r.m = row_origin(m);
    r.none = s == 0.f;
    r.log_s = r.none ? -INFINITY : log1pf(s - 1.f);
    r.entropy = r.none ? 0.f : r.log_s - __fdividef(u * LN2, s);
    return r;
}
__device__ __forceinline__ float log_prob_of(const RowSums& r, float x, float inv_t)
{
    return r.none ? -INFINITY : (x - r.m) * inv_t - r.log_s;
}

// A row's label, read before the row is there: its class, NO_LABEL or BAD_LABEL.
constexpr int NO_LABEL = -1, BAD_LABEL = -2;
__device__ __forceinline__ int row_label(const ScoresArgs& a, int64_t row)
{
    if (!a.labels) return NO_LABEL;
    const int64_t label = load_index(a.labels, a.label_bytes, row);
    return label == a.ignore ? NO_LABEL : (label >= 0 && label < a.K ? (int)label : BAD_LABEL);
}
// The label's log probability is 0 for a row without one, NaN with a status bit for one that is no class.  x: the label's logit
__device__ __forceinline__ void write_row(const ScoresArgs& a, int64_t row, const RowSums& r, int label, float x)
{
    if (a.logp) {
        a.logp[row] = label >= 0 ? log_prob_of(r, x, a.inv_t) : (label == NO_LABEL ? 0.f : NAN);
        if (label == BAD_LABEL) atomicOr(a.status, PTV3_STATUS_BAD_INDEX);
    }
    if (a.entropy) a.entropy[row] = r.entropy;
    if (a.stats) a.stats[row] = make_float4(r.m, r.log_s, r.entropy, 0.f);
}

// A row's alternatives out, get(i) the i-th (i < TOP): as wide as lists are aligned.  (Through shared memory, so that a warp's stores are
// neighbours, they took as long or longer: 407 678 x 20 with 5 alternatives 20.4 us instead of 16.4, with 8 to 64 classes 12.4 and 13.9.)
template <int TOP, typename V, typename F>
__device__ __forceinline__ void write_list(V* out, int top, bool wide, F&& get)
{
    if (TOP >= 4 && wide) {
#pragma unroll
        for (int i = 0; i + 3 < TOP; i += 4) {
            if (i < top) {
                const V v[4] = {get(i), get(i + 1), get(i + 2), get(i + 3)};
                *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(v);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < TOP; ++i)
            if (i < top) out[i] = get(i);
    }
}
__device__ __forceinline__ bool wide_lists(const ScoresArgs& a)
{
    return a.top % 4 == 0 && (((uintptr_t)a.top_logp | (uintptr_t)a.top_class) & 15) == 0;
}

}  // namespace ptv3
