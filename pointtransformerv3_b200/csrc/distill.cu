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
    bool teacher_bf16, list4;     // list4: see RowList
    bool wide, wide_out;          // logits, gradient: see RowTile::wide_rows
    float* loss;              // n
    float4* stats;            // n x {m, log S, log of the outside's sum or the list's largest, M p_r - t_r or 1 / the list's sum}, or NULL
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

// t_r = 1 - sum t: of one large and other small entries the large one's part is taken by expm1
__device__ __forceinline__ float rest_prob(float top, float others) { return fmaxf(-expm1f(fminf(top, 0.f)) - others, 0.f); }

// a list entry as it comes: the teacher's probability before its sum is known
__device__ __forceinline__ float entry_weight(const DistillArgs& a, float v, float top)
{
    return a.rest ? fast_exp2(v * LOG2E) : fast_exp2(below_max(v, row_origin(top)) * (a.inv_t * LOG2E));
}
// What a row's list adds up to: weights w (t itself, or t times their sum W), the largest value.
struct ListSums {
    float top, sum, others;      // others: W without the largest
};
// t (log t - log p) of an entry.  The three logarithms are subtracted from one another entry by entry, and not as sums over the list: near a student
// that has learnt its teacher they nearly cancel.  z: the student's logit from the origin, at the temperature
__device__ __forceinline__ float entry_term(const DistillArgs& a, float w, float scale, float log_sum, float v, float top, float z, float log_s)
{
    const float log_t = a.rest ? v : below_max(v, row_origin(top)) * a.inv_t - log_sum;
    return w == 0.f ? 0.f : w * scale * (log_t - (z - log_s));
}
// The outcome for the rest, from the teacher's t_r, the list's sum and the student's sums inside and outside (far_log: log p_r of an outside that had
// to be summed from its own maximum, or 0).  What is near 1 is taken from what is missing to it: a list that holds a hundredth of both
// teacher and student leaves differences of hundredths.  logf is the fast one of the compiler's flag, off by 2^-21 near 1 and by 3 units in the last
// place elsewhere: here its argument is at most a half, and for far_log what it adds to is beyond 46 in size.
struct Rest {
    float term;          // t_r (log t_r - log p_r)
    float surplus;       // M p_r - t_r = W - M (1 - p_r)
    float log_out;       // log of the outside's sum
    __device__ __forceinline__ Rest(float t_r, float W, float inside, float outside, float far_log, float log_s)
    {
        const float M = W + t_r, p_in = __fdividef(inside, inside + outside);
        const bool small = p_in < 0.5f;
        const float log_near = log1pf(small ? -p_in : __fdividef(inside, outside));        // (one call for both)
        const float log_p = far_log != 0.f ? far_log : (small ? log_near : -log_near);
        const float log_t = W < 0.5f ? log1pf(-W) : logf(t_r);
        term = t_r == 0.f ? 0.f : t_r * (log_t - log_p);
        surplus = small ? W - M * p_in : M * fast_exp2(log_p * LOG2E) - t_r;
        log_out = log_s + log_p;
    }
};

// ---- short rows: a tile of rows, one thread to a row ---------------------------------------------------------------
// A row's list in its thread's registers (N entries; N = 0: read from memory wherever it is walked).
template <int N>
struct RowList {
    int c[N > 0 ? N : 1];
    float v[N > 0 ? N : 1];
    const DistillArgs& a;
    int64_t at;
    __device__ __forceinline__ RowList(const DistillArgs& args, int64_t row) : a(args), at(row * args.k)
    {
        if (N == 0) return;
        if (a.list4) {          // lists of int32 and fp32 that start on 16 bytes
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                if (i >= a.k) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) c[i + q] = PLACE_ABSENT;
                    continue;
                }
                const int4 c4 = reinterpret_cast<const int4*>((const int32_t*)a.list + at)[i / 4];
                const float4 v4 = reinterpret_cast<const float4*>((const float*)a.teacher + at)[i / 4];
                const int cc[4] = {c4.x, c4.y, c4.z, c4.w};
                const float vv[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    c[i + q] = (unsigned)cc[q] < (unsigned)a.K ? cc[q] : (cc[q] == -1 ? PLACE_ABSENT : PLACE_BAD);
                    v[i + q] = vv[q];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                c[i] = i < a.k ? list_class(a, at + i) : PLACE_ABSENT;
                v[i] = i < a.k ? load_value(a.teacher, a.teacher_bf16, at + i) : 0.f;
            }
        }
    }
    // f(entry's number, class, value) of the entries that are there; bad() of those out of range
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const
    {
        if (N > 0) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (c[i] >= 0) f(i, c[i], v[i]);
        } else {
            for (int i = 0; i < a.k; ++i) {
                const int cls = list_class(a, at + i);
                if (cls >= 0) f(i, cls, load_value(a.teacher, a.teacher_bf16, at + i));
            }
        }
    }
    __device__ __forceinline__ bool bad() const
    {
        bool b = false;
        if (N > 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) b |= c[i] == PLACE_BAD;
        } else {
            for (int i = 0; i < a.k; ++i) b |= list_class(a, at + i) == PLACE_BAD;
        }
        return b;
    }
};

// With an outcome for the rest, the list's classes are masked in the tile once they are read: one pass over the row gives the outside's
// sum, and the list's own exponentials make it the row's.
template <typename T, int W, int N>
__global__ void __launch_bounds__(128) distill_tile_kernel(const DistillArgs a)
{
    extern __shared__ __align__(16) unsigned char smem[];
    const RowTile<T> tile(smem, a.K);
    const int64_t row0 = blockIdx.x * (int64_t)blockDim.x;
    const int rows = (int)min((int64_t)blockDim.x, a.n - row0);
    const int64_t row = row0 + threadIdx.x;
    tile.fetch((const T*)a.logits, a.ld, row0, rows, a.wide);
    const RowList<N> list(a, min(row, a.n - 1));
    tile.wait();
    if ((int)threadIdx.x >= rows) return;
    T* x = tile.row(threadIdx.x);

    const float m = tile.template largest<W>(x), origin = row_origin(m), c = a.inv_t * LOG2E;
    bool any = false;
    ListSums l{-INFINITY, 0.f, 0.f};
    if (!a.rest) list.each([&](int, int, float v) { l.top = max_nan(l.top, v); });
    float most = 0.f, inside = 0.f, z[N], parts[4] = {0.f, 0.f, 0.f, 0.f};
    list.each([&](int i, int cls, float v) {
        any = true;
        const float w = entry_weight(a, v, l.top);
        parts[i & 3] += w;
        if (a.rest) {
            const bool up = v > l.top;
            l.others += up ? most : w;
            most = up ? w : most;
            l.top = up ? v : l.top;
        }
        z[i] = (to_f<T>(x[cls]) - origin) * a.inv_t;
    });
    l.sum = (parts[0] + parts[1]) + (parts[2] + parts[3]);
    if (a.rest)
        list.each([&](int, int cls, float) {
            inside += fast_exp2(below_max(to_f<T>(x[cls]), origin) * c);       // (a class that comes again is masked by then)
            x[cls] = from_f<T>(-INFINITY);
        });
    const uint64_t c2 = pack2(c, c), minus = pack2(-origin, -origin);
    RowSum<false> sums;
    sums.clear();
    for (int j = 0; j < a.K; j += 8) sums.add(tile.template read<W>(x, j), minus, c2);
    const float outside = hsum2(sums.s), s = outside + inside;
    const bool none = s == 0.f;
    const float log_s = none ? -INFINITY : log1pf(s - 1.f);
    const float scale = a.rest ? 1.f : (l.sum > 0.f ? __fdividef(1.f, l.sum) : l.sum), log_sum = a.rest || !(l.sum > 0.f) ? 0.f : log1pf(l.sum - 1.f);
    float loss = 0.f, log_out = -INFINITY, surplus = 0.f;
    float terms[4] = {0.f, 0.f, 0.f, 0.f};
    list.each([&](int i, int, float v) { terms[i & 3] += entry_term(a, entry_weight(a, v, l.top), scale, log_sum, v, l.top, z[i], log_s); });
    loss = (terms[0] + terms[1]) + (terms[2] + terms[3]);
    if (none) loss = l.sum > 0.f ? INFINITY : l.sum;
    if (a.rest) {
        float far_log = 0.f;
        bool open = outside >= REST_TOO_SMALL || outside != outside;
        if (!open) {
            const float om = tile.template largest<W>(x);
            open = om != -INFINITY;
            if (open) {
                RowSum<false> again;
                again.clear();
                const uint64_t mo = pack2(-om, -om);
                for (int j = 0; j < a.K; j += 8) again.add(tile.template read<W>(x, j), mo, c2);
                far_log = (om - origin) * a.inv_t + logf(hsum2(again.s)) - log_s;
            }
        }
        if (open) {
            const float t_r = any ? rest_prob(l.top, l.others) : 0.f;
            const Rest r(t_r, l.sum, inside, outside, far_log, log_s);
            loss += r.term;
            log_out = r.log_out;
            surplus = r.surplus;
        }
    }
    if (list.bad()) {
        loss = NAN;
        atomicOr(a.status, PTV3_STATUS_BAD_INDEX);
    }
    a.loss[row] = loss;
    if (a.stats)
        a.stats[row] = a.rest ? make_float4(origin, log_s, log_out, surplus)
                              : make_float4(origin, log_s, row_origin(l.top), scale);
}

// ---- longer rows: G threads, some of a warp, a warp or a block ------------------------------------------------------------
// A thread keeps P pieces of eight logits in registers; the longest rows are read again for every pass (P = 0).  With an outcome
// for the rest, the list's classes are bits in shared memory, which a piece's eight are cut out of.
// the list, entry i with thread i % G of a row's threads
template <int G>
struct ListPart {
    static constexpr int N = G <= LIST_MAX ? LIST_MAX / G : 1;
    int cls[N];
    float v[N];
    __device__ __forceinline__ void load(const DistillArgs& a, int64_t at, int me)
    {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const int i = me + q * G;
            cls[q] = PLACE_ABSENT;
            v[q] = -INFINITY;
            if (q * G < a.k && i < a.k) {
                const float value = load_value(a.teacher, a.teacher_bf16, at + i);      // (on the way with the class)
                cls[q] = list_class(a, at + i);
                v[q] = cls[q] >= 0 ? value : -INFINITY;
            }
        }
    }
};

// words of bits of a row, one more for the last piece's
__host__ __device__ __forceinline__ int bit_words(int K) { return (K + 31) / 32 + 1; }

template <typename T, int G, int P>
__global__ void __launch_bounds__(Group<G>::BLOCK, row_blocks<T>(G, P)) distill_row_kernel(const DistillArgs a)
{
    __shared__ float scratch[4 * Group<G>::WARPS];
    extern __shared__ uint32_t bits_s[];
    const Group<G> group{scratch};
    const bool live = group.row() < a.n;
    const int64_t row = min(group.row(), a.n - 1);        // (threads beyond the last row keep it company)
    const int me = group.rank(), words = bit_words(a.K);
    uint32_t* bits = bits_s + group.slot() * words;
    const RowPieces<T> pieces((const T*)a.logits + row * a.ld, a.K);
    const T* x = pieces.row;
    ListPart<G> list;
    list.load(a, row * a.k, me);
    const RowValues<T, G, P> vals(pieces, me);
    float x_of[ListPart<G>::N];
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q) x_of[q] = list.cls[q] >= 0 ? to_f<T>(x[list.cls[q]]) : 0.f;
    bool twice = false;              // a class comes more than once in the list
    if (a.rest) {
        for (int w = me; w < words; w += G) bits[w] = 0;
        group.sync();
#pragma unroll
        for (int q = 0; q < ListPart<G>::N; ++q)
            if (list.cls[q] >= 0) {
                const uint32_t bit = 1u << (list.cls[q] & 31);
                twice |= (atomicOr(&bits[list.cls[q] >> 5], bit) & bit) != 0;
            }
        twice = group.any(twice);
        group.sync();
    }
    float m = -INFINITY;
    vals.each([&](const Eight<T>& e, int, int) { m = max_nan(m, e.largest()); }, [&](float e, int, int) { m = max_nan(m, e); });
    m = group.max(m);
    const float origin = row_origin(m), c = a.inv_t * LOG2E;
    const uint64_t c2 = pack2(c, c), minus = pack2(-origin, -origin);
    // the classes of the list as bits of a piece
    auto listed = [&](int j) { return __funnelshift_r(bits[j >> 5], bits[(j >> 5) + 1], j & 31) & 0xffu; };
    auto is_listed = [&](int j) { return bits[j >> 5] >> (j & 31) & 1; };
    auto masked = [&](const Eight<T>& e, int j) {
        Eight<T> o = e;
        const uint32_t in = listed(j);
        if (in) {
#pragma unroll
            for (int q = 0; q < 4; ++q) o.set(q, in >> (2 * q) & 1 ? -INFINITY : e.at(2 * q), in >> (2 * q + 1) & 1 ? -INFINITY : e.at(2 * q + 1));
        }
        return o;
    };
    RowSum<false> sums;
    sums.clear();
    EdgeSum edge{0.f, 0.f};
    float inside = 0.f;
    if (a.rest)
        vals.each([&](const Eight<T>& e, int j, int) {
            sums.add(masked(e, j), minus, c2);
            if (const uint32_t in = twice ? listed(j) : 0u) {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (in >> q & 1) inside += fast_exp2(below_max(e.at(q), origin) * c);
            }
        }, [&](float e, int j, int) {
            if (!is_listed(j))
                edge.add(e, origin, c);
            else if (twice)
                inside += fast_exp2(below_max(e, origin) * c);
        });
    else
        vals.each([&](const Eight<T>& e, int, int) { sums.add(e, minus, c2); }, [&](float e, int, int) { edge.add(e, origin, c); });
    // (the sum inside: from the list where every class is there once, else from the row)
    if (a.rest && !twice) {
#pragma unroll
        for (int q = 0; q < ListPart<G>::N; ++q)
            if (list.cls[q] >= 0) inside += fast_exp2(below_max(x_of[q], origin) * c);
    }

    // the list: its largest value, then its sums
    float top = -INFINITY;
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q)
        if (q * G < a.k) top = max_nan(top, list.v[q]);
    top = group.max(top);
    // the row's (or the outside's) sum; the list's weights; the inside's sum
    float all[3] = {hsum2(sums.s) + edge.s, 0.f, inside};
    bool bad = false, any = false;
    // with an outcome for the rest: weights but the largest's, entries that are as large as the largest
    float more[2] = {0.f, 0.f}, w[ListPart<G>::N];
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q) {
        w[q] = 0.f;
        if (q * G >= a.k) continue;
        bad |= list.cls[q] == PLACE_BAD;
        if (list.cls[q] < 0) continue;
        any = true;
        w[q] = entry_weight(a, list.v[q], top);
        all[1] += w[q];
        more[0] += list.v[q] == top ? 0.f : w[q];
        more[1] += list.v[q] == top ? 1.f : 0.f;
    }
    group.sum(all);
    if (a.rest) group.sum(more);
    bad = group.any(bad);
    if (a.rest) any = group.any(any);
    const float s = all[0] + all[2];
    const bool none = s == 0.f;
    const float log_s = none ? -INFINITY : log1pf(s - 1.f);
    const ListSums l{top, all[1], more[0] + fmaxf(more[1] - 1.f, 0.f) * fast_exp2(top * LOG2E)};
    const float scale = a.rest ? 1.f : (l.sum > 0.f ? __fdividef(1.f, l.sum) : l.sum), log_sum = a.rest || !(l.sum > 0.f) ? 0.f : log1pf(l.sum - 1.f);
    float terms[1] = {0.f};
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q)
        if (q * G < a.k && list.cls[q] >= 0)
            terms[0] += entry_term(a, w[q], scale, log_sum, list.v[q], top, (x_of[q] - origin) * a.inv_t, log_s);
    group.sum(terms);
    float loss = terms[0], log_out = -INFINITY, surplus = 0.f;
    if (none) loss = l.sum > 0.f ? INFINITY : l.sum;
    if (a.rest) {
        float far_log = 0.f;
        // (taken by all rows of a warp where one needs it)
        const bool low = all[0] < REST_TOO_SMALL;
        bool open = true;
        if (G < 32 ? __any_sync(~0u, low) : low) {
            float om = -INFINITY;
            vals.each([&](const Eight<T>& e, int j, int) { om = max_nan(om, masked(e, j).largest()); },
                      [&](float e, int j, int) { om = max_nan(om, is_listed(j) ? -INFINITY : e); });
            om = group.max(om);
            const float from = row_origin(om);
            RowSum<false> again;
            again.clear();
            const uint64_t mo = pack2(-from, -from);
            EdgeSum at_edge{0.f, 0.f};
            vals.each([&](const Eight<T>& e, int j, int) { again.add(masked(e, j), mo, c2); },
                      [&](float e, int j, int) { at_edge.add(is_listed(j) ? -INFINITY : e, from, c); });
            float o[1] = {hsum2(again.s) + at_edge.s};
            group.sum(o);
            if (low) {
                open = om != -INFINITY;
                if (open) far_log = (om - origin) * a.inv_t + logf(o[0]) - log_s;
            }
        }
        if (open) {
            const float t_r = any ? rest_prob(l.top, l.others) : 0.f;
            const Rest r(t_r, l.sum, all[2], all[0], far_log, log_s);
            loss += r.term;
            log_out = r.log_out;
            surplus = r.surplus;
        }
    }
    if (me == 0 && live) {
        if (bad) {
            loss = NAN;
            atomicOr(a.status, PTV3_STATUS_BAD_INDEX);
        }
        a.loss[row] = loss;
        if (a.stats)
            a.stats[row] = a.rest ? make_float4(origin, log_s, log_out, surplus)
                                  : make_float4(origin, log_s, row_origin(top), scale);
    }
}

// ---- gradient -------------------------------------------------------------------------------------------------------------
struct DistillGrad {
    float m, c, shift, factor, inside_shift, inside_factor, g;
    bool none;
    // every class as one outside the list
    template <typename T>
    __device__ __forceinline__ void eight(Eight<T>& x) const
    {
        row_gradient<false>(x, pack2(-m, -m), pack2(c, c), pack2(shift, shift), pack2(factor, factor), 0ull);
    }
    __device__ __forceinline__ float outside(float x) const { return fast_exp2(max_nan(fmaf(x - m, c, shift), NO_POWER)) * factor; }
    // M p of a class in the list
    __device__ __forceinline__ float in_list(float x) const
    {
        return fast_exp2(max_nan(fmaf(x - m, c, inside_shift), NO_POWER)) * inside_factor;
    }
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
        // p_j / p_r (M p_r - t_r);  M = W + max(0, 1 - W)
        r.inside_factor = max_nan(mass, 1.f) * r.g;
        r.shift = r.none ? -INFINITY : -st.z * LOG2E;
        r.factor = r.g * st.w;
    }
    return r;
}
// t of an entry from the row's stats
__device__ __forceinline__ float entry_prob(const DistillArgs& a, float4 st, float v)
{
    return a.rest ? fast_exp2(v * LOG2E) : fast_exp2(below_max(v, st.z) * (a.inv_t * LOG2E)) * st.w;
}

template <typename T, int W, int N>
__global__ void __launch_bounds__(128) distill_tile_bwd_kernel(const DistillArgs a)
{
    extern __shared__ __align__(16) unsigned char smem[];
    const RowTile<T> tile(smem, a.K);
    const int64_t row0 = blockIdx.x * (int64_t)blockDim.x;
    const int rows = (int)min((int64_t)blockDim.x, a.n - row0);
    const int64_t row = min(row0 + threadIdx.x, a.n - 1);
    tile.fetch((const T*)a.logits, a.ld, row0, rows, a.wide);
    const RowList<N> list(a, row);
    const float4 st = a.stats[row];
    tile.wait();
    if ((int)threadIdx.x < rows) {
        T* x = tile.row(threadIdx.x);
        const T* logits = (const T*)a.logits + row * a.ld;
        float mass = 0.f;
        list.each([&](int, int, float v) { mass += entry_prob(a, st, v); });
        const DistillGrad r = distill_grad(a, row, st, mass);
        // the list's classes apart: M p - t of each, which goes into the row behind the others
        float own[N];
        list.each([&](int i, int cls, float v) { own[i] = r.in_list(to_f<T>(x[cls])) - r.g * entry_prob(a, st, v); });
        for (int j = 0; j < a.K; j += 8) {
            Eight<T> e = tile.template read<W>(x, j);
            r.eight(e);
            tile.template write<W>(x, j, e);
        }
        // An entry leaves its number at its class first: where it is another's afterwards, a class comes twice, and every entry of the row
        // writes the sum over its class.
        list.each([&](int i, int cls, float) { x[cls] = from_f<T>((float)i); });
        bool twice = false;
        list.each([&](int i, int cls, float) { twice |= to_f<T>(x[cls]) != (float)i; });
        if (!twice) {
            list.each([&](int i, int cls, float) { x[cls] = from_f<T>(own[i]); });
        } else {
            const RowList<0> all(a, row);
            all.each([&](int, int cls, float) {
                float t = 0.f;
                all.each([&](int, int other, float u) { t += other == cls ? entry_prob(a, st, u) : 0.f; });
                x[cls] = from_f<T>(r.in_list(to_f<T>(logits[cls])) - r.g * t);
            });
        }
    }
    __syncthreads();
    tile.store((T*)a.dlogits, row0, rows, a.wide_out);
}

template <typename T, int G, int P>
__global__ void __launch_bounds__(Group<G>::BLOCK, row_blocks<T>(G, P)) distill_row_bwd_kernel(const DistillArgs a)
{
    __shared__ float scratch[4 * Group<G>::WARPS];
    __shared__ __align__(16) int list_c[Group<G>::ROWS][LIST_MAX];
    __shared__ float list_t[Group<G>::ROWS][LIST_MAX];
    const Group<G> group{scratch};
    const bool live = group.row() < a.n;
    const int64_t row = min(group.row(), a.n - 1);
    const int me = group.rank(), slot = group.slot();
    const RowPieces<T> pieces((const T*)a.logits + row * a.ld, a.K);
    const RowValues<T, G, P> vals(pieces, me);
    const T* x = pieces.row;
    T* dx = (T*)a.dlogits + row * a.K;
    const bool alike = (((uintptr_t)dx ^ (uintptr_t)x) & 15) == 0;
    const float4 st = a.stats[row];
    ListPart<G> list;
    list.load(a, row * a.k, me);
    float mass[1] = {0.f}, x_of[ListPart<G>::N], t_of[ListPart<G>::N];
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q) x_of[q] = list.cls[q] >= 0 ? to_f<T>(x[list.cls[q]]) : 0.f;       // (on the way with the row)
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q) {
        t_of[q] = list.cls[q] >= 0 ? entry_prob(a, st, list.v[q]) : 0.f;
        mass[0] += t_of[q];
        if (me + q * G < LIST_MAX) {
            list_c[slot][me + q * G] = list.cls[q];
            list_t[slot][me + q * G] = t_of[q];
        }
    }
    group.sum(mass);
    const DistillGrad r = distill_grad(a, row, st, mass[0]);
    if (live)
        vals.each([&](Eight<T> e, int j, int) {
            r.eight(e);
            pieces.store(dx, alike, j, e);
        }, [&](float e, int j, int) { dx[j] = from_f<T>(r.outside(e)); });
    // the list's classes once more; one that comes twice is written by its first entry, with the sum of both
    group.sync();
#pragma unroll
    for (int q = 0; q < ListPart<G>::N; ++q) {
        if (q * G >= a.k) break;
        const int mine = me + q * G, cls = list.cls[q];
        int same = 0;
        if (G == 32 && a.k <= 32) {
            same = __popc(__match_any_sync(~0u, cls < 0 ? -32 - me : cls));
        } else if (cls >= 0) {
            for (int i = 0; i < a.k; i += 4) {                   // (entries beyond the list's are -1)
                const int4 c = *reinterpret_cast<const int4*>(&list_c[slot][i]);
                same += (c.x == cls) + (c.y == cls) + (c.z == cls) + (c.w == cls);
            }
        }
        if (cls < 0 || !live) continue;
        float t = t_of[q];
        bool is_first = true;
        if (same > 1) {
            t = 0.f;
            for (int i = 0; i < a.k; ++i) {
                if (list_c[slot][i] == cls) {
                    t += list_t[slot][i];
                    is_first &= i >= mine;
                }
            }
        }
        if (is_first) dx[cls] = from_f<T>(r.in_list(x_of[q]) - r.g * t);
    }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------
template <typename T, int W>
static bool launch_tile(const DistillArgs& a, bool backward, cudaStream_t stream)
{
    const TileShape shape = tile_shape<T>(a.K);
    const unsigned blocks = (unsigned)((a.n + shape.rows - 1) / shape.rows);
    auto run = [&](auto kern) {
        if (shape.smem > 48 * 1024 && allow_smem(kern) != cudaSuccess) return false;
        kern<<<blocks, shape.rows, shape.smem, stream>>>(a);
        return true;
    };
    if (a.k <= 4) return backward ? run(distill_tile_bwd_kernel<T, W, 4>) : run(distill_tile_kernel<T, W, 4>);
    if (a.k <= 8) return backward ? run(distill_tile_bwd_kernel<T, W, 8>) : run(distill_tile_kernel<T, W, 8>);
    if (a.k <= 16) return backward ? run(distill_tile_bwd_kernel<T, W, 16>) : run(distill_tile_kernel<T, W, 16>);
    return backward ? run(distill_tile_bwd_kernel<T, W, 32>) : run(distill_tile_kernel<T, W, 32>);
}
template <typename T, int G, int P>
static void launch_row(const DistillArgs& a, bool backward, cudaStream_t stream)
{
    const size_t smem = a.rest ? (size_t)bit_words(a.K) * 4 * Group<G>::ROWS : 0;
    if (backward)
        distill_row_bwd_kernel<T, G, P><<<Group<G>::blocks(a.n), Group<G>::BLOCK, 0, stream>>>(a);
    else
        distill_row_kernel<T, G, P><<<Group<G>::blocks(a.n), Group<G>::BLOCK, smem, stream>>>(a);
}

template <typename T>
static int launch_distill(DistillArgs a, bool backward, cudaStream_t stream)
{
    a.wide = RowTile<T>::wide_rows(a.logits, a.ld, a.K);
    a.wide_out = RowTile<T>::wide_rows(a.dlogits, a.K, a.K);
    a.list4 = a.list_bytes == 4 && !a.teacher_bf16 && a.k % 4 == 0 && (((uintptr_t)a.list | (uintptr_t)a.teacher) & 15) == 0;
    // Lists of up to 32 in a thread's registers: 200 000 x 128 bf16 with 8 and a rest 66.6 us forward and 48.0 backward spread, 23.2 and 30.8 in tiles; x 166
    // fp32 86.3 and 84.2, 36.3 and 60.8; x 250 fp32 92 and 111, 58 and 94, but with 16 of 40 000 rows 25 and 31, 22 and 28; 10 000 x 64 fp32 5.0 and
    // 4.0, 4.7 and 5.3.  Longer lists have the spread form alone.
    const size_t bytes = a.K * sizeof(T);
    if (a.k <= 32 && bytes <= (many_rows(a.n) ? 704 : TILE_BYTES)) {
        bool ok;
        switch (RowTile<T>::row_width(a.K)) {
        case 16: ok = launch_tile<T, 16>(a, backward, stream); break;
        case 8: ok = launch_tile<T, 8>(a, backward, stream); break;
        case 4: ok = launch_tile<T, 4>(a, backward, stream); break;
        default: ok = launch_tile<T, sizeof(T) == 2 ? 2 : 4>(a, backward, stream); break;
        }
        if (!ok) return check_launch("ptv3_distill_topk: shared memory attribute");
    } else {
        // (a list over 8 threads at least)
        for_row_shape<T>(a.K, false, backward, [&](auto g, auto p) {
            constexpr int G = decltype(g)::value, P = decltype(p)::value;
            launch_row<T, (G < 8 ? 8 : G), (G < 8 ? P / 2 : P)>(a, backward, stream);
        });
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
                     (uintptr_t)a.list % a.list_bytes == 0 && (uintptr_t)a.stats % 16 == 0 &&
                     (((uintptr_t)a.loss | (uintptr_t)a.g | (uintptr_t)a.status) & 3) == 0,
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
