// What a row of logits answers: the log probability of a given class, the entropy, the best alternatives, and the gradient
// of all three with respect to the logits.  No counterpart in the reference, whose file ends with the backbone
// (model.py:966-982); the formulas stand in class_rows.cuh and below.
//
//     H = log S - (ln 2 / S) sum e_j t_j,    e_j = 2^t_j, t_j = (x_j - m) log2(e) / T
//     dx_j = 1/T ( p_j (A + B log p_j) + [j = label] g + sum_i [j = t_i] g_i ),   A = -(g + sum g_i) - h H,  B = -h
// with g, h, g_i the gradients of the three.
#include "class_scores.cuh"

namespace ptv3 {

// ---- short rows: a tile of rows, one thread to a row -----------------------------------------------------------------
// TOP: 0, or 1, 2, 4, ... 32 alternatives at least.  The row is read twice from shared memory, for the largest (with their keys) and for
// the sums.
// SHORT: up to 32 classes, read once and kept in registers.
template <typename T, int W, int TOP, bool SHORT>
__global__ void __launch_bounds__(128) scores_tile_kernel(const ScoresArgs a)
{
    using Top = TopKey<T>;
    extern __shared__ __align__(16) unsigned char smem[];
    const RowTile<T> tile(smem, a.K);
    const int64_t row0 = blockIdx.x * (int64_t)blockDim.x;
    const int rows = (int)min((int64_t)blockDim.x, a.n - row0);
    const int64_t row = row0 + threadIdx.x;
    tile.fetch((const T*)a.logits, a.ld, row0, rows, a.wide);
    const int label = row_label(a, min(row, a.n - 1));
    tile.wait();
    if ((int)threadIdx.x >= rows) return;
    const T* x = tile.row(threadIdx.x);

    Eight<T> kept[SHORT ? 4 : 1];
    if (SHORT) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
            if (8 * b < a.K) kept[SHORT ? b : 0] = tile.template read<W>(x, 8 * b);
    }
    // f(eight logits, class of the first)
    auto each = [&](auto&& f) {
        if (SHORT) {
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (8 * b < a.K) f(kept[SHORT ? b : 0], 8 * b);
        } else {
            for (int j = 0; j < a.K; j += 8) f(tile.template read<W>(x, j), j);
        }
    };
    typename Top::Key best[TOP > 0 ? TOP : 1];
    float m = -INFINITY;
    if (TOP == 0) {
        each([&](const Eight<T>& e, int) { m = max_nan(m, e.largest()); });
    } else if (SHORT && TOP <= 8) {
        each([&](const Eight<T>& e, int j) {
            typename Top::Key k[8];
            Top::keys(e, j, k);
#pragma unroll
            for (int b = 0; b < 8; b += (TOP > 0 && TOP <= 8 ? TOP : 8)) {
                sort_keys<(TOP > 0 && TOP <= 8 ? TOP : 8)>(k + b);
                if (b == 0 && j == 0) {
#pragma unroll
                    for (int i = 0; i < TOP; ++i) best[i] = k[i & 7];
                } else {
                    merge_keys<(TOP > 0 && TOP <= 8 ? TOP : 8)>(best, k + b);
                }
            }
        });
        m = Top::value(best[0]);
    } else {
        // (the values beyond the row are minus infinity of classes that do not exist: behind every class that does)
        constexpr int STEP = TOP > 8 ? TOP : 8;        // classes at a time: what a sort takes
        for (int j = 0; j < a.K; j += STEP) {
            typename Top::Key k[STEP];
#pragma unroll
            for (int b = 0; b < STEP; b += 8) {
                if (b == 0 || j + b < a.K) {
                    Top::keys(tile.template read<W>(x, j + b), j + b, k + b);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) k[b + i] = 0;
                }
            }
#pragma unroll
            for (int b = 0; b < STEP; b += (TOP > 0 ? TOP : 1)) {
                sort_keys<TOP>(k + b);
                if (b == 0 && j == 0) {
#pragma unroll
                    for (int i = 0; i < TOP; ++i) best[i] = k[i];
                } else {
                    merge_keys<TOP>(best, k + b);
                }
            }
        }
        m = Top::value(best[0]);                       // (of NaN: one)
    }
    const float origin = row_origin(m);
    const uint64_t c2 = pack2(a.inv_t * LOG2E, a.inv_t * LOG2E), minus = pack2(-origin, -origin);
    RowSum<true> sums;
    sums.clear();
    each([&](const Eight<T>& e, int) { sums.add(e, minus, c2); });
    const RowSums r = row_sums(m, hsum2(sums.s), hsum2(sums.u));
    write_row(a, row, r, label, label >= 0 ? to_f<T>(x[label]) : 0.f);
    if (TOP > 0) {
        const bool wide = wide_lists(a);
        write_list<TOP>(a.top_class + row * a.top, a.top, wide, [&](int i) {
            const int cls = Top::cls(best[i]);
            return (unsigned)cls < (unsigned)a.K ? cls : -1;
        });
        write_list<TOP>(a.top_logp + row * a.top, a.top, wide, [&](int i) {
            return (unsigned)Top::cls(best[i]) < (unsigned)a.K ? log_prob_of(r, Top::value(best[i]), a.inv_t) : -INFINITY;
        });
    }
}

// ---- longer rows: G threads, some of a warp, a warp or a block ------------------------------------------------------------------------
// A thread keeps P pieces of eight logits in registers; the longest rows are read again for every pass (P = 0).
//
// The alternatives.  A row's logits fall into up to 64 parts (128 for more than 32 alternatives), of which the largest are known: two or four of
// each lane where a warp has the row, one of neighbouring threads together where a block has it.  Their k-th largest, by the upper 16 bits of their
// keys, bounds the row's k-th largest from below; a warp takes its parts one after another, a block counts.  The few logits at or above the
// bound (less than twice k of most long rows) are gathered and ranked by counting.  Where more than CANDIDATES are, the best are taken one after
// another, each a maximum over the row of what comes behind the last one.
//
// That is so for rows of equal logits or of few values, and for lists that are long beside the row.  Rows of up to 256 classes have a part for
// every eight of them and one for each lane with values at the edges, not 64: with more alternatives than parts there is no bound and all
// logits are candidates.  From there to 512 and more, 64 of 128 parts still let a large share of the row pass.  60 000 rows of bf16: x 200 with 32,
// 48 and 64 alternatives 348, 480 and 608 us, x 300 with 64 786, x 500 with 64 952, x 600 with 64 400; fp32 the same.
constexpr int CANDIDATES = 192;

// value and class as one number, below ~0 (NaN of class 0); 0 for none
__device__ __forceinline__ unsigned long long wide_key(float x, int j) { return (unsigned long long)order_key(x) << 32 | (0x7fffffffu - j); }
__device__ __forceinline__ int key_class(unsigned long long k) { return k ? (int)(0x7fffffffu - (uint32_t)k) : -1; }

template <int G>
struct TopScratch {
    unsigned long long candidate[CANDIDATES];
    unsigned long long chosen[G / 32];
    uint4 maxima[G > 32 ? 32 : 1];          // 64 or 128 of a block, four to a vector
    uint32_t bound;
    int count;
};

__device__ __forceinline__ void write_alternative(const ScoresArgs& a, int64_t row, const RowSums& r, int i, unsigned long long k)
{
    a.top_class[row * a.top + i] = key_class(k);
    a.top_logp[row * a.top + i] = k ? log_prob_of(r, order_value((uint32_t)(k >> 32)), a.inv_t) : -INFINITY;
}

// the k-th largest (k = 1 ..) of 4 x 32 numbers of 16 bits, four with each lane; 0 where there are not so many
__device__ __forceinline__ uint32_t kth_largest(uint32_t (&v)[4], int k, bool four)
{
    if (!four) {
        v[0] = ::max(v[0], v[2]);
        v[1] = ::max(v[1], v[3]);
        v[2] = v[3] = 0;
    }
    uint32_t bound = 0;
#pragma unroll 1
    while (k > 0) {
        const uint32_t mine = ::max(::max(v[0], v[1]), ::max(v[2], v[3]));
        bound = __reduce_max_sync(~0u, mine);
        if (bound == 0) break;
        // all that are as large
        const int n = four ? (v[0] == bound) + (v[1] == bound) + (v[2] == bound) + (v[3] == bound) : (v[0] == bound) + (v[1] == bound);
        k -= __popc(__ballot_sync(~0u, n > 0));
        if (__any_sync(~0u, n > 1)) k -= __reduce_add_sync(~0u, n > 1 ? n - 1 : 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v[i] == bound ? 0 : v[i];
    }
    return bound;
}

template <typename T, int G, int P>
__device__ __forceinline__ void alternatives(const ScoresArgs& a, int64_t row, const RowSums& r, const RowValues<T, G, P>& vals,
                                             const Group<G>& group, TopScratch<G>& scratch, const float (&part)[4])
{
    const int me = group.rank(), lane = threadIdx.x & 31;
    const bool four = a.top > 32;
    uint32_t bound = 0;
    if (G == 32) {
        // (a part without a logit: minus infinity, which is no more than any)
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = part[i] == -INFINITY ? 0u : order_key(part[i]) >> 16;
        bound = kth_largest(v, a.top, four);
    } else {
        // a block's threads count how many reach each of 64 (128) maxima: in a tenth of the time that one warp takes for 32 of them in turn
        const int per = four ? G / 128 : G / 64, all = four ? 128 : 64;      // threads that share a maximum
        float m = max_nan(max_nan(part[0], part[1]), max_nan(part[2], part[3]));
        for (int o = 1; o < per; o *= 2) m = max_nan(m, __shfl_xor_sync(~0u, m, o));
        const uint32_t key = order_key(m) >> 16;
        if (lane % per == 0) reinterpret_cast<uint32_t*>(scratch.maxima)[me / per] = key;
        if (me == 0) scratch.count = scratch.bound = 0;
        __syncthreads();
        if (lane % per == 0) {
            int reach = 0;
#pragma unroll 4
            for (int i = 0; i < all / 4; ++i) {
                const uint4 v = scratch.maxima[i];
                reach += (v.x >= key) + (v.y >= key) + (v.z >= key) + (v.w >= key);
            }
            if (reach >= a.top) atomicMax(&scratch.bound, key);
        }
        __syncthreads();
        bound = scratch.bound;
    }
    // At or above the bound as logits (NaN is), compared as they are.  A thread's are bits of a mask; those of a row that is read again,
    // which has more than a mask has bits, are gathered as they are found.
    const float least = order_value(bound << 16);
    auto bits_of = [&](const Eight<T>& x) {
        bool any = bound == 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) any |= !(x.at(i) < least);
        uint32_t bits = 0;
        if (any) {
#pragma unroll
            for (int i = 0; i < 8; ++i) bits |= (bound == 0 || !(x.at(i) < least) ? 1u : 0u) << i;
        }
        return bits;
    };
    const T* logits = vals.pieces.row;
    auto put = [&](int at, int j) { scratch.candidate[at] = wide_key(to_f<T>(logits[j]), j); };
    int count = 0;
    if (P > 0) {
        constexpr int WORDS = (P + 3) / 4 > 0 ? (P + 3) / 4 : 1;
        uint32_t mask[WORDS] = {}, edge_mask = 0;
        vals.each([&](const Eight<T>& x, int, int i) { mask[i / 4] |= bits_of(x) << (8 * (i & 3)); },
                  [&](float x, int, int q) { edge_mask |= (bound == 0 || !(x < least) ? 1u : 0u) << q; });
        int own = __popc(edge_mask);
#pragma unroll
        for (int w = 0; w < WORDS; ++w) own += __popc(mask[w]);
        int at = own;
        if (G == 32) {
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int up = __shfl_up_sync(~0u, at, o);
                if (lane >= o) at += up;
            }
            count = __shfl_sync(~0u, at, 31);
            at -= own;
        } else {
            at = own ? atomicAdd(&scratch.count, own) : 0;
        }
        if (at + own <= CANDIDATES) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                for (uint32_t b = mask[w]; b; b &= b - 1) {
                    const int i = __ffs(b) - 1;
                    put(at++, vals.pieces.first((4 * w + (i >> 3)) * G + me) + (i & 7));
                }
            }
            for (; edge_mask; edge_mask &= edge_mask - 1) put(at++, vals.pieces.edge_class((__ffs(edge_mask) - 1) * G + me));
        }
    } else {
        vals.each([&](const Eight<T>& x, int j, int) {
            for (uint32_t mask = bits_of(x); mask; mask &= mask - 1) {
                const int at = atomicAdd(&scratch.count, 1);
                if (at < CANDIDATES) put(at, j + __ffs(mask) - 1);
            }
        }, [&](float x, int j, int) {
            if (bound == 0 || !(x < least)) {
                const int at = atomicAdd(&scratch.count, 1);
                if (at < CANDIDATES) put(at, j);
            }
        });
    }
    group.sync();
    if (G > 32) count = scratch.count;
    if (count <= CANDIDATES) {
        for (int i = me; i < ::max(count, a.top); i += G) {
            if (i < count) {
                const unsigned long long k = scratch.candidate[i];
                int before = 0;
#pragma unroll 4
                for (int q = 0; q < count; ++q) before += scratch.candidate[q] > k;
                if (before < a.top) write_alternative(a, row, r, before, k);
            } else {
                write_alternative(a, row, r, i, 0);          // no such class
            }
        }
        return;
    }
    unsigned long long last = ~0ull, key = 0;
    bool again = true;
    for (int i = 0; i < a.top; ++i) {
        if (again) {
            key = 0;
            auto look = [&](float x, int j) {
                const unsigned long long k = wide_key(x, j);
                if (k < last && k > key) key = k;
            };
            vals.each([&](const Eight<T>& x, int j, int) {
#pragma unroll
                for (int q = 0; q < 8; ++q) look(x.at(q), j + q);
            }, [&](float x, int j, int) { look(x, j); });
        }
        const uint32_t hi = __reduce_max_sync(~0u, (uint32_t)(key >> 32));
        const uint32_t lo = __reduce_max_sync(~0u, (uint32_t)(key >> 32) == hi ? (uint32_t)key : 0u);
        unsigned long long k = (unsigned long long)hi << 32 | lo;
        if (G > 32) {
            __syncthreads();
            if (lane == 0) scratch.chosen[threadIdx.x >> 5] = k;
            __syncthreads();
            k = scratch.chosen[0];
#pragma unroll
            for (int w = 1; w < G / 32; ++w) k = k > scratch.chosen[w] ? k : scratch.chosen[w];
        }
        again = k == key;
        last = k;
        if (me == 0) write_alternative(a, row, r, i, k);
    }
}

template <typename T, int G, int P, bool TOPS>
__global__ void __launch_bounds__(Group<G>::BLOCK, row_blocks<T>(G, P)) scores_row_kernel(const ScoresArgs a)
{
    __shared__ float scratch[4 * Group<G>::WARPS];
    __shared__ TopScratch<TOPS ? G : 32> top_scratch[TOPS ? Group<G>::ROWS : 1];
    const Group<G> group{scratch};
    const int64_t row = group.row(), at = min(row, a.n - 1);        // (threads beyond the last row keep it company)
    const int me = group.rank();
    const RowPieces<T> pieces((const T*)a.logits + at * a.ld, a.K);
    const RowValues<T, G, P> vals(pieces, me);
    const int label = row_label(a, at);
    const float label_x = label >= 0 ? to_f<T>(pieces.row[label]) : 0.f;
    // the largest of a thread's logits, in four parts
    float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    vals.each([&](const Eight<T>& x, int, int i) {
        if (P > 0)
            part[i & 3] = max_nan(part[i & 3], x.largest());
        else
            part[0] = max_nan(part[0], x.largest());
    }, [&](float x, int, int) { part[3] = max_nan(part[3], x); });
    const float mine = max_nan(max_nan(part[0], part[1]), max_nan(part[2], part[3]));
    const float m = group.max(mine), origin = row_origin(m);
    const uint64_t c2 = pack2(a.inv_t * LOG2E, a.inv_t * LOG2E), minus = pack2(-origin, -origin);
    RowSum<true> sums;
    sums.clear();
    EdgeSum edge{0.f, 0.f};
    vals.each([&](const Eight<T>& x, int, int) { sums.add(x, minus, c2); }, [&](float x, int, int) { edge.add(x, origin, a.inv_t * LOG2E); });
    float su[2] = {hsum2(sums.s) + edge.s, hsum2(sums.u) + edge.u};
    group.sum(su);
    const RowSums r = row_sums(m, su[0], su[1]);
    if (me == 0 && row < a.n) write_row(a, row, r, label, label_x);
    if constexpr (TOPS) {
        if (row < a.n) alternatives<T, G, P>(a, row, r, vals, group, top_scratch[group.slot()], part);     // (whole warps)
    }
}

// ---- gradient -------------------------------------------------------------------------------------------------------------
struct RowGrad {
    float m, c, shift, A, B, g, inv_t;      // A, B, g: with 1 / T in them; B for a logarithm of base 2
    int label;
    // LOG: with a gradient of the entropy
    template <bool LOG, typename T>
    __device__ __forceinline__ void eight(Eight<T>& x) const
    {
        row_gradient<LOG>(x, pack2(-m, -m), pack2(c, c), pack2(shift, shift), pack2(A, A), pack2(B, B));
    }
    // one class, with the part of its own
    __device__ __forceinline__ float at(float x, int j, float own) const
    {
        const float t = max_nan(fmaf(x - m, c, shift), NO_POWER);
        return fmaf(fast_exp2(t), fmaf(t, B, A), fmaf(own, inv_t, j == label ? g : 0.f));
    }
};
__device__ __forceinline__ RowGrad row_grad(const ScoresArgs& a, int64_t row, float g_top_sum, bool& none)
{
    RowGrad r;
    const float4 st = a.stats[row];
    none = st.y == -INFINITY;
    r.m = st.x;
    r.c = a.inv_t * LOG2E;
    r.shift = none ? -INFINITY : -st.y * LOG2E;
    r.inv_t = a.inv_t;
    r.label = -1;
    float g = 0.f;
    if (a.g_logp) {
        const int64_t label = load_index(a.labels, a.label_bytes, row);
        if (label != a.ignore && label >= 0 && label < a.K && !none) {
            r.label = (int)label;
            g = a.g_logp[row * a.g_logp_step];
        }
    }
    const float h = a.g_entropy ? a.g_entropy[row * a.g_entropy_step] : 0.f;
    r.g = g * a.inv_t;
    r.A = none ? 0.f : (-(g + g_top_sum) - (a.g_entropy ? h * st.z : 0.f)) * a.inv_t;
    r.B = none ? 0.f : -h * a.inv_t * LN2;
    return r;
}

template <typename T, int W, bool LOG>
__global__ void __launch_bounds__(128) scores_tile_bwd_kernel(const ScoresArgs a)
{
    extern __shared__ __align__(16) unsigned char smem[];
    const RowTile<T> tile(smem, a.K);
    const int64_t row0 = blockIdx.x * (int64_t)blockDim.x;
    const int rows = (int)min((int64_t)blockDim.x, a.n - row0);
    tile.fetch((const T*)a.logits, a.ld, row0, rows, a.wide);
    const int64_t row = min(row0 + threadIdx.x, a.n - 1);
    const float* gt = a.g_top ? a.g_top + row * a.top : nullptr;
    const int32_t* tc = a.g_top ? a.top_class + row * a.top : nullptr;
    float g_sum = 0.f;
    if (gt)
        for (int i = 0; i < a.top; ++i) g_sum += tc[i] >= 0 ? gt[i] : 0.f;
    bool none;
    const RowGrad r = row_grad(a, row, g_sum, none);
    tile.wait();
    if ((int)threadIdx.x < rows) {
        T* x = tile.row(threadIdx.x);
        const T* logits = (const T*)a.logits + row * a.ld;
        const T label = r.label >= 0 ? from_f<T>(r.at(to_f<T>(x[r.label]), r.label, 0.f)) : from_f<T>(0.f);
        for (int j = 0; j < a.K; j += 8) {
            Eight<T> e = tile.template read<W>(x, j);
            r.eight<LOG>(e);
            tile.template write<W>(x, j, e);
        }
        if (r.label >= 0) x[r.label] = label;
        if (gt && !none)
            for (int i = 0; i < a.top; ++i)
                if (tc[i] >= 0) x[tc[i]] = from_f<T>(r.at(to_f<T>(logits[tc[i]]), tc[i], gt[i]));
    }
    __syncthreads();
    tile.store((T*)a.dlogits, row0, rows, a.wide_out);
}

template <typename T, int G, int P, bool LOG>
__global__ void __launch_bounds__(Group<G>::BLOCK, row_blocks<T>(G, P)) scores_row_bwd_kernel(const ScoresArgs a)
{
    __shared__ float scratch[4 * Group<G>::WARPS];
    const Group<G> group{scratch};
    const bool live = group.row() < a.n;
    const int64_t row = min(group.row(), a.n - 1);
    const int me = group.rank();
    const RowPieces<T> pieces((const T*)a.logits + row * a.ld, a.K);
    const RowValues<T, G, P> vals(pieces, me);
    const T* x = pieces.row;
    T* dx = (T*)a.dlogits + row * a.K;
    const bool alike = (((uintptr_t)dx ^ (uintptr_t)x) & 15) == 0;
    const float* gt = a.g_top ? a.g_top + row * a.top : nullptr;
    const int32_t* tc = a.g_top ? a.top_class + row * a.top : nullptr;
    float g_sum[1] = {0.f};
    if (gt) {
        for (int i = me; i < a.top; i += G) g_sum[0] += tc[i] >= 0 ? gt[i] : 0.f;
        group.sum(g_sum);
    }
    bool none;
    const RowGrad r = row_grad(a, row, g_sum[0], none);
    const float label_x = r.label >= 0 ? to_f<T>(x[r.label]) : 0.f;       // (on the way with the row)
    if (live)
        vals.each([&](Eight<T> e, int j, int) {
            r.eight<LOG>(e);
            pieces.store(dx, alike, j, e);
        }, [&](float e, int j, int) { dx[j] = from_f<T>(r.at(e, j, 0.f)); });
    // classes with parts of their own once more: the label, then the alternatives (of which the label may be one)
    group.sync();
    if (me == 0 && live && r.label >= 0) dx[r.label] = from_f<T>(r.at(label_x, r.label, 0.f));
    if (gt) {
        group.sync();
        for (int i = me; i < (live && !none ? a.top : 0); i += G)
            if (tc[i] >= 0) dx[tc[i]] = from_f<T>(r.at(to_f<T>(x[tc[i]]), tc[i], gt[i]));
    }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------
template <typename T, int W>
static bool launch_tile(const ScoresArgs& a, bool backward, cudaStream_t stream)
{
    const TileShape shape = tile_shape<T>(a.K);
    const unsigned blocks = (unsigned)((a.n + shape.rows - 1) / shape.rows);
    auto run = [&](auto kern) {
        if (shape.smem > 48 * 1024 && allow_smem(kern) != cudaSuccess) return false;
        kern<<<blocks, shape.rows, shape.smem, stream>>>(a);
        return true;
    };
    if (backward) return a.g_entropy ? run(scores_tile_bwd_kernel<T, W, true>) : run(scores_tile_bwd_kernel<T, W, false>);
    // (kept in registers a row is read once: 407 678 x 20 with 5 alternatives 16.5 us read twice, 15.8 so)
    const bool few = a.K <= 32;
    if (a.top == 0) return few ? run(scores_tile_kernel<T, W, 0, true>) : run(scores_tile_kernel<T, W, 0, false>);
    if (a.top == 1) return few ? run(scores_tile_kernel<T, W, 1, true>) : run(scores_tile_kernel<T, W, 1, false>);
    if (a.top == 2) return few ? run(scores_tile_kernel<T, W, 2, true>) : run(scores_tile_kernel<T, W, 2, false>);
    if (a.top <= 4) return few ? run(scores_tile_kernel<T, W, 4, true>) : run(scores_tile_kernel<T, W, 4, false>);
    if (a.top <= 8) return few ? run(scores_tile_kernel<T, W, 8, true>) : run(scores_tile_kernel<T, W, 8, false>);
    if (a.top <= 16) return run(scores_tile_kernel<T, W, 16, false>);
    return run(scores_tile_kernel<T, W, 32, false>);
}
template <typename T>
static bool launch_tile_of(const ScoresArgs& a, bool backward, cudaStream_t stream)
{
    switch (RowTile<T>::row_width(a.K)) {
    case 16: return launch_tile<T, 16>(a, backward, stream);
    case 8: return launch_tile<T, 8>(a, backward, stream);
    case 4: return launch_tile<T, 4>(a, backward, stream);
    default: return launch_tile<T, sizeof(T) == 2 ? 2 : 4>(a, backward, stream);
    }
}

template <typename T, int G, int P>
static void launch_row(const ScoresArgs& a, bool backward, cudaStream_t stream)
{
    if (backward)
        a.g_entropy ? scores_row_bwd_kernel<T, G, P, true><<<Group<G>::blocks(a.n), Group<G>::BLOCK, 0, stream>>>(a)
                    : scores_row_bwd_kernel<T, G, P, false><<<Group<G>::blocks(a.n), Group<G>::BLOCK, 0, stream>>>(a);
    else if constexpr (G >= 32)
        a.top ? scores_row_kernel<T, G, P, true><<<Group<G>::blocks(a.n), Group<G>::BLOCK, 0, stream>>>(a)
              : scores_row_kernel<T, G, P, false><<<Group<G>::blocks(a.n), Group<G>::BLOCK, 0, stream>>>(a);
    else
        scores_row_kernel<T, G, P, false><<<Group<G>::blocks(a.n), Group<G>::BLOCK, 0, stream>>>(a);
}

// Sums and gradients: 200 000 x 72 bf16 15.5 and 23.1 us spread, 9.5 and 14.4 in tiles; x 128 16.9 and 29.0, 16.8 and 27.4; x 200 20.5 and 38.0, 24.4 and
// 43.3.  Alternatives, up to 32 of a thread's: few rows of more than 256 bytes finish sooner spread (2 000 x 200 bf16 with 8: 8.7 us in tiles, 4.3), but
// for many of them; many are slower so up to 1 024 bytes of bf16 or 704 of fp32, where keys have 64 bits (60 000 x 333 bf16 with 8 and 32: 65.5 and 154 us
// spread, 37.0 and 52.6 in tiles; x 500 65.8 and 138, 56.5 and 74.0; x 166 fp32 53.2 and 422, 41.6 and 78.0; x 250 with 8 52.5, 61.5).
// These bounds are those of few alternatives.  With 32 the spread form, which is taken, is the slower one beyond them: 10 000 x 166 fp32 78 us, 31 in
// tiles; 60 000 x 250 fp32 275 and 112; 10 000 x 333 bf16 32 and 21; 60 000 x 600 bf16 156 and 112; with 8 of 100 000 x 200 fp32 84 and 74.  The other
// way round, tiles are taken and slower for 2 000 x 100 fp32 with 32 (18.5 us, 14.4 spread) and 20 000 x 500 bf16 with 8 (28.8 and 24.7).  More than 32
// alternatives have the spread form alone.
template <typename T>
static bool in_tiles(const ScoresArgs& a, bool backward)
{
    const size_t bytes = a.K * sizeof(T);
    const bool many = many_rows(a.n);
    if (backward || a.top == 0) return bytes <= (many ? 160 : TILE_BYTES);
    if (a.top > 32) return false;
    if (bytes <= 512) return bytes <= 256 || a.top > 16 || a.n >= SMS * 32;
    return many && bytes <= (sizeof(T) == 2 ? 1024 : 704);
}

template <typename T>
static int launch_scores(ScoresArgs a, bool backward, cudaStream_t stream)
{
    a.wide = RowTile<T>::wide_rows(a.logits, a.ld, a.K);
    a.wide_out = RowTile<T>::wide_rows(a.dlogits, a.K, a.K);
    const char* what = backward ? "ptv3_class_scores_bwd" : "ptv3_class_scores_fwd";
    if (in_tiles<T>(a, backward)) {
        if (!launch_tile_of<T>(a, backward, stream)) return check_launch("ptv3_class_scores: shared memory attribute");
    } else {
        // (where alternatives are chosen, a warp at least)
        for_row_shape<T>(a.K, !backward && a.top, backward, [&](auto g, auto p) { launch_row<T, decltype(g)::value, decltype(p)::value>(a, backward, stream); });
    }
    count_launches(1);
    return check_launch(what);
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
    PTV3_REQUIRE((((uintptr_t)a.logp | (uintptr_t)a.entropy | (uintptr_t)a.top_logp | (uintptr_t)a.top_class | (uintptr_t)a.g_logp |
                   (uintptr_t)a.g_entropy | (uintptr_t)a.g_top | (uintptr_t)a.status) & 3) == 0 && ((uintptr_t)a.stats & 15) == 0 &&
                     (!a.labels || a.label_bytes < 1 || (uintptr_t)a.labels % a.label_bytes == 0),
                 PTV3_ERR_INVALID_ARGUMENT, "%s: unaligned labels, outputs or gradients", what);
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
    a.stats = (float4*)stats;
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
    return dtype == PTV3_DTYPE_F32 ? launch_scores<float>(a, false, (cudaStream_t)stream)
                                   : launch_scores<__nv_bfloat16>(a, false, (cudaStream_t)stream);
}

extern "C" int ptv3_class_scores_bwd(const void* logits, int64_t ld, const void* labels, int label_bytes, int64_t ignore,
                                     const int32_t* top_class, const float* stats,
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
    a.top_class = const_cast<int32_t*>(top_class);
    a.stats = (float4*)stats;
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
    PTV3_REQUIRE(logits && stats && dlogits && (!dlog_prob || labels) && (!a.g_top || top_class),
                 PTV3_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    return dtype == PTV3_DTYPE_F32 ? launch_scores<float>(a, true, (cudaStream_t)stream)
                                   : launch_scores<__nv_bfloat16>(a, true, (cudaStream_t)stream);
}
