// Scores straight from features: the segmentation head's Linear layer and what class_scores.cu answers of its logits, which are
// never in memory, for any number of classes.  No counterpart in the reference, whose file ends with the backbone (model.py:966-982).
//
//     x = feat W^T + bias in fp32;  log p of the label, entropy, alternatives as class_rows.cuh has them
//
// A persistent CTA per SM walks tiles of 128 rows by N classes.  Warp 0 fetches 64-wide pieces of the rows' features, which stay until the
// last class tile has used them, and of W (resident where it fits) by TMA; warp 1 issues the products (tcgen05.mma) into one of NG
// accumulators in tensor memory; NG groups of four warps have an accumulator each, one thread to a row: it reads 32 logits at a time
// (tcgen05.ld), keeps the row's maximum and sums (running: log-sum-exp and entropy need one pass), the label's logit and the best
// classes.  So no value crosses threads, and groups work on different tiles while the next are multiplied.  Where a row has several
// class tiles, the groups' results of it meet in shared memory.
//
// Alternatives: 32 logits go through a sorting network of 32-bit keys, the logit without its last five bits and its place instead of
// them, a maximum and a minimum to an exchange; the best of these, as they are, merge with the row's best so far.  Where logits that differ in
// those bits alone are among the best of the 32, or beside them, the warp takes 64-bit keys, which hold all of both (three times the time).
#include "class_scores.cuh"
#include "tc05.cuh"

namespace ptv3 {

using namespace tc05;

constexpr int HS_ROWS = 128;
constexpr int HS_BK = 64;                              // one 128-byte swizzle span of bf16
constexpr int HS_X_BYTES = HS_ROWS * HS_BK * 2;
constexpr int HS_AREA = 32 * 32;                       // words of a warp: 32 logits of its rows

struct HeadArgs {
    ScoresArgs s;                  // n, labels, outputs, K, top, inv_t, status
    const __nv_bfloat16* bias;     // K or NULL
    int chunks, last_steps;        // pieces of 64 features, products of 16 in the last of these
    int N, col_tiles, row_tiles;
    int x_stages, w_stages;        // w_stages 0: all of W is resident
};

__device__ __forceinline__ unsigned long long head_key(float x, int j) { return x > -INFINITY ? (unsigned long long)order_key(x) << 32 | (0x7fffffffu - j) : 0ull; }

// A row's best logits, sorted, the lowest class first among equals; minus infinity (of any class) where there are no more.
template <int B>
struct Best {
    float v[B];
    int c[B];
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            v[i] = -INFINITY;
            c[i] = -1;
        }
    }
    __device__ __forceinline__ void from_keys(const unsigned long long* k)
    {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            v[i] = k[i] ? order_value((uint32_t)(k[i] >> 32)) : -INFINITY;
            c[i] = (int)(0x7fffffffu - (uint32_t)k[i]);
        }
    }
    // The best of 32 logits, classes from j0 on; those from the `width`-th on and masked ones are minus infinity.  mine: the same, 32 words apart in
    // shared memory
    __device__ __forceinline__ void take(const float (&x)[32], int j0, int width, int top, float* mine)
    {
        constexpr int STEP = B > 8 ? B : 8;
        int best[B], lost = INT32_MIN;
#pragma unroll
        for (int b = 0; b < 32; b += STEP) {
            if (b == 0 || b < width) {
                int k[STEP];
#pragma unroll
                for (int i = 0; i < STEP; ++i) {
                    const int u = __float_as_int(x[b + i]);
                    k[i] = ((u ^ ((u >> 31) & 0x7fffffff)) & ~31) | (31 - (b + i));
                }
#pragma unroll
                for (int q = 0; q < STEP; q += B) {
                    sort_keys<B>(k + q);
                    if (b == 0 && q == 0) {
#pragma unroll
                        for (int i = 0; i < B; ++i) best[i] = k[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < B; ++i) lost = ::max(lost, ::min(best[i], k[q + B - 1 - i]));
                        merge_keys<B>(best, k + q);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int at = 31 - (best[i] & 31);
            c[i] = j0 + at;
            v[i] = mine[32 * at];
        }
        // Keys that differ in the place alone: their logits may be in the other order, or one that was left out larger than the last.
        // (Equal logits are in order: the lower place has the larger key.)
        bool wrong = false;
#pragma unroll
        for (int i = 0; i + 1 < B; ++i) wrong |= v[i] < v[i + 1];
        const bool edge = (unsigned)(best[B - 1] ^ lost) < 32u && v[B - 1] > -INFINITY;
        if (__any_sync(~0u, edge)) {
            // (where nothing larger was left out, all that are better than the last are in the list, before those that equal it)
            int better = 0, kept = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) better += x[i] > v[B - 1];
#pragma unroll
            for (int i = 0; i + 1 < B; ++i) kept += v[i] > v[B - 1];
            wrong |= edge && better > kept;
        }
        if (__any_sync(~0u, wrong)) {
            unsigned long long wide[B];
#pragma unroll
            for (int i = 0; i < B; ++i) wide[i] = 0;
#pragma unroll
            for (int b = 0; b < 32; b += STEP) {
                if (b == 0 || b < width) {
                    unsigned long long k[STEP];
#pragma unroll
                    for (int i = 0; i < STEP; ++i) k[i] = head_key(x[b + i], j0 + b + i);
#pragma unroll
                    for (int q = 0; q < STEP; q += B) {
                        sort_keys<B>(k + q);
                        merge_keys<B>(wide, k + q);
                    }
                }
            }
            from_keys(wide);
        }
    }
    // with the best of later classes
    __device__ __forceinline__ void merge(const Best& o)
    {
        bool equal = false;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const bool up = o.v[B - 1 - i] > v[i];
            v[i] = up ? o.v[B - 1 - i] : v[i];
            c[i] = up ? o.c[B - 1 - i] : c[i];
        }
#pragma unroll
        for (int d = B / 2; d >= 1; d /= 2)
#pragma unroll
            for (int i = 0; i < B; ++i)
                if ((i & d) == 0) exchange(i, i + d, v[i + d] > v[i]);
#pragma unroll
        for (int i = 0; i + 1 < B; ++i) equal |= v[i] == v[i + 1] && v[i] > -INFINITY;
        // (the half-cleaners leave equal logits in any order)
        if (__any_sync(~0u, equal)) {
#pragma unroll 1
            for (int r = 0; r < B / 2; ++r) {
#pragma unroll
                for (int i = 0; i + 1 < B; i += 2) exchange(i, i + 1, v[i] == v[i + 1] && c[i + 1] < c[i]);
#pragma unroll
                for (int i = 1; i + 1 < B; i += 2) exchange(i, i + 1, v[i] == v[i + 1] && c[i + 1] < c[i]);
            }
        }
    }
    // one logit of a later class that is better than the last; a thread with none passes minus infinity
    __device__ __forceinline__ void insert(float x, int j)
    {
        bool up = false;         // from the first smaller one on, everything moves
#pragma unroll
        for (int i = 0; i < B; ++i) {
            up |= x > v[i];
            const float vi = v[i];
            const int ci = c[i];
            v[i] = up ? x : vi;
            c[i] = up ? j : ci;
            x = up ? vi : x;
            j = up ? ci : j;
        }
    }
    __device__ __forceinline__ float at(int n) const
    {
        float x = v[0];
#pragma unroll
        for (int i = 1; i < B; ++i) x = i == n ? v[i] : x;
        return x;
    }
    __device__ __forceinline__ void exchange(int i, int j, bool swap)
    {
        const float vi = v[i];
        const int ci = c[i];
        v[i] = swap ? v[j] : vi;
        c[i] = swap ? c[j] : ci;
        v[j] = swap ? vi : v[j];
        c[j] = swap ? ci : c[j];
    }
};
template <>
struct Best<0> {
    __device__ __forceinline__ void clear() {}
};

// Of 32 logits behind n, 32 k / n are better than the k-th best on average.  One costs 5 B operations in a warp and the row with most of them
// decides, the network 28 B and the merge 20 B: from 8 B on one after another is cheaper (100 003 x 64 to 1 201 classes with 16: 506 us with the network
// alone, 282 so).
constexpr int HS_FEW = 8;

// a row's running answers
struct HeadRow {
    float m, s, u, label_x;
    __device__ __forceinline__ void clear()
    {
        m = -INFINITY;
        s = u = label_x = 0.f;
    }
    // sums relative to `to` instead of the present maximum
    __device__ __forceinline__ void rebase(float to, float c)
    {
        if (m != -INFINITY) {
            // (a maximum that is no number makes the sums none)
            const float d = to < INFINITY ? fmaxf((m - row_origin(to)) * c, NO_POWER) : NAN, f = fast_exp2(d);
            u = f * fmaf(d, s, u);
            s *= f;
        }
        m = to;
    }
    __device__ __forceinline__ void merge(HeadRow o, float c)
    {
        const float to = max_nan(m, o.m);
        rebase(to, c);
        o.rebase(to, c);
        s += o.s;
        u += o.u;
    }
};

template <int NG, int B>
__global__ void __launch_bounds__(64 + NG * 128, 1) head_scores_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                       const __grid_constant__ CUtensorMap map_w, const HeadArgs a)
{
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + (-smem_u32_generic(smem_raw) & 1023u);       // (plain arithmetic: it stays known to be shared)
    const uint32_t sbase = smem_u32_generic(smem);
    const int w_bytes = a.N * HS_BK * 2;
    const int w_count = a.w_stages ? a.w_stages : a.col_tiles * a.chunks;
    const uint32_t x_base = sbase, w_base = sbase + a.x_stages * HS_X_BYTES;
    unsigned char* after = smem + a.x_stages * HS_X_BYTES + w_count * w_bytes;
    float* bias_s = reinterpret_cast<float*>(after);                                     // NG x N
    // words of each warp; where groups meet, they leave their parts in the same place
    constexpr int MEET_ROW = 16 + B * 8, PENDING_BYTES = B ? NG * 4 * HS_AREA * 4 : 0, MEET_BYTES = (NG - 1) * HS_ROWS * MEET_ROW;
    unsigned char* pending = reinterpret_cast<unsigned char*>(bias_s + NG * a.N);
    uint64_t* bars = reinterpret_cast<uint64_t*>(pending + (a.col_tiles > 1 && MEET_BYTES > PENDING_BYTES ? MEET_BYTES : PENDING_BYTES));
    const int nbar = 2 * a.x_stages + 2 * a.w_stages + 2 * NG + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + nbar);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t bar0 = smem_u32_generic(bars);
    const uint32_t x_full = bar0, x_empty = x_full + 8 * a.x_stages, w_full = x_empty + 8 * a.x_stages, w_empty = w_full + 8 * a.w_stages,
                   acc_full = w_empty + 8 * a.w_stages, acc_empty = acc_full + 8 * NG, w_all = acc_empty + 8 * NG;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int columns = 32;
    while (columns < NG * a.N) columns *= 2;
    if (tid == 0) {
        for (int i = 0; i < a.x_stages; ++i) {
            mbar_init(x_full + 8 * i, 1);
            mbar_init(x_empty + 8 * i, 1);
        }
        for (int i = 0; i < a.w_stages; ++i) {
            mbar_init(w_full + 8 * i, 1);
            mbar_init(w_empty + 8 * i, 1);
        }
        for (int i = 0; i < NG; ++i) {
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, 4);             // one arrival for each warp of the group
        }
        mbar_init(w_all, 1);
        *abort = 0;
        fence_barrier_init();
        prefetch_tensormap(&map_x);
        prefetch_tensormap(&map_w);
    }
    if (warp == 1) tmem_alloc(smem_u32_generic(tmem_slot), columns);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;
    pdl_wait();

    if (warp == 0) {
        // ---- producer: a row tile's features, then its pieces of W ----------------------------------------------------
        if (!a.w_stages && elect_one()) {
            mbar_expect_tx(w_all, (uint32_t)(w_count * w_bytes));
            for (int t = 0; t < a.col_tiles; ++t)
                for (int k = 0; k < a.chunks; ++k)
                    tma_load_2d(w_base + (t * a.chunks + k) * w_bytes, &map_w, k * HS_BK, t * a.N, w_all);
        }
        __syncwarp();
        int xs = 0, x_phase = 1, ws = 0, w_phase = 1;
        for (int rt = blockIdx.x; rt < a.row_tiles; rt += gridDim.x) {
            for (int k = 0; k < a.chunks; ++k) {
                ok &= mbar_wait(x_empty + 8 * xs, x_phase, abort);
                if (elect_one()) {
                    mbar_expect_tx(x_full + 8 * xs, HS_X_BYTES);
                    tma_load_2d(x_base + xs * HS_X_BYTES, &map_x, k * HS_BK, rt * HS_ROWS, x_full + 8 * xs);
                }
                __syncwarp();
                if (++xs == a.x_stages) {
                    xs = 0;
                    x_phase ^= 1;
                }
            }
            if (a.w_stages)
                for (int t = 0; t < a.col_tiles; ++t)
                    for (int k = 0; k < a.chunks; ++k) {
                        ok &= mbar_wait(w_empty + 8 * ws, w_phase, abort);
                        if (elect_one()) {
                            mbar_expect_tx(w_full + 8 * ws, (uint32_t)w_bytes);
                            tma_load_2d(w_base + ws * w_bytes, &map_w, k * HS_BK, t * a.N, w_full + 8 * ws);
                        }
                        __syncwarp();
                        if (++ws == a.w_stages) {
                            ws = 0;
                            w_phase ^= 1;
                        }
                    }
        }
    } else if (warp == 1) {
        // ---- issuer -------------------------------------------------------------------------------------------------------
        const uint32_t idesc = umma_idesc_bf16(HS_ROWS, a.N);
        const uint64_t dx0 = umma_desc_kmajor(x_base, 128), dw0 = umma_desc_kmajor(w_base, 128);
        int xs = 0, x_phase = 0, ws = 0, w_phase = 0, g = 0, acc_phase = 1;
        if (!a.w_stages) ok &= mbar_wait(w_all, 0, abort);
        for (int rt = blockIdx.x; rt < a.row_tiles; rt += gridDim.x) {
            int x_at = xs, x_ph = x_phase;
            for (int t = 0; t < a.col_tiles; ++t) {
                // the group has read this accumulator's tile before
                ok &= mbar_wait(acc_empty + 8 * g, acc_phase, abort);
                fence_after_sync();
                x_at = xs;
                x_ph = x_phase;
                for (int k = 0; k < a.chunks; ++k) {
                    if (t == 0) ok &= mbar_wait(x_full + 8 * x_at, x_ph, abort);
                    if (a.w_stages) ok &= mbar_wait(w_full + 8 * ws, w_phase, abort);
                    fence_after_sync();
                    const uint64_t dx = dx0 + (uint64_t)x_at * (HS_X_BYTES >> 4);
                    const uint64_t dw = dw0 + (uint64_t)(a.w_stages ? ws : t * a.chunks + k) * (w_bytes >> 4);
                    const int steps = k == a.chunks - 1 ? a.last_steps : HS_BK / 16;
                    if (elect_one()) {
#pragma unroll
                        for (int q = 0; q < HS_BK / 16; ++q)
                            if (q < steps) umma_bf16(tmem + g * a.N, dx + 2 * q, dw + 2 * q, idesc, k > 0 || q > 0);
                        if (a.w_stages) umma_commit(w_empty + 8 * ws);
                        if (t == a.col_tiles - 1) umma_commit(x_empty + 8 * x_at);
                        if (k == a.chunks - 1) umma_commit(acc_full + 8 * g);
                    }
                    __syncwarp();
                    if (++x_at == a.x_stages) {
                        x_at = 0;
                        x_ph ^= 1;
                    }
                    if (a.w_stages && ++ws == a.w_stages) {
                        ws = 0;
                        w_phase ^= 1;
                    }
                }
                if (++g == NG) {
                    g = 0;
                    acc_phase ^= 1;
                }
            }
            xs = x_at;
            x_phase = x_ph;
        }
    } else {
        // ---- groups: thread = row of the tile ----------------------------------------------------------------------------
        const int group = (warp - 2) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t my_tmem = tmem + group * a.N + ((uint32_t)(quarter * 32) << 16);
        float* my_bias = bias_s + group * a.N;
        // (a row's places are 32 lanes apart, so that a warp's stores meet no conflict)
        uint32_t* area = reinterpret_cast<uint32_t*>(pending) + (group * 4 + quarter) * HS_AREA;
        float* my_logits = reinterpret_cast<float*>(area) + lane;
        const float c = a.s.inv_t * LOG2E;
        const uint64_t c2 = pack2(c, c);
        int turn = 0, phase = 0;         // class tiles so far, modulo NG; of this group's accumulator
        bool bias_there = false;
        int tile_no = 0;
        for (int rt = blockIdx.x; rt < a.row_tiles; rt += gridDim.x, ++tile_no) {
            if (a.col_tiles == 1 && tile_no % NG != group) continue;
            const int64_t row = (int64_t)rt * HS_ROWS + r;
            HeadRow h;
            h.clear();
            Best<B> best;
            best.clear();
            int seen = 0;                        // classes of the row that the group has had
            const int label = row_label(a.s, min(row, a.s.n - 1));       // (read early: it has until the first tile is there)
            bool mine = false;
            for (int t = 0; t < a.col_tiles; ++t) {
                if (a.col_tiles > 1) {
                    const bool here = turn == group;
                    turn = turn + 1 == NG ? 0 : turn + 1;
                    if (!here) continue;
                }
                mine = true;
                const int col0 = t * a.N;
                if (!bias_there || a.col_tiles > 1) {
                    if (bias_there) named_barrier(1 + group, 128);     // every warp has finished with the tile before
                    for (int i = r; i < a.N; i += HS_ROWS)
                        my_bias[i] = a.bias && col0 + i < a.s.K ? __bfloat162float(a.bias[col0 + i]) + 0.f : 0.f;    // (no zero below zero)
                    named_barrier(1 + group, 128);
                    bias_there = true;
                }
                ok &= mbar_wait(acc_full + 8 * group, phase, abort);
                phase ^= 1;
                fence_after_sync();
                const int width = min(a.N, a.s.K - col0);
                for (int b = 0; b < width; b += 32) {
                    uint32_t v[32];
                    tmem_ld32(my_tmem + b, v);
                    tmem_ld_wait();
                    tmem_ld_fence(v);
                    float x[32];
                    const ulonglong2* bias2 = reinterpret_cast<const ulonglong2*>(my_bias + b);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const ulonglong2 bb = bias2[i / 4];
                        unpack2(add2(pack2u(v[i], v[i + 1]), bb.x), x[i], x[i + 1]);
                        unpack2(add2(pack2u(v[i + 2], v[i + 3]), bb.y), x[i + 2], x[i + 3]);
                    }
                    const int j0 = col0 + b;
                    if (b + 32 > width) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = i < width - b ? x[i] : -INFINITY;
                    }
                    // running sums, eight classes at a time as far as there are any
                    float top = -INFINITY;
#pragma unroll
                    for (int q = 0; q < 32; q += 8) {
                        if (q == 0 || b + q < width) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) top = max_nan(top, x[q + i]);
                        }
                    }
                    h.rebase(max_nan(h.m, top), c);
                    const float origin = row_origin(h.m);
                    const uint64_t minus = pack2(-origin, -origin);
                    uint64_t s2[2] = {0, 0}, u2[2] = {0, 0};
#pragma unroll
                    for (int q = 0; q < 32; q += 8) {
                        if (q == 0 || b + q < width) {
#pragma unroll
                            for (int i = q; i < q + 8; i += 2) {
                                float lo, hi;
                                unpack2(mul2(add2(pack2(x[i], x[i + 1]), minus), c2), lo, hi);
                                lo = max_nan(lo, NO_POWER);
                                hi = max_nan(hi, NO_POWER);
                                const uint64_t e = pack2(fast_exp2(lo), fast_exp2(hi));
                                s2[i / 2 & 1] = add2(s2[i / 2 & 1], e);
                                u2[i / 2 & 1] = fma2(e, pack2(lo, hi), u2[i / 2 & 1]);
                            }
                        }
                    }
                    h.s += hsum2(add2(s2[0], s2[1]));
                    h.u += hsum2(add2(u2[0], u2[1]));
                    // alternatives
                    if constexpr (B > 0) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) my_logits[32 * i] = x[i];
                        if ((unsigned)(label - j0) < 32u) h.label_x = my_logits[32 * (label - j0)];
                        const int so_far = seen;
                        seen += 32;
                        if (so_far == 0) {
                            best.take(x, j0, width - b, a.s.top, my_logits);
                        } else if (so_far < HS_FEW * B) {
                            Best<B> more;
                            more.take(x, j0, width - b, a.s.top, my_logits);
                            best.merge(more);
                        } else {
                            // few of 32 are better than the row's k-th best by now: one after another, a row of the warp's with each thread
                            float least = best.at(a.s.top - 1);
                            if (__any_sync(~0u, top > least)) {
                                uint32_t better = 0;
#pragma unroll
                                for (int i = 0; i < 32; ++i) better |= x[i] > least ? 1u << i : 0u;
                                while (__any_sync(~0u, better != 0)) {
                                    const int i = better ? __ffs(better) - 1 : 0;
                                    const float y = better ? my_logits[32 * i] : -INFINITY;
                                    best.insert(y, j0 + i);
                                    better &= better - 1;
                                }
                            }
                        }
                    }
                    if (b + 32 >= width) {
                        // the accumulator may be overwritten
                        fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_one(acc_empty + 8 * group);
                    }
                    // the label's logit (last: the label has had time to come)
                    if (B == 0 && (unsigned)(label - j0) < 32u) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (label == j0 + i) h.label_x = x[i];
                    }
                }
            }
            if (a.col_tiles > 1) {
                // the groups' parts of the row meet where the short lists were: the group whose turn it is collects
                const int collector = tile_no % NG, place_no = (group + NG - collector) % NG - 1;
                const bool has_label = mine && label >= 0 && (label / a.N + tile_no * a.col_tiles) % NG == group;
                named_barrier(1 + NG, NG * 128);
                if (place_no >= 0) {
                    unsigned char* place = pending + (size_t)(place_no * HS_ROWS + r) * MEET_ROW;
                    *reinterpret_cast<float4*>(place) = make_float4(h.m, h.s, h.u, has_label ? h.label_x : 0.f);
                    if constexpr (B > 0) {
#pragma unroll
                        for (int i = 0; i < B; ++i) reinterpret_cast<unsigned long long*>(place + 16)[i] = head_key(best.v[i], best.c[i]);
                    }
                }
                named_barrier(1 + NG, NG * 128);
                if (place_no >= 0) {
                    named_barrier(1 + NG, NG * 128);
                    continue;
                }
                float label_x = has_label ? h.label_x : 0.f;
                unsigned long long keys[B > 0 ? B : 1];
                if constexpr (B > 0) {
#pragma unroll
                    for (int i = 0; i < B; ++i) keys[i] = head_key(best.v[i], best.c[i]);
                }
                for (int o = 0; o < NG - 1; ++o) {
                    const unsigned char* other = pending + (size_t)(o * HS_ROWS + r) * MEET_ROW;
                    const float4 f = *reinterpret_cast<const float4*>(other);
                    HeadRow oh{f.x, f.y, f.z, 0.f};
                    h.merge(oh, c);
                    label_x += f.w;
                    if constexpr (B > 0) {
                        unsigned long long k[B];
#pragma unroll
                        for (int i = 0; i < B; ++i) k[i] = reinterpret_cast<const unsigned long long*>(other + 16)[i];
                        merge_keys<B>(keys, k);
                    }
                }
                if constexpr (B > 0) best.from_keys(keys);
                h.label_x = label_x;
                named_barrier(1 + NG, NG * 128);           // the place is free
            }
            const RowSums sums = row_sums(h.m, h.s, h.u);
            if (row < a.s.n) write_row(a.s, row, sums, label, h.label_x);
            if constexpr (B > 0) {
                const bool nan = h.s != h.s, wide = wide_lists(a.s);
                if (row < a.s.n) {
                    write_list<B>(a.s.top_class + row * a.s.top, a.s.top, wide, [&](int i) { return nan || best.v[i] == -INFINITY ? -1 : best.c[i]; });
                    write_list<B>(a.s.top_logp + row * a.s.top, a.s.top, wide, [&](int i) {
                        return nan ? NAN : (best.v[i] > -INFINITY ? log_prob_of(sums, best.v[i], a.s.inv_t) : -INFINITY);
                    });
                }
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        fence_after_sync();
        tmem_dealloc(tmem, columns);
    }
    if (lane == 0 && (!ok || (tid == 0 && *abort))) atomicOr(a.s.status, PTV3_STATUS_WAIT_LIMIT);
}

// shared memory beside the features and W
static size_t head_extra(int NG, int B, int N, int col_tiles)
{
    const size_t pending = B ? (size_t)NG * 4 * HS_AREA * 4 : 0, meet = col_tiles > 1 ? (size_t)(NG - 1) * HS_ROWS * (16 + B * 8) : 0;
    return (size_t)NG * N * 4 + (pending > meet ? pending : meet) + 8 * (2 * 32 + 2 * 8 + 2 * NG + 1) + 16 + 1024;
}
constexpr size_t HS_SMEM = 227 * 1024;

template <int NG, int B>
static int launch_head(const void* feat, const void* weight, HeadArgs a, int channels, cudaStream_t stream)
{
    // Classes of a tile: as many as the accumulators leave, half of it where fewer than four pieces of W would fit beside the features.
    const size_t x_tile = (size_t)a.chunks * HS_X_BYTES;
    size_t room = 0, w_piece = 0;
    for (a.N = a.s.K <= 32 ? 32 : a.s.K <= 64 ? 64 : a.s.K <= 128 ? 128 : NG == 2 ? 256 : 128;; a.N /= 2) {
        a.col_tiles = (a.s.K + a.N - 1) / a.N;
        room = HS_SMEM - head_extra(NG, B, a.N, a.col_tiles);
        w_piece = (size_t)a.N * HS_BK * 2;
        if (a.N <= 128 || x_tile + 4 * w_piece <= room) break;
    }
    // Features of a tile and of as much of the next as there is room for; W whole where it fits, else a ring of its pieces.
    const size_t w_whole = w_piece * a.chunks * a.col_tiles;
    if (w_whole <= 96 * 1024 && w_whole + x_tile <= room) {
        a.w_stages = 0;
        a.x_stages = (int)((room - w_whole) / HS_X_BYTES);
    } else {
        const bool two = 2 * x_tile + 4 * w_piece <= room;
        a.x_stages = two ? 2 * a.chunks : a.chunks;
        a.w_stages = (int)((room - a.x_stages * (size_t)HS_X_BYTES) / w_piece);
        a.w_stages = a.w_stages > 8 ? 8 : a.w_stages;
        PTV3_REQUIRE(a.w_stages >= 2, PTV3_ERR_UNSUPPORTED, "ptv3_seg_head_scores_fwd: %d channels do not fit shared memory", channels);
    }
    a.x_stages = a.x_stages > 4 * a.chunks ? 4 * a.chunks : a.x_stages;
    a.x_stages = a.x_stages > 32 ? 32 : a.x_stages;
    const size_t smem = head_extra(NG, B, a.N, a.col_tiles) + (size_t)a.x_stages * HS_X_BYTES + (a.w_stages ? a.w_stages * w_piece : w_whole);
    CUtensorMap mx, mw;
    int rc = make_tensor_map_bf16(&mx, feat, (uint64_t)a.s.n, (uint64_t)channels, (uint64_t)channels * 2, HS_ROWS, HS_BK);
    if (rc) return rc;
    rc = make_tensor_map_bf16(&mw, weight, (uint64_t)a.s.K, (uint64_t)channels, (uint64_t)channels * 2, (uint32_t)a.N, HS_BK);
    if (rc) return rc;
    auto kern = head_scores_kernel<NG, B>;
    if (allow_smem(kern) != cudaSuccess) return check_launch("ptv3_seg_head_scores_fwd: shared memory attribute");
    const unsigned grid = (unsigned)(a.row_tiles < SMS ? a.row_tiles : SMS);
    launch_dependent(kern, dim3(grid), dim3(64 + NG * 128), smem, stream, mx, mw, a);
    count_launches(1);
    return check_launch("ptv3_seg_head_scores_fwd");
}

}  // namespace ptv3

extern "C" int ptv3_seg_head_scores_fwd(const void* feat, const void* weight, const void* bias, const void* labels, int label_bytes,
                                        int64_t ignore, float* log_prob, float* entropy, float* top_log_prob, int32_t* top_class,
                                        int64_t n, int channels, int classes, int top, float temperature, int dtype,
                                        uint32_t* status, void* stream)
{
    using namespace ptv3;
    const char* what = "ptv3_seg_head_scores_fwd";
    PTV3_REQUIRE(n >= 0 && n < (1ll << 31) - HS_ROWS, PTV3_ERR_INVALID_ARGUMENT, "%s: n out of range", what);
    PTV3_REQUIRE(dtype == PTV3_DTYPE_BF16, PTV3_ERR_UNSUPPORTED, "%s: bf16 only (dtype %d)", what, dtype);
    PTV3_REQUIRE(classes >= 1 && classes <= CLASSES_MAX, PTV3_ERR_UNSUPPORTED, "%s: %d classes (1..%d)", what, classes, CLASSES_MAX);
    PTV3_REQUIRE(channels >= 8 && channels <= 512 && channels % 8 == 0, PTV3_ERR_UNSUPPORTED, "%s: %d channels (a multiple of 8 up to 512)",
                 what, channels);
    PTV3_REQUIRE(top >= 0 && top <= PTV3_HEAD_TOP_MAX, PTV3_ERR_UNSUPPORTED, "%s: %d alternatives (0..%d)", what, top, PTV3_HEAD_TOP_MAX);
    PTV3_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, PTV3_ERR_INVALID_ARGUMENT, "%s: temperature out of range", what);
    PTV3_REQUIRE(!labels || label_bytes == 4 || label_bytes == 8, PTV3_ERR_INVALID_ARGUMENT, "%s: labels of %d bytes", what, label_bytes);
    if (n == 0) return PTV3_OK;
    PTV3_REQUIRE(feat && weight && status && entropy && (!log_prob || labels) && (top == 0 || (top_log_prob && top_class)),
                 PTV3_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    PTV3_REQUIRE((((uintptr_t)feat | (uintptr_t)weight) & 15) == 0 && ((uintptr_t)bias & 1) == 0, PTV3_ERR_INVALID_ARGUMENT,
                 "%s: features and weights must be 16-byte aligned", what);
    PTV3_REQUIRE((((uintptr_t)log_prob | (uintptr_t)entropy | (uintptr_t)top_log_prob | (uintptr_t)top_class | (uintptr_t)status) & 3) == 0 &&
                     (!labels || (uintptr_t)labels % label_bytes == 0),
                 PTV3_ERR_INVALID_ARGUMENT, "%s: unaligned labels or outputs", what);
    HeadArgs a{};
    a.s.n = n;
    a.s.labels = log_prob ? labels : nullptr;
    a.s.label_bytes = label_bytes;
    a.s.ignore = ignore;
    a.s.logp = log_prob;
    a.s.entropy = entropy;
    a.s.top_logp = top_log_prob;
    a.s.top_class = top_class;
    a.s.K = classes;
    a.s.top = top;
    a.s.inv_t = (float)(1.0 / temperature);
    a.s.status = status;
    a.bias = (const __nv_bfloat16*)bias;
    a.chunks = (channels + HS_BK - 1) / HS_BK;
    a.last_steps = (channels - (a.chunks - 1) * HS_BK + 15) / 16;
    a.row_tiles = (int)((n + HS_ROWS - 1) / HS_ROWS);
    // Groups of warps: a thread's best take registers (four groups leave 96 to a thread, three 128), the words of
    // their warps shared memory that wide features need for W.
    const cudaStream_t s = (cudaStream_t)stream;
    if (top == 0) return launch_head<4, 0>(feat, weight, a, channels, s);
    if (top <= 8 && a.chunks <= 4) return launch_head<3, 8>(feat, weight, a, channels, s);
    if (top <= 8) return launch_head<2, 8>(feat, weight, a, channels, s);
    if (top <= 16) return launch_head<3, 16>(feat, weight, a, channels, s);
    return launch_head<2, 32>(feat, weight, a, channels, s);
}
