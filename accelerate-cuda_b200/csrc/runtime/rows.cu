/*
 * rows.cu -- operators over rows of scores: the best entries of a row
 * (accb_top_rows), one index drawn from a row (accb_sample_rows), and the
 * divergence of a row from a teacher's best entries with its gradient
 * (accb_distill_rows, accb_distill_rows_backward).
 *
 * They stand beside the folds over rows (fold.cuh): a matrix comes in, every
 * row is reduced.  rows.cuh says how a row is held on chip.
 */
#include <algorithm>

#include "common.h"
#include "rows.cuh"

namespace accb_rows {

struct RowsIn {
    const void *x;
    long long rows, pitch; /* pitch in elements */
    int cols;
};

/* ----------------------------------------------------- finding candidates */
/* A vector of a row as this block sees it: entries that `bits` does not allow are -inf. */
template <class T> __device__ __noinline__ uint4 only_allowed(uint4 w, int e0, int n, const unsigned *bits) {
    constexpr int E = Elem<T>::E;
    float f[E];
    Elem<T>::unpack(w, f);
    unsigned m = 0;
    if (e0 >= 0 && e0 + E <= n) {
        const unsigned lo = bits[e0 >> 5], hi = (e0 & 31) + E > 32 ? bits[(e0 >> 5) + 1] : 0u;
        m = __funnelshift_r(lo, hi, e0 & 31);
    } else {
        for (int i = 0; i < E; ++i)
            if (e0 + i >= 0 && e0 + i < n) m |= ((bits[(e0 + i) >> 5] >> ((e0 + i) & 31)) & 1u) << i;
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (!((m >> i) & 1u)) f[i] = neg_inf();
    return Elem<T>::pack(f);
}

/* Lists the entries of the row that are not below `least` (finite) in `list` of the block `to` of the cluster, which
 * finishes the row: a part of `room / size` places for every block.  `most` is the largest of this thread's scores:
 * where few threads have any such entry, a warp looks through their vectors together, a lane each.  `own`, zero
 * before, counts this block's; a block lists its own first, since a place in its own shared memory costs a fraction of
 * one in another block's.  The counts still have to be told; returns this block's. */
template <class T, bool R, class Raw>
__device__ unsigned gather(const Share<T, R> &share, Raw raw, float most, float least, u64 *mine, u64 *list, unsigned room, unsigned &own,
                           unsigned rank, unsigned size, unsigned to) {
    constexpr int E = Elem<T>::E;
    const unsigned part = room / size;
    const int lane = threadIdx.x & 31, start = share.first - lane;
    /* a round: lane by lane of those that have any, or vector by vector of all lanes, whichever takes fewer */
    unsigned have = __ballot_sync(~0u, most >= least);
    const bool by_lane = 32 * __popc(have) < share.last - start;
    const int far = by_lane ? 32 * 32 : 32;
    int v = start + lane;
    for (;;) {
        if (by_lane) {
            if (!have) break;
            v = start + __ffs(have) - 1 + 32 * lane;
            have &= have - 1;
        }
        for (; v < share.last; v += far) {
            const uint4 w = raw(v);
            typename Elem<T>::Max largest;
            largest.add(w);
            if (!(largest.get() >= least)) continue;
            float f[E];
            Elem<T>::unpack(w, f);
            unsigned found = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) found |= (unsigned)(f[i] >= least) << i;
            unsigned at = atomicAdd(&own, __popc(found));
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (((found >> i) & 1u) && at < part) mine[at++] = entry_of(f[i], share.entry(v) + i);
        }
        if (!by_lane) break;
    }
    __syncthreads();
    const unsigned n = own, base = peer_addr(shared_addr(list + rank * part), to);
    for (unsigned i = threadIdx.x; i < min(n, part); i += kThreads) peer_store1(base + i * 8, mine[i]);
    return n;
}

/* Puts the parts of a list side by side, by all threads of its block; parts hold counts(0 .. size - 1) entries. */
template <class C> __device__ void close_up(u64 *list, unsigned room, unsigned size, C counts) {
    const unsigned part = room / size;
    unsigned at = counts(0);
    for (unsigned r = 1; r < size; ++r) { /* a part moves down by less than it is away: entries first, then places */
        const unsigned n = counts(r);
        for (unsigned i0 = 0; i0 < n; i0 += kThreads) {
            const unsigned i = i0 + threadIdx.x;
            u64 e = 0;
            if (i < n) e = list[r * part + i];
            __syncthreads();
            if (i < n) list[at + i] = e;
            __syncthreads();
        }
        at += n;
    }
}

/* One message of every block to all blocks of its cluster, and the barrier after it; every exchange of a launch has a
 * buffer of its own. */
struct Told {
    alignas(16) u64 block[4][kMaxCluster][2];
};
__device__ __forceinline__ void tell_all(u64 (&buffer)[kMaxCluster][2], u64 a, u64 b, unsigned rank, unsigned size) {
    if (threadIdx.x < size) peer_store(peer_addr(shared_addr(&buffer[rank][0]), threadIdx.x), a, b);
    cluster_sync(size);
}

/* sums over the block, the same in all threads; two barriers */
__device__ __forceinline__ u64 block_sum(u64 v, u64 *scratch) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 s = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += scratch[w];
    __syncthreads();
    return s;
}
/* sum over the threads before this one and itself */
__device__ __forceinline__ u64 block_scan(u64 v, u64 *scratch) {
    v = warp_scan(v);
    if ((threadIdx.x & 31) == 31) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int w = 0; w < (int)(threadIdx.x >> 5); ++w) v += scratch[w];
    __syncthreads();
    return v;
}

/* ------------------------------------------------------------- sampling */
struct SampleParams {
    RowsIn in;
    const unsigned *allowed; /* bit j % 32 of word j / 32: entry j may be drawn; or null */
    long long allowed_pitch; /* words */
    const float *uniform, *temperature, *top_p, *min_p;
    const int *top_k;
    int *token;
    float *logprob;
};
constexpr int kSampleRoom = 512; /* candidates of a row that a block lists and sorts, ... */
constexpr int kListed = 192;     /* ... asked for where top_k is no more */

/* A row whose candidates are listed and that waits for its block to draw from them. */
struct PendingDraw {
    long long row;
    u64 total;
    double temperature;
    float most, lowest, top_p, uniform;
    int k;
    unsigned n[kMaxCluster]; /* candidates by block */
};

/* the whole part of uniform * total below total */
__device__ __forceinline__ u64 drawn(float uniform, u64 total) {
    const double want = floor((double)uniform * (double)total);
    return want > 0.0 ? min((u64)want, total - 1) : 0;
}

__device__ __forceinline__ void put_token(const SampleParams &p, long long row, int index, float value, float most, double temperature, u64 total) {
    p.token[row] = index;
    if (p.logprob) {
        const double below = value == most ? 0.0 : ((double)value - (double)most) / temperature;
        p.logprob[row] = (float)(below - log_64((double)total * (1.0 / (double)(1ull << kUnitLog2))));
    }
}

/* Draws from the candidates in `list`, which hold every entry that top_k and top_p could keep; by one block. */
template <class W> __device__ __noinline__ void draw_from_list(const SampleParams &p, const PendingDraw &d, u64 *list, u64 *scratch, unsigned size, const double *table) {
    const W weigh(d.most, d.temperature, table);
    const int k = d.k;
    const float top_p = d.top_p, lowest = d.lowest;
    u64 total = d.total;
    int n = 0;
    for (unsigned r = 0; r < size; ++r) n += (int)d.n[r];
    close_up(list, kSampleRoom, size, [&](unsigned r) { return d.n[r]; });
    __syncthreads();
    sort_down(list, n, kSampleRoom);
    if (k > 0) n = min(n, k);
    /* weights, and how many of the sorted candidates are kept: a thread has `per` of them side by side */
    const int per = (n + kThreads - 1) / kThreads, from = min(n, (int)threadIdx.x * per), to = min(n, from + per);
    u64 mine = 0;
    for (int i = from; i < to; ++i) mine += weigh.weight(score_of(list[i]));
    u64 upto = block_scan(mine, scratch);
    if (total == 0) total = block_sum(mine, scratch);
    const u64 limit = top_p < 1.0f ? (u64)ceil((top_p > 0.0f ? (double)top_p : 0.0) * (double)total) : ~0ull;
    u64 before = upto - mine, kept = 0;
    for (int i = from; i < to; ++i) {
        const float x = score_of(list[i]);
        const u64 w = weigh.weight(x);
        const bool keep = (before < limit || i == 0) && x >= lowest;
        before += w;
        kept += keep ? w : 0;
        /* next: in the order of the indices, without the keys of those that are not kept */
        list[i] = list[i] << 32 | (keep ? key_of(x) : 0u);
    }
    total = block_sum(kept, scratch);
    const u64 target = drawn(d.uniform, total);
    sort_down(list, n, kSampleRoom);
    mine = 0;
    for (int i = from; i < to; ++i)
        if ((unsigned)list[i]) mine += weigh.weight(value_of((unsigned)list[i]));
    upto = block_scan(mine, scratch);
    before = upto - mine;
    if (before <= target && target < upto) {
        for (int i = from; i < to; ++i) {
            const float x = value_of((unsigned)list[i]);
            if ((unsigned)list[i]) before += weigh.weight(x);
            if (target < before) {
                put_token(p, d.row, index_of(list[i] >> 32), x, d.most, d.temperature, total);
                return;
            }
        }
    }
}

template <class T, bool R> __global__ void __launch_bounds__(kThreads, 3) sample_rows(const __grid_constant__ SampleParams p) {
    constexpr int E = Elem<T>::E;
    extern __shared__ uint4 stage[];
    __shared__ Told told_by_turns[2];
    __shared__ union {
        u64 mine[kSampleRoom];
        FineBins bins;
        Level level;
    } sh;
    __shared__ u64 list[kSampleRoom];
    __shared__ u64 warp_part[kWarps][2];
    __shared__ double table[kTable * kTableCopies];
    __shared__ u64 scratch[kWarps];
    __shared__ unsigned own;
    __shared__ PendingDraw pending;
    __shared__ Extent extent;
    const unsigned size = cluster_size(), rank = cluster_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T *x = static_cast<const T *>(p.in.x);
    const long long step = gridDim.x / size;
    if (size > 1) cluster_arrive(); /* every block of the cluster has started: waited for before the first message */

    Share<T, R> share;
    share.init(x + (blockIdx.x / size) * p.in.pitch, p.in.cols, rank, size, stage);
    share.fetch();
    fill_table(table);
    if (size > 1) cluster_wait();
    int turn = 0;
    unsigned finisher = 0; /* the block that draws from this row's list: blocks take it in turns and draw side by side */
    bool waiting = false;  /* a list waits in this block */
    for (long long row = blockIdx.x / size; row < p.in.rows; row += step, turn ^= 1) {
    Told &told = told_by_turns[turn];
    const bool more = row + step < p.in.rows;
    auto draw = [&] {
        if (!waiting) return;
        draw_from_list<Weigh<sizeof(T) == 4>>(p, pending, list, scratch, size, table);
        waiting = false;
        __syncthreads(); /* the list is used again */
    };
    auto next = [&] { /* the scores of the next row take the place of this one's, which this thread has read */
        if (!more) return;
        share.init(x + (row + step) * p.in.pitch, p.in.cols, rank, size, stage);
        share.fetch();
    };
    const unsigned *bits = p.allowed ? p.allowed + row * p.allowed_pitch : nullptr;
    float warmth = p.temperature ? p.temperature[row] : 1.0f;
    int k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f;
    const float min_p = p.min_p ? p.min_p[row] : 0.0f;
    const float uniform = p.uniform[row];
    if (!(warmth > 0.0f)) k = 1;
    const double temperature = warmth > 0.0f ? warmth : 1.0f;
    if (k >= p.in.cols || k < 0) k = 0;
    if (threadIdx.x == 0) own = 0;
    share.wait();

    bool infinite = false; /* the row's maximum is +inf: its like weigh 1, all others nothing */
    auto raw = [&](int v) {
        uint4 w = share.get(v);
        if (!R) {
            if (bits) w = only_allowed<T>(w, share.entry(v), share.n, bits);
            if (infinite) {
                float f[E];
                Elem<T>::unpack(w, f);
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] = f[i] == __uint_as_float(0x7f800000u) ? 0.0f : neg_inf();
                w = Elem<T>::pack(f);
            }
        }
        return w;
    };
    auto get = [&](int v, float *f) {
        Elem<T>::unpack(raw(v), f);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = not_nan(f[i]);
    };

    /* the maximum, and where at least k entries lie above: a k-th part of the blocks' threads in each block */
    typename Elem<T>::Max largest;
#pragma unroll 4
    for (int v = share.first; v < share.last; v += 32) {
        uint4 w = raw(v);
        if (R && bits) stage[v - share.v0] = w = only_allowed<T>(w, share.entry(v), share.n, bits);
        largest.add(w);
    }
    float thread_most = largest.get();
    const float2 ext = extent_of(thread_most, k > 1 ? (k + (int)size - 1) / (int)size : 0, extent);
    float most = ext.x, bound = ext.y;
    tell_all(told.block[0], __float_as_uint(most), __float_as_uint(bound), rank, size);
    for (int i = 0; i < (int)size; ++i) {
        most = fmaxf(most, __uint_as_float((unsigned)told.block[0][i][0]));
        bound = fminf(bound, __uint_as_float((unsigned)told.block[0][i][1]));
    }
    if (most == neg_inf()) { /* nothing may be drawn: the same in every block of the row */
        if (rank == 0 && threadIdx.x == 0) {
            p.token[row] = -1;
            if (p.logprob) p.logprob[row] = neg_inf();
        }
        next();
        if (!more) draw();
        continue;
    }
    if (most == __uint_as_float(0x7f800000u)) {
        if (R) {
            for (int v = share.first; v < share.last; v += 32) {
                float f[E];
                get(v, f);
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] = f[i] == most ? 0.0f : neg_inf();
                stage[v - share.v0] = Elem<T>::pack(f);
            }
        }
        infinite = true;
        most = 0.0f, bound = neg_inf(), thread_most = thread_most == __uint_as_float(0x7f800000u) ? 0.0f : neg_inf();
    }

    /* the lowest score that min_p keeps */
    float lowest = -3.402823466e+38f;
    if (min_p > 0.0f) {
        const double low = (double)most + log_64(fmin((double)min_p, 1.0)) * temperature;
        if (low > -3.0e38) lowest = __double2float_ru(low);
    }
    const Weigh<sizeof(T) == 4> weigh(most, temperature, table);
    if (k == 1) bound = most;

    /* weight above a border and number of entries on it, of this thread: the weight in quarters of the warp's piece,
     * which are kept to find the token's */
    u64 quarter[4];
    unsigned ties = 0;
    const int start = share.first - lane; /* of the warp's piece */
    const int per_quarter = (max(0, share.last - start) + 127) >> 7;
    auto pass = [&](const Border &border, bool most_count) {
        const float above = value_of(max(border.key, key_of(-3.402823466e+38f) - 1u)), on = value_of(border.key);
        const bool count = border.ties != 0;
        const float from = fmaxf(weigh.least, value_of(border.key + 1u));
        ties = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            quarter[q] = 0;
            const int end = min(share.last, share.first + 32 * per_quarter * (q + 1));
#pragma unroll 1
            for (int v = share.first + 32 * per_quarter * q; v < end; v += 32) {
                const uint4 w = raw(v);
                typename Elem<T>::Max best;
                best.add(w);
                if (!(most_count ? best.get() >= from : count ? best.get() >= on : best.get() > above)) continue;
                float f[E];
                Elem<T>::unpack(w, f);
                if (most_count) { /* without a branch: the weights of a vector are computed side by side */
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const u64 x = weigh.of(f[i]);
                        quarter[q] += f[i] >= from ? x : 0;
                    }
                    continue;
                }
                quarter[q] += weigh.template some<E>(f, [&](float x) { return x > above; });
                if (count) {
#pragma unroll
                    for (int i = 0; i < E; ++i) ties += f[i] == on;
                }
            }
        }
    };
    u64 total = 0;
    const bool cut = k > 0 || top_p < 1.0f;
    BlockPart part{0, 0, false};
    bool passed = false;
    Border border{key_of(cut ? -3.402823466e+38f : lowest) - 1u, 0, 0}; /* without cuts: of min_p */
    if (cut) {
        float least = fmaxf(bound, -3.402823466e+38f);
        bool listed = k > 0 && k <= kListed;
        if (k == 0) { /* top_p alone */
            least = weigh.least;
            /* counts by bin say what a row of bfloat16 weighs; else, or where min_p leaves few to list, a pass does, and
             * how far down entries lie that all of them together weigh less than what is cut off */
            if (Elem<T>::kShift != 16 || min_p > 0.0f) {
                pass(border, true);
                const u64 block_total = block_sum((quarter[0] + quarter[1]) + (quarter[2] + quarter[3]), scratch);
                tell_all(told.block[1], block_total, 0, rank, size);
                for (int i = 0; i < (int)size; ++i) total += told.block[1][i][0];
                const double left = (1.0 - (double)top_p) * ((double)total * (1.0 / (double)(1ull << kUnitLog2)));
                const double low = (double)most + (log_64(left / (double)p.in.cols) - 0.01) * temperature;
                if (left > 1e-5 && low > (double)least) least = __double2float_rd(low);
                listed = true;
            }
        }
        /* what min_p drops is not needed to weigh the rest, unless top_p takes its share of what top_k keeps */
        const float above = k == 0 || !(top_p < 1.0f) ? fmaxf(least, lowest) : least;
        if (listed) {
            const unsigned n = gather(share, raw, thread_most, above, sh.mine, list, kSampleRoom, own, rank, size, finisher);
            tell_all(told.block[2], n, 0, rank, size);
            unsigned longest = 0;
            for (int i = 0; i < (int)size; ++i) longest = max(longest, (unsigned)told.block[2][i][0]);
            if (longest <= kSampleRoom / size) { /* the same in every block of the row */
                next();
                if (rank == finisher) {
                    waiting = true;
                    if (threadIdx.x < size) pending.n[threadIdx.x] = (unsigned)told.block[2][threadIdx.x][0];
                    if (threadIdx.x == 0) {
                        pending.row = row, pending.total = total, pending.temperature = temperature, pending.most = most;
                        pending.lowest = lowest, pending.top_p = top_p, pending.uniform = uniform, pending.k = k;
                    }
                    __syncthreads();
                }
                finisher = finisher + 1 == size ? 0 : finisher + 1;
                if (finisher == 0 || !more) draw();
                continue;
            }
        }
        /* too many for a list */
        border = k == 1 ? Border{key_of(most), 1, 1}
                        : border_by_bins<T, R>(share, raw, get, sh.bins, sh.level, size, weigh, k > 0 ? least : weigh.least, most, (u64)k,
                                               top_p < 1.0f ? (top_p > 0.0f ? (double)top_p : 0.0) : 1.0, total, part);
        const unsigned below = key_of(lowest) - 1u;
        if (below >= border.key) border = Border{below, 0, 0}, part.known = false;
    }

    /* what every block holds of what is kept; the token lies in the one that its random number points to */
    if (!part.known) {
        pass(border, !cut);
        passed = true;
        part.mass = block_sum((quarter[0] + quarter[1]) + (quarter[2] + quarter[3]), scratch);
        part.ties = border.ties ? (unsigned)block_sum(ties, scratch) : 0;
    }
    tell_all(told.block[3], part.mass, part.ties, rank, size);
    const u64 tie_weight = border.ties ? weigh.weight(value_of(border.key)) : 0;
    u64 before = 0, here = 0;
    unsigned ties_seen = 0, quota = 0;
    total = 0;
    for (int i = 0; i < (int)size; ++i) {
        const unsigned n = (unsigned)told.block[3][i][1], kept = min(ties_seen + n, border.ties) - min(ties_seen, border.ties);
        const u64 w = told.block[3][i][0] + kept * tie_weight;
        if (i == (int)rank) before = total, here = w, quota = kept;
        total += w, ties_seen += n;
    }
    /* the first entry whose running sum exceeds uniform * total */
    const u64 target = drawn(uniform, total);
    if (!more) draw();
    if (!(before <= target && target < before + here)) { /* in another block */
        next();
        continue;
    }
    if (!passed) pass(border, false);
    {
        const u64 mass = warp_sum((quarter[0] + quarter[1]) + (quarter[2] + quarter[3]));
        const unsigned n = warp_sum(ties);
        if (lane == 0) warp_part[warp][0] = mass, warp_part[warp][1] = n;
        __syncthreads();
        unsigned seen = 0, block_quota = quota;
        for (int w = 0; w <= warp; ++w) {
            const unsigned m = (unsigned)warp_part[w][1];
            quota = min(seen + m, block_quota) - min(seen, block_quota);
            here = warp_part[w][0] + quota * tie_weight;
            if (w < warp) before += here;
            seen += m;
        }
        __syncthreads();
    }
    if (!(before <= target && target < before + here)) { /* in another warp's piece */
        next();
        continue;
    }

    int v0 = start;
    if (quota == 0) { /* which quarter of the warp's piece */
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const u64 w = warp_sum(quarter[q]);
            if (v0 == start + 32 * per_quarter * q && before + w <= target) before += w, v0 += 32 * per_quarter;
        }
    }
    unsigned left = quota;
    u64 sum = before;
    for (; v0 < share.last; v0 += 32) {
        const int v = v0 + lane;
        float f[E];
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = neg_inf();
        if (v < share.last) get(v, f);
        unsigned n = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) n += key_of(f[i]) == border.key && v < share.last;
        const unsigned upto = warp_scan(n);
        unsigned may = left > upto - n ? left - (upto - n) : 0;
        u64 w[E], mine = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const unsigned key = key_of(f[i]);
            w[i] = 0;
            if (key > border.key) {
                w[i] = weigh.weight(f[i]);
            } else if (key == border.key && may) {
                w[i] = tie_weight;
                --may;
            }
            mine += w[i];
        }
        const u64 reach = sum + warp_scan(mine);
        const unsigned hit = __ballot_sync(~0u, target < reach);
        if (hit) {
            if (lane == __ffs(hit) - 1) {
                u64 c = reach - mine;
                int at = 0;
                float value = 0.0f;
                bool done = false;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    c += w[i];
                    if (!done && target < c) at = share.entry(v) + i, value = f[i], done = true;
                }
                put_token(p, row, at, value, most, temperature, total);
            }
            break;
        }
        sum = __shfl_sync(~0u, reach, 31);
        const unsigned took = __shfl_sync(~0u, upto, 31);
        left = left > took ? left - took : 0;
    }
    next();
    }
}

/* ---------------------------------------------------------- best entries */
struct TopParams {
    RowsIn in;
    void *values;
    int *index;
    float *lse;
    double temperature;
    int k;
    int room; /* of the list of candidates, a power of two from 256 */
};

template <class T, bool R> __global__ void __launch_bounds__(kThreads, 3) top_rows(const __grid_constant__ TopParams p) {
    constexpr int E = Elem<T>::E;
    extern __shared__ uint4 dynamic[];
    __shared__ Told told_by_turns[2];
    __shared__ u64 scratch[kWarps];
    __shared__ unsigned own, taken, counts[kMaxCluster];
    __shared__ u64 ties_of[kMaxCluster * kWarps]; /* entries on the border, by warp */
    __shared__ Extent extent;
    const unsigned size = cluster_size(), rank = cluster_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    u64 *list = reinterpret_cast<u64 *>(dynamic), *mine = list + p.room; /* `mine`: room / size places, or a Level */
    Level &level = *reinterpret_cast<Level *>(mine);
    const T *x = static_cast<const T *>(p.in.x);
    const long long step = gridDim.x / size;
    if (size > 1) cluster_arrive(); /* every block of the cluster has started: waited for before the first message */

    Share<T, R> share;
    share.init(x + (blockIdx.x / size) * p.in.pitch, p.in.cols, rank, size, dynamic + (p.room + max(p.room / (int)size, (int)sizeof(Level) / 8)) / 2);
    share.fetch();
    if (size > 1) cluster_wait();
    int turn = 0;
    unsigned finisher = 0;       /* the block that sorts this row's list: blocks take it in turns and sort side by side */
    long long waiting = -1;      /* the row whose list waits in this block */
    for (long long row = blockIdx.x / size; row < p.in.rows; row += step, turn ^= 1) {
    Told &told = told_by_turns[turn];
    const bool more = row + step < p.in.rows;
    if (threadIdx.x == 0) own = taken = 0;
    share.wait();
    auto raw = [&](int v) { return share.get(v); };
    auto get = [&](int v, float *f) {
        Elem<T>::unpack(share.get(v), f);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = not_nan(f[i]);
    };
    auto next = [&] { /* the scores of the next row take the place of this one's, which this thread has read */
        if (!more) return;
        share.init(x + (row + step) * p.in.pitch, p.in.cols, rank, size, share.stage);
        share.fetch();
    };
    typename Elem<T>::Max largest;
#pragma unroll 4
    for (int v = share.first; v < share.last; v += 32) largest.add(share.get(v));
    /* threads of each block whose maxima make up k entries */
    const float thread_most = largest.get();
    const float2 ext = extent_of(thread_most, (p.k + (int)size - 1) / (int)size, extent);
    float most = ext.x, bound = ext.y;
    tell_all(told.block[0], __float_as_uint(most), __float_as_uint(bound), rank, size);
    for (int i = 0; i < (int)size; ++i) {
        most = fmaxf(most, __uint_as_float((unsigned)told.block[0][i][0]));
        bound = fminf(bound, __uint_as_float((unsigned)told.block[0][i][1]));
    }
    unsigned n = 0, longest = 0;
    double sum = 0.0;
    if (most > neg_inf()) {
        if (p.lse) {
            const float c = (float)(1.4426950408889634 / p.temperature);
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (most < __uint_as_float(0x7f800000u)) {
#pragma unroll 2
                for (int v = share.first; v < share.last; v += 32) {
                    float f[E];
                    get(v, f);
#pragma unroll
                    for (int i = 0; i < E; ++i) part[i & 3] += fast_exp2((f[i] - most) * c);
                }
            }
            const float warp_part = warp_sum((part[0] + part[1]) + (part[2] + part[3]));
            __syncthreads();
            if (lane == 0) scratch[warp] = __float_as_uint(warp_part);
        }
        n = gather(share, raw, thread_most, fmaxf(bound, -3.402823466e+38f), mine, list, (unsigned)p.room, own, rank, size, finisher);
        if (p.lse)
            for (int w = 0; w < kWarps; ++w) sum += (double)__uint_as_float((unsigned)scratch[w]);
        tell_all(told.block[1], n, (u64)__double_as_longlong(sum), rank, size);
        sum = 0.0;
        for (int i = 0; i < (int)size; ++i) longest = max(longest, (unsigned)told.block[1][i][0]), sum += __longlong_as_double((long long)told.block[1][i][1]);
    }
    if (p.lse && rank == 0 && threadIdx.x == 0)
        p.lse[row] = most > neg_inf() && most < __uint_as_float(0x7f800000u) ? (float)((double)most / p.temperature + log_64(sum)) : most;

    const bool crowded = longest > (unsigned)p.room / size;
    if (crowded) {
        /* too many (ties, or rows of few large entries side by side): find the border, then list what is above it and
         * the first of what is on it */
        const Weigh<sizeof(T) == 4> none(0.0f, 1.0, nullptr);
        const Border border = find_border<T, R, false>(share, get, level, size, key_of(bound), key_of(most), (u64)p.k, none, 0.0, 0);
        unsigned ties = 0;
        for (int v = share.first; v < share.last; v += 32) {
            float f[E];
            get(v, f);
#pragma unroll
            for (int i = 0; i < E; ++i) ties += key_of(f[i]) == border.key;
        }
        ties = warp_sum(ties);
        if (lane < (int)size) peer_store1(peer_addr(shared_addr(&ties_of[rank * kWarps + warp]), lane), ties);
        cluster_sync(size);
        unsigned quota = 0, seen = 0;
        const int nwarps = (int)size * kWarps, self = (int)rank * kWarps + warp;
        for (int i0 = 0; i0 < nwarps; i0 += 32) {
            const int i = i0 + lane;
            const unsigned m = i < nwarps ? (unsigned)ties_of[i] : 0;
            const unsigned upto = seen + warp_scan(m);
            if (i == self) quota = min(upto, border.ties) - min(upto - m, border.ties);
            seen = __shfl_sync(~0u, upto, 31);
        }
        quota = __shfl_sync(~0u, quota, self & 31);
        const unsigned lowest = key_of(neg_inf()), to = peer_addr(shared_addr(list), finisher), count = peer_addr(shared_addr(&taken), finisher);
        for (int v0 = share.first - lane; v0 < share.last; v0 += 32) {
            const int v = v0 + lane;
            float f[E];
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = neg_inf();
            if (v < share.last) get(v, f);
            unsigned on = 0, above = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const unsigned key = key_of(f[i]);
                if (key > lowest && v < share.last) on |= (unsigned)(key == border.key) << i, above |= (unsigned)(key > border.key) << i;
            }
            if (!__any_sync(~0u, on | above)) continue;
            const unsigned m = __popc(on), upto = warp_scan(m);
            unsigned may = quota > upto - m ? quota - (upto - m) : 0;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                bool take = (above >> i) & 1u;
                if (((on >> i) & 1u) && may) take = true, --may;
                if (take) {
                    const unsigned at = peer_count(count, 1);
                    if (at < (unsigned)p.k) peer_store1(to + at * 8, entry_of(f[i], share.entry(v) + i));
                }
            }
            const unsigned took = __shfl_sync(~0u, upto, 31);
            quota = quota > took ? quota - took : 0;
        }
        cluster_sync(size);
    }
    next();
    if (rank == finisher) {
        waiting = row;
        if (threadIdx.x < size) counts[threadIdx.x] = most == neg_inf() ? 0 : crowded ? (threadIdx.x == 0 ? taken : 0) : (unsigned)told.block[1][threadIdx.x][0];
        __syncthreads();
    }
    finisher = finisher + 1 == size ? 0 : finisher + 1;
    if ((finisher == 0 || !more) && waiting >= 0) {
        unsigned all = 0;
        for (unsigned r = 0; r < size; ++r) all += counts[r];
        close_up(list, (unsigned)p.room, size, [&](unsigned r) { return counts[r]; });
        __syncthreads();
        sort_down(list, (int)all, p.room);
        for (int i = threadIdx.x; i < p.k; i += kThreads) {
            const u64 e = i < (int)all ? list[i] : 0;
            static_cast<T *>(p.values)[waiting * p.k + i] = Elem<T>::down(e ? score_of(e) : neg_inf());
            p.index[waiting * p.k + i] = e ? index_of(e) : -1;
        }
        waiting = -1;
        __syncthreads(); /* the list is used again */
    }
    }
}

/* ---------------------------------------------------------- distillation */
struct DistillParams {
    RowsIn in;
    const void *teacher; /* rows x k, element type teacher_type */
    const int *index;
    const float *teacher_lse, *weight, *upstream;
    float *loss, *stats; /* stats: rows x 4, see accb_distill_rows */
    void *grad;          /* element type of the scores */
    long long grad_pitch;
    double temperature;
    int k, teacher_type;
    int map_words; /* 32-bit words of the map of named entries of a block's share */
};

__device__ __forceinline__ float teacher_value(const DistillParams &p, long long i) {
    if (p.teacher_type == ACCB_ROWS_F32) return static_cast<const float *>(p.teacher)[i];
    if (p.teacher_type == ACCB_ROWS_F16) return __half2float(static_cast<const __half *>(p.teacher)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p.teacher)[i]);
}

/* What a block keeps of an entry that the teacher names.  Probabilities are 64-bit: what they leave of 1 is the
 * difference of like numbers. */
struct Named {
    double p;
    float score; /* of the teacher */
    float z;     /* of the student, if the entry lies in this block's share */
    int at;      /* index, or -1 for an entry that names nothing or lies in another share */
    int first;   /* the first of its index that was met */
};

/* The row as all its blocks know it. */
struct RowSums {
    float top, others_top;         /* maximum of the row, and of the entries not named (-inf: none) */
    double sum, others_sum, cross; /* sums of exponentials below those maxima; sum of p (teacher's - student's score) / tau */
};

/* What the loss is computed from, by one warp of the row: its logarithms are taken by four lanes at once. */
__device__ __noinline__ float row_loss(const RowSums &all, double named, double teacher_sum, double rest, double inv) {
    const int lane = threadIdx.x & 31;
    const double of = lane == 0 ? all.sum : lane == 1 ? teacher_sum : lane == 2 ? rest : all.others_sum;
    const double l = lane < 4 ? log_64(of) : 0.0;
    const double log_sum = __shfl_sync(~0u, l, 0), log_teacher = __shfl_sync(~0u, l, 1), log_rest = __shfl_sync(~0u, l, 2),
                 log_others = __shfl_sync(~0u, l, 3);
    const double lse = (double)all.top * inv + log_sum;
    double loss = all.cross + named * (lse - log_teacher);
    if (rest > 0.0) loss += rest * (log_rest - ((double)all.others_top * inv + log_others - lse));
    return (float)loss;
}

/* BACKWARD: the statistics are given, and no block needs the others. */
template <class T, bool R, bool BACKWARD> __global__ void __launch_bounds__(kThreads, 3) distill_rows(const __grid_constant__ DistillParams p) {
    constexpr int E = Elem<T>::E;
    extern __shared__ uint4 dynamic[];
    __shared__ double scratch[kWarps];
    __shared__ float warp_top[kWarps];
    __shared__ alignas(16) u64 told[kMaxCluster * kWarps][4];
    __shared__ int twice;
    Named *named = reinterpret_cast<Named *>(dynamic);
    unsigned *map = reinterpret_cast<unsigned *>(named + p.k);
    uint4 *stage = dynamic + (p.map_words * 4 + p.k * sizeof(Named) + 15) / 16;
    const unsigned size = cluster_size(), rank = cluster_rank();
    const long long row = blockIdx.x / size;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    Share<T, R> share;
    share.init(static_cast<const T *>(p.in.x) + row * p.in.pitch, p.in.cols, rank, size, stage);
    T *grad = p.grad ? static_cast<T *>(p.grad) + row * p.grad_pitch : nullptr;
    const bool same = ((reinterpret_cast<unsigned long long>(grad) ^ reinterpret_cast<unsigned long long>(share.base + share.lead)) & 15u) == 0;
    const float weight = p.weight ? p.weight[row] : 1.0f;
    float top = 0.0f, inverse = 0.0f, at_named = 0.0f, elsewhere = 0.0f;
    bool live = weight != 0.0f;
    if (BACKWARD) {
        const float *st = p.stats + row * 4;
        top = st[0], inverse = st[1], at_named = st[2], elsewhere = st[3];
        live = live && inverse != 0.0f;
    }
    if (!BACKWARD && size > 1) cluster_arrive(); /* every block of the row has started: waited for before the first message */
    const bool rest = p.teacher_lse != nullptr;
    const double inv = 1.0 / p.temperature;
    double shift = 0.0, total = 0.0, named_p = 0.0;
    float teacher_top = neg_inf();
    if (live) {
        /* the first entries are asked for before the copies of the row fill the queues */
        int index = -1;
        float score = neg_inf();
        if ((int)threadIdx.x < p.k) index = p.index[row * p.k + threadIdx.x], score = teacher_value(p, row * p.k + threadIdx.x);
        if (rest) shift = p.teacher_lse[row];
        share.fetch();
        for (int i = threadIdx.x; i < p.map_words; i += kThreads) map[i] = 0;
        if (threadIdx.x == 0) twice = 0;
        for (int j = threadIdx.x; j < p.k; j += kThreads) {
            if (j >= kThreads) index = p.index[row * p.k + j], score = teacher_value(p, row * p.k + j);
            const bool names = index >= 0 && index < p.in.cols && score > neg_inf();
            named[j].at = names ? index : -1;
            named[j].score = score;
            if (names) teacher_top = fmaxf(teacher_top, score);
        }
        teacher_top = warp_max(teacher_top);
        if (lane == 0) warp_top[warp] = teacher_top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) teacher_top = fmaxf(teacher_top, warp_top[w]);
        live = teacher_top > neg_inf();
    }
    /* rows that do not count: nothing of the scores is looked at */
    auto nothing = [&] {
        share.wait();
        if (grad)
            for (int v = share.first; v < share.last; v += 32) put(share, grad, same, v, make_uint4(0, 0, 0, 0));
        if (!BACKWARD && rank == 0 && threadIdx.x < 4) {
            if (threadIdx.x == 0) p.loss[row] = 0.0f;
            if (p.stats) p.stats[row * 4 + threadIdx.x] = 0.0f;
        }
    };
    if (!live) {
        if (!BACKWARD && size > 1) cluster_wait();
        nothing();
        return;
    }

    /* the teacher's probabilities: exp(score / tau - shift), over their sum unless that is given with teacher_lse */
    if (!rest) shift = (double)teacher_top * inv;
    double sum_p = 0.0;
    for (int j = threadIdx.x; j < p.k; j += kThreads) {
        const double e = named[j].at >= 0 ? exp_64((double)named[j].score * inv - shift) : 0.0;
        named[j].p = e;
        sum_p += e;
    }
    if (warp * 32 < p.k) sum_p = warp_sum(sum_p);
    if (lane == 0) scratch[warp] = sum_p;
    share.wait();
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += scratch[w];
    const double norm = rest ? 1.0 : 1.0 / total;
    named_p = total * norm;

    /* which entries of the share the teacher names; an entry named twice is counted once */
    const int origin = share.entry(share.v0), width = (share.v1 - share.v0) * E;
    const float c = (float)(1.4426950408889634 / p.temperature);
    float most_named = neg_inf();
    double cross = 0.0;
    for (int j = threadIdx.x; j < p.k; j += kThreads) {
        Named &n = named[j];
        const int at = n.at, e = at - origin;
        const bool here = at >= 0 && e >= 0 && e < width;
        const double prob = n.p * norm;
        n.first = 0;
        if (here) {
            n.first = !((atomicOr(&map[e >> 5], 1u << (e & 31)) >> (e & 31)) & 1u);
            if (!n.first) twice = 1;
            n.z = R ? Elem<T>::up(reinterpret_cast<const T *>(stage)[e]) : Elem<T>::up(share.base[share.lead + at]);
            if (n.first) most_named = fmaxf(most_named, n.z);
            /* sum of p (log p - z / tau): what is left of the loss is the two log-sum-exps */
            if (prob > 0.0) cross += prob * (((double)n.score - (double)n.z) * inv);
        }
        n.p = prob;
        n.at = here ? at : -1;
    }
    __syncthreads();

    if (!BACKWARD) {
        /* the rest of the row (all of it without teacher_lse) and the named entries, each as maximum and sum */
        if (R && rest) { /* named entries leave the staged row */
            for (int j = threadIdx.x; j < p.k; j += kThreads)
                if (named[j].first) reinterpret_cast<T *>(stage)[named[j].at - origin] = Elem<T>::down(neg_inf());
            __syncthreads();
        }
        auto get = [&](int v) {
            uint4 w = share.get(v);
            if (!R && rest) {
                const int e = (v - share.v0) * E;
                const unsigned m = map[e >> 5] >> (e & 31);
                float f[E];
                Elem<T>::unpack(w, f);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if ((m >> i) & 1u) f[i] = neg_inf();
                w = Elem<T>::pack(f);
            }
            return w;
        };
        typename Elem<T>::Max largest;
#pragma unroll 4
        for (int v = share.first; v < share.last; v += 32) largest.add(get(v));
        const float most = warp_max(largest.get()), base = most > neg_inf() ? most : 0.0f;
        const Pair less(-base, -base), by(c, c);
        Pair part[2] = {Pair(0.0f, 0.0f), Pair(0.0f, 0.0f)};
#pragma unroll 2
        for (int v = share.first; v < share.last; v += 32) {
            float f[E];
            Elem<T>::unpack(get(v), f);
#pragma unroll
            for (int i = 0; i < E / 2; ++i) part[i & 1] = part[i & 1] + fast_exp2((Pair(f[2 * i], f[2 * i + 1]) + less) * by);
        }
        float part_a, part_b;
        (part[0] + part[1]).get(part_a, part_b);
        double named_sum = 0.0;
        if (warp * 32 < p.k) {
            if (rest) {
                most_named = warp_max(most_named);
                const float named_base = most_named > neg_inf() ? most_named : 0.0f;
                for (int j = threadIdx.x; j < p.k; j += kThreads)
                    if (named[j].first) named_sum += (double)fast_exp2((named[j].z - named_base) * c);
                named_sum = warp_sum(named_sum);
            }
            cross = warp_sum(cross);
        }
        const double others = warp_sum((double)part_a + (double)part_b);
        if (size > 1) cluster_wait();
        if (lane < (int)size) {
            const unsigned to = peer_addr(shared_addr(&told[rank * kWarps + warp][0]), lane);
            peer_store(to, __double_as_longlong(others), __double_as_longlong(named_sum));
            peer_store(to + 16, __double_as_longlong(cross), (u64)__float_as_uint(most) << 32 | __float_as_uint(rest ? most_named : neg_inf()));
        }
        cluster_sync(size);
        if (!grad && rank != 0) return;
        /* every warp adds up what all warps of the row found */
        const int n = (int)size * kWarps;
        RowSums all{neg_inf(), neg_inf(), 0.0, 0.0, 0.0};
        for (int i = lane; i < n; i += 32) {
            all.others_top = fmaxf(all.others_top, __uint_as_float((unsigned)(told[i][3] >> 32)));
            all.top = fmaxf(all.top, __uint_as_float((unsigned)told[i][3]));
        }
        all.others_top = warp_max(all.others_top), all.top = fmaxf(all.others_top, warp_max(all.top));
        for (int i = lane; i < n; i += 32) {
            /* a sum that is 0 belongs to no entry; one that is not, at a maximum of -inf, to entries that are NaN */
            const double a = __longlong_as_double((long long)told[i][0]), b = __longlong_as_double((long long)told[i][1]);
            const float at_a = __uint_as_float((unsigned)(told[i][3] >> 32)), at_b = __uint_as_float((unsigned)told[i][3]);
            if (a != 0.0) all.others_sum += a * (double)fast_exp2((at_a - all.others_top) * c);
            if (b != 0.0) all.sum += b * (double)fast_exp2((at_b - all.top) * c);
            all.cross += __longlong_as_double((long long)told[i][2]);
        }
        all.others_sum = warp_sum(all.others_sum), all.sum = warp_sum(all.sum);
        const float down = fast_exp2((all.others_top - all.top) * c); /* from one maximum to the other */
        if (all.others_sum != 0.0) all.sum += all.others_sum * (double)down;
        if (all.top == neg_inf() && all.sum == 0.0) { /* the student excludes every entry: the same in every block of the row */
            nothing();
            return;
        }
        top = all.top;
        inverse = (float)(1.0 / all.sum);
        double r = rest ? fmax(0.0, 1.0 - named_p) : 0.0;
        if (!(all.others_top > neg_inf())) r = 0.0;
        at_named = (float)(named_p + r);
        /* r over the student's share of the others, which may be too small for its own exponential */
        elsewhere = at_named;
        if (r > 0.0) {
            const double over = down > 0.0f ? all.sum / (all.others_sum * (double)down)
                                            : all.sum / all.others_sum * exp_64(((double)all.top - (double)all.others_top) * inv);
            elsewhere = (float)(named_p + r - r * over);
        }
        if (rank == 0 && warp == 0) {
            all.cross = warp_sum(all.cross);
            /* log of the teacher's sum: with teacher_lse the scores are relative to it, else to their maximum */
            const double shifted = all.cross; /* sum of p (score - z) / tau */
            const float loss = row_loss(RowSums{all.top, all.others_top, all.sum, all.others_sum, shifted - named_p * shift}, named_p,
                                        rest ? 1.0 : total, r, inv);
            if (lane == 0) {
                p.loss[row] = weight * loss;
                if (p.stats) {
                    float *s = p.stats + row * 4;
                    s[0] = top, s[1] = inverse, s[2] = at_named, s[3] = elsewhere;
                }
            }
        }
        if (!grad) return;
    }

    /* gradient: elsewhere * q everywhere, then the named entries once more with their own value */
    float g = (float)((double)weight * inv);
    if (BACKWARD && p.upstream) g *= p.upstream[row];
    const float factor = g * elsewhere * inverse;
    const Pair times(factor, factor), less(-top, -top), by(c, c);
#pragma unroll 2
    for (int v = share.first; v < share.last; v += 32) {
        float f[E];
        Elem<T>::unpack(share.get(v), f);
#pragma unroll
        for (int i = 0; i < E / 2; ++i)
            (times * fast_exp2((Pair(f[2 * i], f[2 * i + 1]) + less) * by)).get(f[2 * i], f[2 * i + 1]);
        put(share, grad, same, v, Elem<T>::pack(f));
    }
    __syncthreads();
    for (int j = threadIdx.x; j < p.k; j += kThreads) {
        const int at = named[j].at;
        if (at < 0) continue;
        double sum = named[j].p;
        if (twice) { /* the first entry of an index in the list writes the sum of all of them, in the list's order */
            bool earlier = false;
            sum = 0.0;
            for (int o = 0; o < p.k; ++o)
                if (named[o].at == at) {
                    if (o < j) earlier = true;
                    sum += named[o].p;
                }
            if (earlier) continue;
        }
        const float q = inverse * fast_exp2((named[j].z - top) * c);
        grad[at] = Elem<T>::down(g * (float)((double)at_named * q - sum));
    }
}

/* ----------------------------------------------------------------- host */
constexpr size_t kSharedMost = 192u << 10; /* dynamic shared memory a block may ask for (227 KB less what it declares) */
constexpr long long kShareBytes = 64 << 10; /* the share of a row a block aims to hold */

/* Blocks per row: as few as hold the row in shares of 64 KB (two or three blocks of an SM then overlap one another's
 * phases), more while rows are too few to give every SM a block, as long as a share stays worth a block. */
static int cluster_for(long long rows, long long row_bytes, int sm_count) {
    int size = 1;
    while (size < kMaxCluster && row_bytes > kShareBytes * size) size *= 2;
    while (size < kMaxCluster && rows * size < sm_count && row_bytes > (8 << 10) * size) size *= 2;
    return size;
}

}  // namespace accb_rows

using namespace accb_rt;
using namespace accb_rows;

#define LOCK(ctx)                                                   \
    if (!(ctx)) return fail(nullptr, ACCB_EINVAL, "null context"); \
    std::lock_guard<std::recursive_mutex> lock_((ctx)->mu);         \
    CtxGuard guard_(ctx)
#define TRY(expr)                     \
    do {                              \
        int st_ = (expr);             \
        if (st_ != ACCB_OK) return st_; \
    } while (0)

static size_t size_of(int type) { return type == ACCB_ROWS_F32 ? 4 : 2; }

static int check_rows(accb_context *ctx, const accb_rows_array *a, const char *what) {
    if (!a) return fail(ctx, ACCB_EINVAL, "%s: null array", what);
    if (a->type != ACCB_ROWS_F32 && a->type != ACCB_ROWS_F16 && a->type != ACCB_ROWS_BF16)
        return fail(ctx, ACCB_EINVAL, "%s: unknown element type %d", what, a->type);
    if (a->rows < 0 || a->rows > 0x7fffffffLL / kMaxCluster) return fail(ctx, ACCB_EINVAL, "%s: bad number of rows %lld", what, a->rows);
    if (a->cols < 1) return fail(ctx, ACCB_EBOUNDS, "%s: rows without entries", what);
    if (a->cols > kMaxCols) return fail(ctx, ACCB_EINVAL, "%s: rows of %d entries (at most %lld)", what, a->cols, kMaxCols);
    if (a->rows > 1 && a->pitch < a->cols) return fail(ctx, ACCB_EINVAL, "%s: rows of %d entries every %lld entries overlap", what, a->cols, a->pitch);
    if (a->rows > 0 && a->pitch > (1LL << 62) / (a->rows * 4)) return fail(ctx, ACCB_EINVAL, "%s: row pitch %lld too large", what, a->pitch);
    if (a->rows > 0 && !a->ptr) return fail(ctx, ACCB_EINVAL, "%s: null pointer", what);
    if (reinterpret_cast<uintptr_t>(a->ptr) % size_of(a->type)) return fail(ctx, ACCB_EINVAL, "%s: misaligned pointer", what);
    return ACCB_OK;
}

static RowsIn rows_in(const accb_rows_array *a) { return RowsIn{a->ptr, a->rows, a->pitch, a->cols}; }

/* shared memory of a block's share of a row */
static size_t share_bytes(const accb_rows_array *a, int size) {
    return 16 * (size_t)(a->type == ACCB_ROWS_F32 ? Share<float, true>::per_block(a->cols, size) : Share<__half, true>::per_block(a->cols, size));
}

/* one launch with `size` blocks per row; `fixed` bytes of dynamic shared memory besides the share */
template <class P>
static int launch_rows(accb_context *ctx, void (*resident)(const P), void (*streaming)(const P), const P &p, const accb_rows_array *a, int size,
                       size_t fixed, bool persistent, cudaStream_t stream, const char *name) {
    const size_t share = share_bytes(a, size);
    const bool fits = fixed + share <= kSharedMost;
    void (*kernel)(const P) = fits ? resident : streaming;
    const size_t smem = fixed + (fits ? share : 0);
    if (!std::count(ctx->rows_ready, ctx->rows_ready + ctx->rows_ready_count, (const void *)kernel)) {
        int st = check_cuda(ctx, cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSharedMost), name);
        if (st == ACCB_OK)
            st = check_cuda(ctx, cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100), name);
        if (st != ACCB_OK) return st;
        ctx->rows_ready[ctx->rows_ready_count++] = (const void *)kernel;
    }
    long long clusters = a->rows;
    cudaLaunchAttribute attr;
    memset(&attr, 0, sizeof attr);
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)size;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(clusters * size));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (persistent) { /* as many clusters as the GPU holds at a time, if there are more rows */
        int &most = ctx->rows_clusters[std::make_tuple((const void *)kernel, size, smem)];
        if (most == 0) {
            const int st = check_cuda(ctx, cudaOccupancyMaxActiveClusters(&most, (const void *)kernel, &cfg), name);
            if (st != ACCB_OK) return st;
            most = std::max(1, most);
        }
        clusters = std::min<long long>(clusters, most);
        cfg.gridDim = dim3((unsigned)(clusters * size));
    }
    if (ctx->trace_exec)
        fprintf(stderr, "[accb exec] %s<<<%lld,%d,%zu>>> rows=%lld cols=%d\n", name, clusters * size, kThreads, smem, a->rows, a->cols);
    void *args[] = {const_cast<P *>(&p)};
    const int st = check_cuda(ctx, cudaLaunchKernelExC(&cfg, (const void *)kernel, args), name);
    if (st == ACCB_OK) ctx->launches++;
    return st;
}

#define BY_TYPE(type, call)                                        \
    ((type) == ACCB_ROWS_F32   ? call(float)                       \
     : (type) == ACCB_ROWS_F16 ? call(__half)                      \
                               : call(__nv_bfloat16))

extern "C" {

int accb_top_rows(accb_context *ctx, accb_stream stream, const accb_rows_array *x, double temperature, int k, void *values, int32_t *index,
                  float *lse) {
    LOCK(ctx);
    TRY(check_rows(ctx, x, "top_rows"));
    if (k < 1 || k > kMaxK || k > x->cols) return fail(ctx, ACCB_EINVAL, "top_rows: %d entries of rows of %d (at most %d)", k, x->cols, kMaxK);
    if (!(temperature > 1e-30) || temperature > 1e30) return fail(ctx, ACCB_EINVAL, "top_rows: bad temperature %g", temperature);
    if (x->rows == 0) return ACCB_OK;
    if (!values || !index) return fail(ctx, ACCB_EINVAL, "top_rows: null result");
    int room = 256;
    while (room < 2 * k) room *= 2;
    const TopParams p{rows_in(x), values, index, lse, temperature, k, room};
    const int size = cluster_for(x->rows, (long long)x->cols * size_of(x->type), ctx->sm_count);
    const size_t fixed = room * sizeof(u64) + std::max(room / size * sizeof(u64), sizeof(Level));
#define CALL(T) launch_rows(ctx, top_rows<T, true>, top_rows<T, false>, p, x, size, fixed, true, (cudaStream_t)stream, "top_rows")
    return BY_TYPE(x->type, CALL);
#undef CALL
}

int accb_sample_rows(accb_context *ctx, accb_stream stream, const accb_rows_array *x, const uint32_t *allowed, long long allowed_pitch,
                     const float *uniform, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                     int32_t *token, float *logprob) {
    LOCK(ctx);
    TRY(check_rows(ctx, x, "sample_rows"));
    if (allowed && allowed_pitch < (x->cols + 31) / 32)
        return fail(ctx, ACCB_EINVAL, "sample_rows: %lld words of allowed bits for rows of %d entries", allowed_pitch, x->cols);
    if (x->rows == 0) return ACCB_OK;
    if (!uniform || !token) return fail(ctx, ACCB_EINVAL, "sample_rows: null random numbers or result");
    const SampleParams p{rows_in(x), allowed, allowed_pitch, uniform, temperature, top_p, min_p, top_k, token, logprob};
    const int size = cluster_for(x->rows, (long long)x->cols * size_of(x->type), ctx->sm_count);
#define CALL(T) launch_rows(ctx, sample_rows<T, true>, sample_rows<T, false>, p, x, size, 0, true, (cudaStream_t)stream, "sample_rows")
    return BY_TYPE(x->type, CALL);
#undef CALL
}

static int distill(accb_context *ctx, accb_stream stream, const accb_rows_array *student, const accb_rows_array *grad, DistillParams &p,
                   bool backward) {
    const char *what = backward ? "distill_rows_backward" : "distill_rows";
    TRY(check_rows(ctx, student, what));
    if (p.k < 1 || p.k > kMaxK) return fail(ctx, ACCB_EINVAL, "%s: %d entries of the teacher (1 to %d)", what, p.k, kMaxK);
    if (p.teacher_type != ACCB_ROWS_F32 && p.teacher_type != ACCB_ROWS_F16 && p.teacher_type != ACCB_ROWS_BF16)
        return fail(ctx, ACCB_EINVAL, "%s: unknown element type %d of the teacher", what, p.teacher_type);
    if (!(p.temperature > 1e-30) || p.temperature > 1e30) return fail(ctx, ACCB_EINVAL, "%s: bad temperature %g", what, p.temperature);
    if (grad) {
        TRY(check_rows(ctx, grad, what));
        if (grad->rows != student->rows || grad->cols != student->cols || grad->type != student->type)
            return fail(ctx, ACCB_EINVAL, "%s: the gradient has another shape or type than the scores", what);
        p.grad = grad->ptr;
        p.grad_pitch = grad->pitch;
    }
    if (student->rows == 0) return ACCB_OK;
    if (!p.teacher || !p.index) return fail(ctx, ACCB_EINVAL, "%s: null teacher", what);
    if (backward ? !p.stats || !grad : !p.loss) return fail(ctx, ACCB_EINVAL, "%s: null result or statistics", what);
    p.in = rows_in(student);
    const int size = cluster_for(student->rows, (long long)student->cols * size_of(student->type), ctx->sm_count);
    const long long share = (long long)share_bytes(student, size) / size_of(student->type); /* entries of a block's share, at most */
    p.map_words = (int)((share + 31) / 32 + 3) & ~3;
    const size_t fixed = (size_t)(p.map_words * 4 + p.k * sizeof(Named) + 15) / 16 * 16;
#define CALL(T)                                                                                                                       \
    (backward ? launch_rows(ctx, distill_rows<T, true, true>, distill_rows<T, false, true>, p, student, size, fixed, false, (cudaStream_t)stream, what) \
              : launch_rows(ctx, distill_rows<T, true, false>, distill_rows<T, false, false>, p, student, size, fixed, false, (cudaStream_t)stream, what))
    return BY_TYPE(student->type, CALL);
#undef CALL
}

int accb_distill_rows(accb_context *ctx, accb_stream stream, const accb_rows_array *student, const void *teacher, int teacher_type,
                      const int32_t *index, int k, const float *teacher_lse, const float *weight, double temperature, float *loss,
                      float *stats, const accb_rows_array *grad) {
    LOCK(ctx);
    DistillParams p;
    memset(&p, 0, sizeof p);
    p.teacher = teacher, p.index = index, p.teacher_lse = teacher_lse, p.weight = weight;
    p.loss = loss, p.stats = stats, p.temperature = temperature, p.k = k, p.teacher_type = teacher_type;
    return distill(ctx, stream, student, grad, p, false);
}

int accb_distill_rows_backward(accb_context *ctx, accb_stream stream, const accb_rows_array *student, const void *teacher,
                               int teacher_type, const int32_t *index, int k, const float *teacher_lse, const float *weight,
                               double temperature, const float *stats, const float *upstream, const accb_rows_array *grad) {
    LOCK(ctx);
    DistillParams p;
    memset(&p, 0, sizeof p);
    p.teacher = teacher, p.index = index, p.teacher_lse = teacher_lse, p.weight = weight, p.upstream = upstream;
    p.stats = const_cast<float *>(stats), p.temperature = temperature, p.k = k, p.teacher_type = teacher_type;
    return distill(ctx, stream, student, grad, p, true);
}

} /* extern "C" */
