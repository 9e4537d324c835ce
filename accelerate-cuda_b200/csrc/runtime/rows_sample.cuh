/*
 * rows_sample.cuh -- one index drawn from every row (accb_sample_rows): temperature, top_k, top_p and min_p, from a
 * given random number.
 */
#pragma once
#include "rows_search.cuh"

namespace accb_rows {

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

__device__ __forceinline__ void put_token(const SampleParams &p, long long row, int index, float value, const Weigh &weigh, double temperature, u64 total) {
    p.token[row] = index;
    if (p.logprob) {
        const double below = value == weigh.top ? 0.0 : ((double)value - (double)weigh.top) / temperature;
        /* the total as a multiple of the maximum's weight as it was added up, which is among what is kept: 0 for the only
         * entry, and never above */
        p.logprob[row] = (float)(below - log_64((double)total / (double)weigh.of(weigh.top)));
    }
}

/* Draws from the candidates in `list`, which hold every entry that top_k and top_p could keep; by one block. */
static __device__ __noinline__ void draw_from_list(const SampleParams &p, const PendingDraw &d, u64 *list, u64 *scratch, unsigned size, const double *table) {
    const Weigh weigh(d.most, d.temperature, table);
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
    const u64 limit = top_p < 1.0f ? (u64)ceil((double)top_p * (double)total) : ~0ull;
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
                put_token(p, d.row, index_of(list[i] >> 32), x, weigh, d.temperature, total);
                return;
            }
        }
    }
}

/* What top_k and top_p need of shared memory besides. */
struct CutSpace {
    union {
        u64 mine[kSampleRoom];
        FineBins bins;
        Level level;
    };
    u64 list[kSampleRoom];
    PendingDraw pending;
    Extent extent;
    alignas(16) u64 parts[kMaxCluster * kWarps][2]; /* weight above the border and entries on it, by part of the share */
};
struct NoCutSpace {
    Extent extent;
};

/* A token is the first kept entry, in index order, at which the running sum of exact weights exceeds uniform * total.
 *   no cuts, min_p   one pass for the maximum, one for the weights -- by warp and, within a warp's piece, by quarter, so
 *                    that the warp in which the sum is met walks a quarter of its piece
 *   top_k, or top_p with few candidates   a bound as in top_rows, or from the row's weight: what lies more than
 *                    log(cols / (1 - top_p)) below the maximum weighs less than what is cut off.  One block lists, sorts
 *                    and draws, the blocks of a cluster by turns
 *   others           the border by counting bins (border_by_bins), then as without cuts above it; where the bins also say
 *                    what every block holds (bfloat16), only the share with the token is looked through, by all blocks
 * Clusters stay for row after row, as in top_rows.
 *
 * 1024 x 131072 bf16: without cuts 238 us (1.1 TB/s, 17 % of the copy rate), issue slots 57 % and the 64-bit
 * pipe 32 % busy: eight operations a weight; the best entry 70 us (58 %), top_k 50 146 us, top_k 400 416 us, top_p 0.9 533 us, min_p 0.05 138 us.
 * Weights in 32 bits with a bound on their error, and again in 64 where the bound could not tell two indices apart, took
 * 343 us: with a hundred thousand like entries it seldom can.
 *
 * CUTS: the caller gives top_k or top_p.  Two kernels, because a block waits for every instruction that is not in the
 * SM's cache: what a launch cannot need is not in its way.  The first gets the registers of two blocks an SM for
 * 16-bit scores (top_k 50 of 1024 x 131072 bf16: 146 us, with those of three 176) and of three for 32-bit ones (top_p of
 * 48 x 50257: 78 us, with those of two 108). */
template <class T, bool R, bool CUTS> __global__ void __launch_bounds__(kThreads, CUTS && sizeof(T) == 2 ? 2 : 3) sample_rows(const __grid_constant__ SampleParams p) {
    constexpr int E = Elem<T>::E;
    constexpr float kLowest = -3.402823466e+38f;
    extern __shared__ uint4 stage[];
    __shared__ Told told_by_turns[2];
    __shared__ std::conditional_t<CUTS, CutSpace, NoCutSpace> sh;
    __shared__ double table[kTable * kTableCopies];
    __shared__ u64 scratch[kWarps], warp_part[kWarps][2];
    __shared__ unsigned own;
    const unsigned size = cluster_size(), rank = cluster_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T *x = static_cast<const T *>(p.in.x);
    const long long step = gridDim.x / size;
    if (size > 1) cluster_arrive(); /* every block of the cluster has started: waited for before the first message */

    Row<T, R> share;
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
            if constexpr (CUTS) {
                if (!waiting) return;
                draw_from_list(p, sh.pending, sh.list, scratch, size, table);
                waiting = false;
                __syncthreads(); /* the list is used again */
            }
        };
        auto next = [&] { /* the scores of the next row take the place of this one's, which this thread has read */
            if (!more) return;
            share.init(x + (row + step) * p.in.pitch, p.in.cols, rank, size, stage);
            share.fetch();
        };
        share.bits = p.allowed ? p.allowed + row * p.allowed_pitch : nullptr;
        share.infinite = false;
        const float warmth = p.temperature ? p.temperature[row] : 1.0f;
        int k = CUTS && p.top_k ? p.top_k[row] : 0;
        float top_p = CUTS && p.top_p ? p.top_p[row] : 1.0f;
        if (top_p < 0.0f) top_p = 0.0f; /* the first entry, as 0; a NaN stays, and is off */
        const float min_p = p.min_p ? p.min_p[row] : 0.0f;
        const float uniform = p.uniform[row];
        if (!(warmth > 0.0f)) k = 1;
        const double temperature = warmth > 0.0f ? fminf(warmth, 1e30f) : 1.0f;
        if (k >= p.in.cols || k < 0) k = 0;
        if (threadIdx.x == 0) own = 0;
        share.wait();
        if (share.bits) share.apply();

        /* the maximum, and where at least k entries lie above: a k-th part of the blocks' threads in each block */
        typename Elem<T>::Max largest;
#pragma unroll 4
        for (int v = share.first; v < share.last; v += 32) largest.add(share.raw(v));
        float thread_most = largest.get();
        const float2 ext = extent_of(thread_most, CUTS && k > 1 ? (k + (int)size - 1) / (int)size : 0, sh.extent);
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
            share.infinite = true;
            share.apply();
            most = 0.0f, bound = neg_inf(), thread_most = thread_most == __uint_as_float(0x7f800000u) ? 0.0f : neg_inf();
        }

        if (!CUTS && k == 1) { /* the best entry: the threads that hold it look for it */
            unsigned at = 0xffffffffu;
            if (thread_most == most)
                for (int v = share.first; v < share.last; v += 32) {
                    float f[E];
                    share.floats(v, f);
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        if (f[i] == most) at = min(at, (unsigned)(share.entry(v) + i));
                }
            at = __reduce_min_sync(~0u, at);
            if (lane == 0) scratch[warp] = at;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; ++w) at = min(at, (unsigned)scratch[w]);
            tell_all(told.block[1], at, 0, rank, size);
            for (int i = 0; i < (int)size; ++i) at = min(at, (unsigned)told.block[1][i][0]);
            if (rank == 0 && threadIdx.x == 0) {
                p.token[row] = (int)at;
                if (p.logprob) p.logprob[row] = 0.0f;
            }
            next();
            continue;
        }

        /* the lowest score that min_p keeps */
        float lowest = kLowest;
        if (min_p > 0.0f) {
            const double low = (double)most + log_64(fmin((double)min_p, 1.0)) * temperature;
            if (low > -3.0e38) lowest = __double2float_ru(low);
        }
        const Weigh weigh(most, temperature, table);
        if (k == 1) bound = most;

        /* weight above a border and number of entries on it, of this thread: the weight in quarters of the warp's
         * piece, which are kept to find the token's */
        u64 quarter[4];
        unsigned ties = 0;
        const int start = share.first - lane; /* of the warp's piece */
        const int per_quarter = (max(0, share.last - start) + 127) >> 7;
        auto pass = [&](const Border &border, bool most_count) {
            const float on = value_of(border.key);
            const bool count = border.ties != 0;
            const float from = fmaxf(weigh.least, value_of(max(border.key, key_of(kLowest) - 1u) + 1u));
            ties = 0;
            int v0 = start;
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
                double sum = 0.0;
                const int end = min(share.last, start + 32 * per_quarter * (q + 1));
#pragma unroll 1
                for (; v0 < end; v0 += 32) { /* the same turns in all lanes */
                    uint4 w = make_uint4(Elem<T>::kLowest, Elem<T>::kLowest, Elem<T>::kLowest, Elem<T>::kLowest);
                    if (v0 + lane < end) w = share.raw(v0 + lane);
                    typename Elem<T>::Max best;
                    best.add(w);
                    if (!__any_sync(~0u, count ? best.get() >= on : best.get() >= from)) continue;
                    float f[E];
                    Elem<T>::unpack(w, f);
                    if (count) {
#pragma unroll
                        for (int i = 0; i < E; ++i) ties += f[i] == on;
                    }
                    sum += weigh.some<E>(f, from, most_count);
                }
                quarter[0] = quarter[1], quarter[1] = quarter[2], quarter[2] = quarter[3], quarter[3] = (u64)sum;
            }
        };
        u64 total = 0;
        const bool cut = k > 0 || top_p < 1.0f;
        BlockPart part{0, 0, false};
        bool passed = false;
        Border border{key_of(cut ? kLowest : lowest) - 1u, 0, 0}; /* without cuts: of min_p */
        if constexpr (CUTS) {
            if (cut) {
                float least = fmaxf(bound, kLowest);
                bool listed = k > 0 && k <= kListed;
                if (k == 0) { /* top_p alone */
                    least = weigh.least;
                    /* counts by bin say what a row of bfloat16 weighs; else, or where min_p leaves few to list, a pass
                     * does, and how far down entries lie that all of them together weigh less than what is cut off: below
                     * the maximum, since that is at most all of the weight, and the weight at most `cols` times the maximum's */
                    if (Elem<T>::kShift != 16 || min_p > 0.0f) {
                        pass(border, true);
                        const u64 block_total = block_sum((quarter[0] + quarter[1]) + (quarter[2] + quarter[3]), scratch);
                        tell_all(told.block[1], block_total, 0, rank, size);
                        for (int i = 0; i < (int)size; ++i) total += told.block[1][i][0];
                        const double left = (1.0 - (double)top_p) * ((double)total * (1.0 / (double)(1ull << kUnitLog2)));
                        const double low = (double)most + (log_64(left / (double)p.in.cols) - weigh.log_of_top() - 0.01) * temperature;
                        if (left > 1e-5 && low > (double)least) least = __double2float_rd(low);
                        listed = true;
                    }
                }
                /* what min_p drops is not needed to weigh the rest, unless top_p takes its share of what top_k keeps */
                const float from = k == 0 || !(top_p < 1.0f) ? fmaxf(least, lowest) : least;
                if (listed) {
                    const unsigned n = gather(share, thread_most, from, sh.mine, sh.list, kSampleRoom, own, rank, size, finisher);
                    tell_all(told.block[2], n, 0, rank, size);
                    unsigned longest = 0;
                    for (int i = 0; i < (int)size; ++i) longest = max(longest, (unsigned)told.block[2][i][0]);
                    if (longest <= kSampleRoom / size) { /* the same in every block of the row */
                        next();
                        if (rank == finisher) {
                            waiting = true;
                            if (threadIdx.x < size) sh.pending.n[threadIdx.x] = (unsigned)told.block[2][threadIdx.x][0];
                            if (threadIdx.x == 0) {
                                PendingDraw &d = sh.pending;
                                d.row = row, d.total = total, d.temperature = temperature, d.most = most;
                                d.lowest = lowest, d.top_p = top_p, d.uniform = uniform, d.k = k;
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
                                : border_by_bins<T, R>(share, sh.bins, sh.level, size, weigh, k > 0 || Elem<T>::kShift != 16 ? least : weigh.least, most,
                                                       (u64)k, top_p < 1.0f ? (double)top_p : 1.0, total, part);
                const unsigned below = key_of(lowest) - 1u;
                if (below >= border.key) border = Border{below, 0, 0}, part.known = false;
            }
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
        const bool here_in_block = before <= target && target < before + here;
        int v0 = start;
        const bool shared_search = CUTS && R && part.known && size > 1;
        if constexpr (CUTS && R) {
            if (shared_search) {
                /* Bins do not say where the weight lies.  The blocks of the cluster look for it side by side in the share of
                 * the block that holds the token, each in one part of every warp's piece. */
                unsigned holder = 0;
                u64 upto = 0;
                ties_seen = 0;
                for (unsigned i = 0; i < size; ++i) {
                    const unsigned n = (unsigned)told.block[3][i][1], kept = min(ties_seen + n, border.ties) - min(ties_seen, border.ties);
                    upto += told.block[3][i][0] + kept * tie_weight, ties_seen += n;
                    holder += upto <= target;
                }
                const int per = share.per_block(p.in.cols, (int)size), piece = ((per + kWarps - 1) / kWarps + 31) & ~31;
                const int turns = (piece / 32 + (int)size - 1) / (int)size; /* of 32 vectors, a part */
                const int from0 = warp * piece, end = min(min(per, share.vectors() - (int)holder * per), from0 + piece);
                const unsigned staged = peer_addr(shared_addr(stage), holder);
                const float on = value_of(border.key), from = fmaxf(weigh.least, value_of(max(border.key, key_of(kLowest) - 1u) + 1u));
                double sum = 0.0;
                ties = 0;
#pragma unroll 1
                for (int i = from0 + 32 * turns * (int)rank; i < min(end, from0 + 32 * turns * ((int)rank + 1)); i += 32) {
                    uint4 w = make_uint4(Elem<T>::kLowest, Elem<T>::kLowest, Elem<T>::kLowest, Elem<T>::kLowest);
                    if (i + lane < end) w = peer_load(staged + 16 * (i + lane));
                    float f[E];
                    Elem<T>::unpack(w, f);
#pragma unroll
                    for (int e = 0; e < E; ++e) ties += f[e] == on;
                    sum += weigh.some<E>(f, from, false);
                }
                const u64 mass = warp_sum((u64)sum);
                ties = warp_sum(ties);
                if (lane == 0) peer_store(peer_addr(shared_addr(&sh.parts[warp * size + rank][0]), holder), mass, ties);
                cluster_sync(size);
                if (here_in_block) {
                    /* the part: two a lane */
                    const int n = kWarps * (int)size, i0 = 2 * lane;
                    u64 m[2];
                    unsigned q[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) m[i] = i0 + i < n ? sh.parts[i0 + i][0] : 0, q[i] = i0 + i < n ? (unsigned)sh.parts[i0 + i][1] : 0;
                    const unsigned seen = warp_scan(q[0] + q[1]) - q[1] - q[0], block_quota = quota;
                    const unsigned k0 = min(seen, block_quota), k1 = min(seen + q[0], block_quota), k2 = min(seen + q[0] + q[1], block_quota);
                    const u64 w0 = m[0] + (k1 - k0) * tie_weight, w1 = m[1] + (k2 - k1) * tie_weight;
                    const u64 after = before + warp_scan(w0 + w1), first = after - w1 - w0;
                    const unsigned found = __ballot_sync(~0u, target < after);
                    const int l = __ffs(found) - 1; /* one of them: the block holds the token */
                    const bool second = target >= first + w0;
                    const int at = __shfl_sync(~0u, i0 + (int)second, l);
                    before = __shfl_sync(~0u, second ? first + w0 : first, l);
                    here = __shfl_sync(~0u, second ? w1 : w0, l);
                    quota = __shfl_sync(~0u, second ? k2 - k1 : k1 - k0, l);
                    if (at / (int)size != warp) here = 0;
                    v0 = start + 32 * turns * (at % (int)size);
                }
            }
        }
        if (!here_in_block) { /* in another block */
            next();
            continue;
        }
        if (!shared_search) {
            if (!passed) pass(border, false);
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

        if (!shared_search && quota == 0) { /* which quarter of the warp's piece */
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const u64 w = warp_sum(quarter[q]);
                if (v0 == start + 32 * per_quarter * q && before + w <= target) before += w, v0 += 32 * per_quarter;
            }
        }
        unsigned left = quota;
        u64 sum = before;
#pragma unroll 1
        for (; v0 < share.last; v0 += 32) {
            const int v = v0 + lane;
            float f[E];
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = neg_inf();
            if (v < share.last) share.floats(v, f);
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
                    put_token(p, row, at, value, weigh, temperature, total);
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

}  // namespace accb_rows
