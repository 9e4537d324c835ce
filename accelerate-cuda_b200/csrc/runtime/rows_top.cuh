/*
 * rows_top.cuh -- the best entries of every row and its log-sum-exp (accb_top_rows).
 */
#pragma once
#include "rows_search.cuh"

namespace accb_rows {

struct TopParams {
    RowsIn in;
    void *values;
    int *index;
    float *lse;
    double temperature;
    int k;
    int room; /* of the list of candidates, a power of two from 256 */
};

/* Places of a block's own candidates, or of a Level, which the same memory holds: an even number, since the share of the
 * row comes behind them and starts with a whole vector. */
static __host__ __device__ __forceinline__ int own_places(int room, int size) {
    const int part = room / size, level = (int)(sizeof(Level) / sizeof(u64));
    return ((part > level ? part : level) + 1) & ~1;
}

/* The k largest are found in one pass over the row's maximum, one over its exponentials (if asked for) and one over the
 * few entries above a bound: ceil(k / size) of every block's 256 threads hold a maximum at or above the bound, so at
 * least k entries do, and seldom many more.  They are listed in one block's memory, and sorted; the blocks of a cluster
 * take the rows' lists in turns and sort side by side.  Rows whose list overflows (ties, large entries side by side)
 * search for the border with counting bins and list again.  So do all rows of which a block is asked for more entries than
 * it has threads, since the threads' maxima then give no bound: the 64, 256, 257, 512 and 1024 best of 2000 x 32000 bf16
 * rows, which have one block each, take 78, 248, 369, 379 and 436 us.
 * Clusters stay for row after row: the next row is fetched as soon as the listing has read this one, under the sort.
 *
 * 64 of 2048 x 131072 bf16 with log-sum-exp: 243 us, 2.2 TB/s, a third of the copy rate; 512 of 24 x 50257 floats: 23 us.
 * A row takes its blocks 13 us, three an SM, most of it waiting for copies, barriers and instructions; the special function
 * unit is busy for a third of the time.  The search by bins in place of lists took 947 us, one row per cluster without
 * the turns 311. */
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
    u64 *list = reinterpret_cast<u64 *>(dynamic), *mine = list + p.room;
    Level &level = *reinterpret_cast<Level *>(mine);
    const T *x = static_cast<const T *>(p.in.x);
    const long long step = gridDim.x / size;
    if (size > 1) cluster_arrive(); /* every block of the cluster has started: waited for before the first message */

    Row<T, R> share;
    share.init(x + (blockIdx.x / size) * p.in.pitch, p.in.cols, rank, size, dynamic + (p.room + own_places(p.room, (int)size)) / 2);
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
                const Pair less(-most, -most), by(c, c);
                Pair part[2] = {Pair(0.0f, 0.0f), Pair(0.0f, 0.0f)};
                if (most < __uint_as_float(0x7f800000u)) {
#pragma unroll 2
                    for (int v = share.first; v < share.last; v += 32) {
                        float f[E];
                        Elem<T>::unpack(share.raw(v), f);
#pragma unroll
                        for (int i = 0; i < E / 2; ++i) {
                            float y[2];
                            ((Pair(f[2 * i], f[2 * i + 1]) + less) * by).get(y[0], y[1]);
                            part[i & 1] = part[i & 1] + fast_exp2(Pair(fmaxf(y[0], -200.0f), fmaxf(y[1], -200.0f))); /* NaN: 0 */
                        }
                    }
                }
                float part_a, part_b;
                (part[0] + part[1]).get(part_a, part_b);
                const float warp_part = warp_sum(part_a + part_b);
                __syncthreads();
                if (lane == 0) scratch[warp] = __float_as_uint(warp_part);
            }
            n = gather(share, thread_most, fmaxf(bound, -3.402823466e+38f), mine, list, (unsigned)p.room, own, rank, size, finisher);
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
            const Weigh none(0.0f, 1.0, nullptr);
            const Border border = find_border<T, R, false>(share, level, size, key_of(bound), key_of(most), (u64)p.k, none, 0.0, 0);
            unsigned ties = 0;
            for (int v = share.first; v < share.last; v += 32) {
                float f[E];
                share.floats(v, f);
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
                if (v < share.last) share.floats(v, f);
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

}  // namespace accb_rows
