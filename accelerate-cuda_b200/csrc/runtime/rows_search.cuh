/*
 * rows_search.cuh -- the best entries of a row that a cluster holds (rows.cuh): candidate lists and their sorting, a
 * bound that enough entries reach, and the border of what a count or a share of the weight keeps.
 */
#pragma once
#include "rows.cuh"

namespace accb_rows {

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

/* ------------------------------------------------------ candidate lists */
/* An entry as one number: larger for larger scores and, among equal ones, for lower indices.  0 is no entry. */
__device__ __forceinline__ u64 entry_of(float f, int index) { return (u64)key_of(f) << 32 | (0xffffffffu - (unsigned)index); }
__device__ __forceinline__ float score_of(u64 e) { return value_of((unsigned)(e >> 32)); }
__device__ __forceinline__ int index_of(u64 e) { return (int)(0xffffffffu - (unsigned)e); }

/* Lists the entries of the row that are not below `least` (finite) in `list` of the block `to` of the cluster, which
 * finishes the row: a part of `room / size` places for every block.  `most` is the largest of this thread's scores:
 * where few threads have any such entry, a warp looks through their vectors together, a lane each.  `own`, zero
 * before, counts this block's; a block lists its own first, since a place in its own shared memory costs a fraction of
 * one in another block's.  The counts still have to be told; returns this block's. */
template <class T, bool R>
__device__ unsigned gather(const Row<T, R> &share, float most, float least, u64 *mine, u64 *list, unsigned room, unsigned &own,
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
            const uint4 w = share.raw(v);
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

/* Sorts a list in shared memory, largest first; `room`, a power of two, numbers fit.  Up to 256 different numbers are
 * ranked by counting, one thread each, which takes two barriers; more by bitonic merging. */
static __device__ __noinline__ void sort_down(u64 *list, int n, int room) {
    if (n <= kThreads) {
        const int t = threadIdx.x;
        const u64 e = t < n ? list[t] : 0;
        int above = 0;
        if ((t & ~31) < n) {
#pragma unroll 8
            for (int j = 0; j < n; ++j) above += list[j] > e;
        }
        __syncthreads();
        if (t < n) list[above] = e;
        __syncthreads();
        return;
    }
    int m = 2 * kThreads;
    while (m < n) m *= 2;
    m = min(m, room);
    for (int i = n + threadIdx.x; i < m; i += kThreads) list[i] = 0;
    for (int len = 2; len <= m; len *= 2)
        for (int d = len / 2; d; d /= 2) {
            __syncthreads();
            for (int i = threadIdx.x; i < m / 2; i += kThreads) {
                const int a = ((i & ~(d - 1)) << 1) | (i & (d - 1)), b = a + d;
                const u64 u = list[a], w = list[b];
                if ((u < w) == ((a & len) == 0)) list[a] = w, list[b] = u;
            }
        }
    __syncthreads();
}

/* The largest of the block's scores, and one that at least `want` of its threads reach with the largest of theirs: the
 * want-th largest of these, or of the largest of four neighbours each where that leaves enough, rounded down to a
 * bfloat16 (-inf where want is 0 or more than there are threads).  A thread counts how many are above its own, two at a
 * time. */
struct Extent {
    alignas(16) __nv_bfloat16 thread[kThreads];
    float warp[kWarps][2];
};
static __device__ __noinline__ float2 extent_of(float most, int want, Extent &x) {
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    float bound = neg_inf();
    if (want > 0 && want <= kThreads) {
        const bool fours = want <= kThreads / 8;
        float group = most;
        if (fours) {
            group = fmaxf(group, __shfl_xor_sync(~0u, group, 1));
            group = fmaxf(group, __shfl_xor_sync(~0u, group, 2));
        }
        const __nv_bfloat16 own = __float2bfloat16_rd(group);
        const __nv_bfloat162 pair = __halves2bfloat162(own, own);
        if (!fours || (lane & 3) == 0) x.thread[fours ? t >> 2 : t] = own;
        __syncthreads();
        __nv_bfloat162 above[2] = {__floats2bfloat162_rn(0.0f, 0.0f), __floats2bfloat162_rn(0.0f, 0.0f)}; /* exact up to 256 */
        const int vectors = (fours ? kThreads / 4 : kThreads) / 8;
#pragma unroll 4
        for (int i = 0; i < vectors; ++i) {
            const uint4 w = reinterpret_cast<const uint4 *>(x.thread)[i];
            const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) above[j & 1] = __hadd2(above[j & 1], __hgt2(*reinterpret_cast<const __nv_bfloat162 *>(&u[j]), pair));
        }
        const float2 a = __bfloat1622float2(above[0]), b = __bfloat1622float2(above[1]);
        bound = a.x + a.y + b.x + b.y < (float)want ? __bfloat162float(own) : __uint_as_float(0x7f800000u);
        bound = warp_min(bound);
    }
    most = warp_max(most);
    if (lane == 0) x.warp[warp][0] = most, x.warp[warp][1] = bound;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) most = fmaxf(most, x.warp[w][0]), bound = fminf(bound, x.warp[w][1]);
    return make_float2(most, bound);
}

/* ---------------------------------------------------------------- borders */
/* The best entries of a row, in the order of falling value and, among equals, rising index: every entry whose key is
 * above `key`, and the first `ties` of those whose key it is. */
struct Border {
    unsigned key;
    unsigned ties;
    unsigned equals; /* entries with that key */
};

struct Level { /* one level of the border search */
    alignas(16) u64 mass[kBins];
    alignas(16) unsigned count[kBins];
    u64 warp_total[kWarps];
    u64 before;
    unsigned bin, bin_count;
    int found;
};

/* Finds the border of the shortest run of best entries, among those with klo <= key <= khi (khi >= every key of the
 * row, or what is above them is left out), that holds `target` entries (BY_MASS false) or, BY_MASS, the weight
 * `target`, or where that is 0 the given fraction of what the range holds less the weight of `spare` entries of key klo.
 *
 * Every level lays 256 bins over the range of keys, counts (and weighs) the entries of each, finds the bin in which
 * the border lies and goes on with that bin's range; when a bin is one key, the rest is arithmetic.  Bins are summed
 * over the cluster by reading the other blocks' bins, one per thread; every block does that for itself and so learns
 * the result without another message.
 * The way for rows whose candidates are too many for a list.  All threads of the cluster call it with the same
 * arguments. */
template <class T, bool RESIDENT, bool BY_MASS>
__device__ __noinline__ Border find_border(const Row<T, RESIDENT> share, Level &lv, unsigned size, unsigned klo, unsigned khi,
                              u64 target, const Weigh weigh, double fraction, unsigned spare) {
    constexpr int E = Elem<T>::E, S0 = Elem<T>::kShift;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const unsigned bottom = klo;
    bool have_target = target != 0;
    for (;;) {
        const unsigned span = khi - klo;
        const int shift = max(S0, 24 - __clz(span)); /* span >> shift < 256 */
        const bool by_entry = BY_MASS && shift > S0;
        lv.count[t] = 0, lv.mass[t] = 0;
        if (t == 0) lv.found = 0;
        __syncthreads();
        for (int v = share.first; v < share.last; v += 32) {
            float f[E];
            share.floats(v, f);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const unsigned k = key_of(f[i]);
                if (k - klo <= span) {
                    const unsigned b = (khi - k) >> shift;
                    atomicAdd(&lv.count[b], 1u);
                    if (by_entry) atomicAdd(&lv.mass[b], weigh.weight(f[i]));
                }
            }
        }
        cluster_sync(size);
        unsigned count = 0;
        u64 sum = 0;
        for (unsigned r = 0; r < size; ++r) {
            count += peer_load32(peer_addr(shared_addr(&lv.count[t]), r));
            if (by_entry) sum += peer_load1(peer_addr(shared_addr(&lv.mass[t]), r));
        }
        /* the one key of a bin once a bin is one key: keys of 16-bit types end in zeros above zero and in ones below */
        auto key_at = [&](unsigned bin) {
            const unsigned hi = khi - (bin << shift), low = (1u << S0) - 1u;
            return (hi & 0x80000000u) ? (hi & ~low) : ((hi + 1u) & ~low) - 1u;
        };
        if (BY_MASS && !by_entry && count) sum = count * weigh.weight(value_of(key_at(t)));
        if (!BY_MASS) sum = count;
        u64 upto = warp_scan(sum);
        if (lane == 31) lv.warp_total[warp] = upto;
        __syncthreads();
        u64 all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) upto += lv.warp_total[w];
            all += lv.warp_total[w];
        }
        if (!have_target) { /* the weight of the range is the total that the fraction is of */
            all -= spare * weigh.weight(value_of(bottom));
            target = max(1ull, (u64)ceil(fraction * (double)all));
            have_target = true;
        }
        if (upto - sum < target && target <= upto) {
            lv.bin = t;
            lv.bin_count = count;
            lv.before = upto - sum;
            lv.found = 1;
        }
        cluster_sync(size); /* the result is there, and no block reads the bins any more */
        if (!lv.found) return Border{klo, 0xffffffffu, 0xffffffffu}; /* less than was asked for: all of the range */
        const unsigned bin = lv.bin, bin_count = lv.bin_count;
        target -= lv.before;
        __syncthreads(); /* lv is used again */
        if (shift == S0) {
            const unsigned key = key_at(bin);
            u64 ties = target;
            if (BY_MASS) {
                const u64 w = weigh.weight(value_of(key));
                ties = (target + w - 1) / w; /* w > 0: the bin held some of the weight that was looked for */
            }
            return Border{key, (unsigned)min(ties, (u64)bin_count), bin_count};
        }
        khi -= bin << shift;
        const unsigned width = (1u << shift) - 1u;
        if (khi - klo > width) klo = khi - width;
    }
}

/* ------------------------------------------------------------------- bins */
/* For rows with too many candidates for a list: one pass counts entries by the 16 leading bits of their keys -- sign,
 * exponent and seven bits of mantissa, which is all there is of a bfloat16.  Keys near zero, 2^-10 of the largest
 * magnitude and below, would be most of the keys and hold next to no entries: they share the middle bin.  Keys below
 * minus the largest magnitude share the last.  The weights of these two are added up entry by entry. */
constexpr int kFineBins = 12 * kThreads; /* 11 octaves of 128 keys on either side of zero, the two shared bins: 2818 */
constexpr int kNear = 512;
struct FineBins {
    alignas(16) unsigned count[kFineBins]; /* of this block */
    float near[kNear];                     /* scores of its shared bins, if they are so few */
    unsigned n_near;
    u64 warp[kWarps];
    alignas(16) u64 shared[kMaxCluster][2]; /* weights of the middle bin and the last, by block */
    u64 total[2][kMaxCluster];    /* of the blocks' slices; by search */
    alignas(16) u64 found[2][2];  /* what precedes the bin that was looked for; its count << 32 | bin, or ~0 */
};

/* The order of bins: 0 for the largest scores. */
struct BinOrder {
    unsigned high, low, far, gap, top; /* leading bits of the smallest key above the middle bin, the largest below, the
                                          largest of the last bin; keys left out; squeezed key of the maximum */
    float zero, end;                   /* scores between -zero and zero are in the middle, -end and below in the last */
    int middle, last;                  /* the shared bins; middle may lie beyond the maximum, below 0 */
    __device__ __forceinline__ BinOrder(float most, float from) {
        const float reach = fmaxf(fabsf(most), fminf(fabsf(from), fmaxf(2.0f * fabsf(most), 64.0f)));
        const int e = (int)(__float_as_uint(reach) >> 23); /* biased exponent of the largest magnitude */
        const float z = __uint_as_float((unsigned)max(1, e - 10) << 23), m = __uint_as_float((unsigned)min(254, e + 1) << 23);
        high = key_of(z) >> 16, low = key_of(-z) >> 16, far = key_of(-m) >> 16, gap = high - low - 2;
        top = squeeze(key_of(most) >> 16);
        zero = z, end = m;
        middle = (int)(top - (low + 1)), last = (int)(top - far);
    }
    __device__ __forceinline__ int of(float f) const { return (int)bin((__float_as_uint(f) >> 16) ^ ((unsigned)((int)__float_as_uint(f) >> 31) >> 16 | 0x8000u)); }
    __device__ __forceinline__ bool shared(float f) const { return fabsf(f) < zero || f <= -end; }
    __device__ __forceinline__ unsigned squeeze(unsigned k) const { return k >= high ? k - gap : k > low ? low + 1 : max(k, far); }
    __device__ __forceinline__ unsigned bin(unsigned k) const { return top - squeeze(k); }
    /* the bin's keys, leading bits */
    __device__ __forceinline__ unsigned lowest(unsigned bin) const {
        const unsigned c = top - bin;
        return c > low + 1 ? c + gap : c == far ? 0 : c;
    }
    __device__ __forceinline__ unsigned highest(unsigned bin) const {
        const unsigned c = top - bin;
        return c > low + 1 ? c + gap : c == low + 1 ? high - 1 : c;
    }
};

/* Counts this block's entries that are not below `from`; returns its weights of the two shared bins.  All threads of the
 * block call it; barriers follow its writes. */
template <class T, bool RESIDENT>
__device__ __forceinline__ void count_bins(const Row<T, RESIDENT> &share, FineBins &bins, const BinOrder &order, const Weigh &weigh, float from,
                           u64 (&coarse)[2]) {
    constexpr int E = Elem<T>::E;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
#pragma unroll
    for (int i = 0; i < kFineBins / kThreads / 4; ++i) *reinterpret_cast<uint4 *>(&bins.count[4 * (t + i * kThreads)]) = make_uint4(0, 0, 0, 0);
    if (t < 2) bins.found[t][1] = ~0ull;
    if (t == 0) bins.n_near = 0;
    const unsigned counts = shared_addr(bins.count);
    __syncthreads();
    for (int v = share.first; v < share.last; v += 32) {
        const uint4 w = share.raw(v);
        typename Elem<T>::Max best;
        best.add(w);
        if (!(best.get() >= from)) continue;
        float f[E];
        Elem<T>::unpack(w, f);
        unsigned near = 0, at[E], in[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            in[i] = f[i] >= from;
            at[i] = counts + 4 * (unsigned)order.of(f[i]);
            near |= (unsigned)(in[i] && order.shared(f[i])) << i;
        }
#pragma unroll
        for (int i = 0; i < E; ++i) /* no branch, which would wait for every address by itself */
            asm volatile(
                "{\n"
                ".reg .pred p;\n"
                "setp.ne.u32 p, %1, 0;\n"
                "@p red.shared::cta.add.u32 [%0], 1;\n"
                "}\n" ::"r"(at[i]),
                "r"(in[i])
                : "memory");
        if (near) {
            unsigned place = atomicAdd(&bins.n_near, __popc(near));
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (((near >> i) & 1u) && place < kNear) bins.near[place++] = f[i];
        }
    }
    __syncthreads();
    coarse[0] = coarse[1] = 0;
    const int n = (int)bins.n_near;
    if (n == 0) return; /* the same in all threads */
    if (n <= kNear) {
        for (int i = t; i < n; i += kThreads) coarse[bins.near[i] <= -order.end] += weigh.weight(bins.near[i]);
    } else {
        for (int v = share.first; v < share.last; v += 32) {
            float f[E];
            Elem<T>::unpack(share.raw(v), f);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const u64 w = f[i] >= from && order.shared(f[i]) ? weigh.weight(f[i]) : 0;
                coarse[0] += f[i] <= -order.end ? 0 : w, coarse[1] += f[i] <= -order.end ? w : 0;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const u64 w = warp_sum(coarse[i]);
        if (lane == 0) bins.warp[warp] = w;
        __syncthreads();
        coarse[i] = 0;
#pragma unroll
        for (int j = 0; j < kWarps; ++j) coarse[i] += bins.warp[j];
        __syncthreads();
    }
}

/* the weight of n entries of a bin that is not shared: of its highest or its lowest score, which are one for a bfloat16
 * (whose key ends in zeros above zero and in ones below) */
template <bool EXACT> __device__ __forceinline__ unsigned key_of_bin(const BinOrder &order, int bin, bool high) {
    return high || (EXACT && order.highest(bin) < 0x8000u) ? order.highest(bin) << 16 | 0xffffu : order.lowest(bin) << 16;
}

/* The weight of this block's counted entries in the bins before `end`, by all threads; two barriers. */
static __device__ u64 weight_before(FineBins &bins, const BinOrder &order, const Weigh &weigh, const u64 (&coarse)[2], int end) {
    u64 mine = 0;
#pragma unroll 1
    for (int bin = threadIdx.x; bin < min(end, kFineBins); bin += kThreads) {
        const unsigned n = bins.count[bin];
        if (n && bin != order.middle && bin != order.last) mine += n * weigh.weight(value_of(key_of_bin<true>(order, bin, false)));
    }
    if (threadIdx.x == 0) mine += (order.middle < end ? coarse[0] : 0) + (order.last < end ? coarse[1] : 0);
    mine = warp_sum(mine);
    if ((threadIdx.x & 31) == 0) bins.warp[threadIdx.x >> 5] = mine;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all += bins.warp[w];
    __syncthreads();
    return all;
}

/* What a block holds of the entries that are kept, where the bins say so. */
struct BlockPart {
    u64 mass;      /* above the border */
    unsigned ties; /* on it */
    bool known;
};

/* The border of the entries not below `from` that top_k (0: off) and then the fraction top_p (1: off) of their weight
 * keep.  `total`: the weight of the row, needed where k is 0 and a bin is not one key.  All threads of the cluster call it with the
 * same arguments; `lv` may lie in the place of `bins`.  (Copies of the row and the weights: references would keep the
 * caller's in memory.) */
template <class T, bool RESIDENT>
__device__ __noinline__ Border border_by_bins(const Row<T, RESIDENT> share, FineBins &bins, Level &lv, unsigned size,
                                              const Weigh weigh, float from, float most, u64 k, double top_p, u64 total, BlockPart &part) {
    constexpr int E = Elem<T>::E;
    constexpr bool EXACT = Elem<T>::kShift == 16; /* a bin that is not shared is one key */
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const unsigned rank = cluster_rank();
    const BinOrder order(most, from);
    u64 coarse[2], own_coarse[2];
    count_bins(share, bins, order, weigh, from, own_coarse);
    if (t < (int)size) peer_store(peer_addr(shared_addr(&bins.shared[rank][0]), t), own_coarse[0], own_coarse[1]);
    cluster_sync(size);
    coarse[0] = coarse[1] = 0;
    for (unsigned r = 0; r < size; ++r) coarse[0] += bins.shared[r][0], coarse[1] += bins.shared[r][1];
    /* every block adds up a slice of the bins of all */
    const int slice = (kFineBins + (int)size - 1) / (int)size, per = (slice + kThreads - 1) / kThreads;
    const int bin0 = min(kFineBins, (int)rank * slice + min(slice, t * per)), bin1 = min(kFineBins, (int)rank * slice + min(slice, t * per + per));
    const int middle = order.middle, last = order.last;
    auto counted = [&](int bin) -> u64 {
        const unsigned at = shared_addr(&bins.count[bin]);
        unsigned n = 0;
#pragma unroll
        for (unsigned r = 0; r < kMaxCluster; ++r)
            if (r < size) n += peer_load32(peer_addr(at, r));
        return n;
    };
    auto weighed = [&](int bin, bool high) -> u64 {
        if (bin == middle) return coarse[0];
        if (bin == last) return coarse[1];
        const u64 n = counted(bin);
        /* the maximum's bin ends above the maximum, where scores have no weight */
        return n ? n * weigh.weight(fminf(value_of(key_of_bin<EXACT>(order, bin, high)), weigh.top)) : 0;
    };
    /* the first bin up to which the sum of `of` reaches what `goal` makes of the whole sum, or -1; what precedes it.
     * Search 0 and 1 of a call. */
    u64 before = 0;
    unsigned equals = 0;
    auto find = [&](int search, auto of, auto goal) {
        u64 mine = 0;
#pragma unroll 3
        for (int bin = bin0; bin < bin1; ++bin) mine += of(bin);
        u64 upto = warp_scan(mine), block = 0, all = 0;
        if (lane == 31) bins.warp[warp] = upto;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) upto += bins.warp[w];
            block += bins.warp[w];
        }
        if (t < (int)size) peer_store1(peer_addr(shared_addr(&bins.total[search][rank]), t), block);
        cluster_sync(size);
        for (unsigned r = 0; r < size; ++r) {
            if (r < rank) upto += bins.total[search][r];
            all += bins.total[search][r];
        }
        const u64 target = goal(all);
        u64 sum = upto - mine;
        if (sum < target && target <= upto) {
#pragma unroll 1
            for (int bin = bin0; bin < bin1; ++bin) {
                const u64 w = of(bin);
                if (sum < target && target <= sum + w)
                    for (unsigned r = 0; r < size; ++r)
                        peer_store(peer_addr(shared_addr(&bins.found[search][0]), r), sum, counted(bin) << 32 | (unsigned)bin);
                sum += w;
            }
        }
        cluster_sync(size);
        before = bins.found[search][0];
        const u64 f = bins.found[search][1];
        equals = (unsigned)(f >> 32);
        __syncthreads();
        return f == ~0ull ? -1 : (int)(unsigned)f;
    };
    if (k > 0) {
        const int bin = find(0, counted, [&](u64) { return k; });
        if (bin < 0) { /* fewer than k */
            if (!(top_p < 1.0)) return Border{key_of(neg_inf()), 0, 0};
            return find_border<T, RESIDENT, true>(share, lv, size, key_of(from), key_of(most), 0, weigh, top_p, 0);
        }
        Border border{key_of_bin<EXACT>(order, bin, false), (unsigned)(k - before), equals};
        if (!EXACT || bin == middle || bin == last) {
            border = find_border<T, RESIDENT, false>(share, lv, size, order.lowest(bin) << 16, order.highest(bin) << 16 | 0xffffu, k - before, weigh, 0.0, 0);
        } else if (!(top_p < 1.0)) {
            part.mass = weight_before(bins, order, weigh, own_coarse, bin), part.ties = bins.count[bin], part.known = true;
            __syncthreads();
        }
        if (!(top_p < 1.0)) return border;
        const Border b = find_border<T, RESIDENT, true>(share, lv, size, border.key, key_of(most), 0, weigh, top_p, border.equals - border.ties);
        return b.ties != 0xffffffffu ? b : border;
    }
    /* by weight: of a bin that is not one key only bounds are known, that of its lowest and of its highest score */
    u64 target = 0;
    auto goal = [&](u64 all) { return target = max(1ull, (u64)ceil(top_p * (double)(EXACT ? all : total))); };
    int to = find(0, [&](int bin) { return weighed(bin, false); }, goal), first = to;
    if (EXACT && to >= 0 && to != middle && to != last) {
        const unsigned key = key_of_bin<EXACT>(order, to, false);
        const u64 w = weigh.weight(value_of(key));
        part.mass = weight_before(bins, order, weigh, own_coarse, to), part.ties = bins.count[to], part.known = true;
        __syncthreads();
        return Border{key, (unsigned)min((target - before + w - 1) / w, (u64)equals), equals};
    }
    if (!EXACT) first = find(1, [&](int bin) { return weighed(bin, true); }, goal);
    const unsigned klo = to < 0 ? key_of(from) : max(key_of(from), order.lowest(to) << 16);
    const unsigned khi = first < 0 ? key_of(most) : order.highest(first) << 16 | 0xffffu;
    if (!EXACT) { /* what lies above the first bin that may hold the border */
        u64 more = 0;
        const float above = value_of(khi);
        for (int v = share.first; v < share.last; v += 32) {
            const uint4 w = share.raw(v);
            typename Elem<T>::Max best;
            best.add(w);
            if (!(best.get() > above)) continue;
            float f[E];
            Elem<T>::unpack(w, f);
            more += (u64)weigh.some<E>(f, fmaxf(weigh.least, value_of(khi + 1u)), true);
        }
        more = warp_sum(more);
        if (lane == 0) bins.warp[warp] = more;
        __syncthreads();
        more = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) more += bins.warp[w];
        if (t < (int)size) peer_store1(peer_addr(shared_addr(&bins.shared[rank][0]), t), more);
        cluster_sync(size);
        before = 0;
        for (unsigned r = 0; r < size; ++r) before += bins.shared[r][0];
        __syncthreads();
    }
    const Border b = find_border<T, RESIDENT, true>(share, lv, size, klo, khi, target - before, weigh, 0.0, 0);
    return b.ties != 0xffffffffu ? b : Border{klo - 1, 0, 0};
}

}  // namespace accb_rows
