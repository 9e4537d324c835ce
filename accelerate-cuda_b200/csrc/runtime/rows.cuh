/*
 * rows.cuh -- what the operators over rows of scores (rows.cu) share: a row
 * held on chip by a cluster of blocks, exchanges between its warps, and the
 * search for the border of a row's best entries.
 *
 * A row of scores is longer than what the folds over rows see (10^4 to 10^6
 * entries) and has to be looked at several times: for its maximum, its sum of
 * exponentials, the value of its k-th entry, and once more for what is written.
 * So a row belongs to a cluster of 1 to 8 blocks.  Every block copies its
 * share of the row to shared memory once (cp.async, 16 bytes a thread), all
 * passes read that copy, and the blocks tell one another what they found
 * through distributed shared memory.  HBM sees the row once.  No scratch
 * memory is used at all: launches on different streams or in captured graphs
 * share nothing.
 *
 * Inside a block every warp owns a contiguous piece of the share, so that
 * sums over warps in order are sums over the row in order; a thread reads the
 * same vectors in every pass, which makes its own copies visible to it
 * without a barrier.
 *
 * accelerate-cuda has no counterpart: its folds reduce a row with one block in
 * one pass (Data/Array/Accelerate/CUDA/CodeGen/Reduction.hs:221-367).
 */
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace accb_rows {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = kThreads;        /* bins of one level of the border search: one per thread */
constexpr int kMaxK = 1024;            /* most entries of a top list */
constexpr long long kMaxCols = 1 << 20;

typedef unsigned long long u64;

/* ------------------------------------------------------- element types */
template <class T> struct Elem;
template <> struct Elem<float> {
    static constexpr int E = 4;
    static constexpr int kShift = 0; /* low bits of key_of() that never tell two values apart */
    static constexpr unsigned kLowest = 0xff800000u; /* -inf, as often as it fits into 32 bits */
    static __device__ __forceinline__ void unpack(const uint4 &w, float *f) {
        f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ uint4 pack(const float *f) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
    /* running maximum of whole vectors; a NaN is passed over */
    struct Max {
        float m;
        __device__ __forceinline__ Max() : m(-__builtin_huge_valf()) {}
        __device__ __forceinline__ void add(const uint4 &w) {
            m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(w.x), __uint_as_float(w.y))), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
        }
        __device__ __forceinline__ float get() const { return m; }
    };
};
template <> struct Elem<__half> {
    static constexpr int E = 8;
    static constexpr int kShift = 13;
    static constexpr unsigned kLowest = 0xfc00fc00u;
    static __device__ __forceinline__ void unpack(const uint4 &w, float *f) {
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            f[2 * i] = p.x, f[2 * i + 1] = p.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float *f) {
        unsigned u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            u[i] = *reinterpret_cast<const unsigned *>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
    static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
    struct Max {
        unsigned m = 0xfc00fc00u;
        static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
            const __half2 r = __hmax2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
            return *reinterpret_cast<const unsigned *>(&r);
        }
        __device__ __forceinline__ void add(const uint4 &w) { m = larger(larger(m, larger(w.x, w.y)), larger(w.z, w.w)); }
        __device__ __forceinline__ float get() const {
            const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&m));
            return fmaxf(p.x, p.y);
        }
    };
};
template <> struct Elem<__nv_bfloat16> {
    static constexpr int E = 8;
    static constexpr int kShift = 16;
    static constexpr unsigned kLowest = 0xff80ff80u;
    static __device__ __forceinline__ void unpack(const uint4 &w, float *f) {
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(u[i] << 16), f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
    static __device__ __forceinline__ uint4 pack(const float *f) {
        unsigned u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            u[i] = *reinterpret_cast<const unsigned *>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
    static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
    struct Max {
        unsigned m = 0xff80ff80u;
        static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
            const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
            return *reinterpret_cast<const unsigned *>(&r);
        }
        __device__ __forceinline__ void add(const uint4 &w) { m = larger(larger(m, larger(w.x, w.y)), larger(w.z, w.w)); }
        __device__ __forceinline__ float get() const {
            const float2 p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&m));
            return fmaxf(p.x, p.y);
        }
    };
};

/* ------------------------------------------- two 32-bit floats at a time
 * Blackwell adds, multiplies and fuses pairs of 32-bit floats in one instruction; the passes over a row are bound by
 * instruction issue, so they use them. */
struct Pair {
    u64 v;
    __device__ __forceinline__ Pair() {}
    __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void get(float &a, float &b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
/* 2^x by the special function unit (relative error 2^-22, results below 2^-126 are 0) */
__device__ __forceinline__ float fast_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ Pair fast_exp2(Pair x) {
    float a, b;
    x.get(a, b);
    return Pair(fast_exp2(a), fast_exp2(b));
}

__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xff800000u); }
/* a NaN is an entry that cannot be chosen, like -inf (fmaxf returns the operand that is a number) */
__device__ __forceinline__ float not_nan(float f) { return fmaxf(f, neg_inf()); }

/* unsigned keys in the order of the values; -0 and +0 are equal */
__device__ __forceinline__ unsigned key_of(float f) {
    const unsigned b = __float_as_uint(f + 0.0f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k); }

/* ------------------------------------------------------------- clusters */
__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_size() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync(unsigned size) {
    if (size == 1) {
        __syncthreads();
    } else {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
}
__device__ __forceinline__ unsigned shared_addr(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
/* the address of this block's shared variable in the block of the given rank */
__device__ __forceinline__ unsigned peer_addr(unsigned addr, unsigned rank) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void peer_store(unsigned addr, u64 a, u64 b) { /* 16-byte aligned */
    asm volatile("st.shared::cluster.v2.u64 [%0], {%1, %2};" ::"r"(addr), "l"(a), "l"(b) : "memory");
}
__device__ __forceinline__ void peer_store1(unsigned addr, u64 a) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(a) : "memory");
}
__device__ __forceinline__ uint4 peer_load(unsigned addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ u64 peer_load1(unsigned addr) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ unsigned peer_load32(unsigned addr) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ unsigned peer_count(unsigned addr, unsigned n) {
    unsigned old;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(n) : "memory");
    return old;
}

/* ----------------------------------------------------------------- rows */
/* A block runs most of its code once per row, so what counts of rarely run code is its size: every instruction that
 * is not in the SM's instruction cache is waited for.  Edges and 64-bit functions are therefore calls. */
template <class T> __device__ __noinline__ uint4 edge(const T *base, int v, int lead, int n) {
    constexpr int E = Elem<T>::E;
    T f[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int e = v * E - lead + i;
        f[i] = e >= 0 && e < n ? base[v * E + i] : Elem<T>::down(neg_inf());
    }
    uint4 w;
    memcpy(&w, f, sizeof w);
    return w;
}
template <class T> __device__ __noinline__ void put_edge(T *row, int v, int lead, int n, uint4 w) {
    constexpr int E = Elem<T>::E;
    T f[E];
    memcpy(f, &w, sizeof w);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int e = v * E - lead + i;
        if (e >= 0 && e < n) row[e] = f[i];
    }
}
static __device__ __noinline__ double exp_64(double x) { return exp(x); }
static __device__ __noinline__ double log_64(double x) { return log(x); }

/* A block's share of one row, in vectors of 16 bytes counted from the row's address rounded down to 16 bytes.
 * Entries of an edge vector that lie outside the row read as -inf.  Which vectors a thread has, and where they are
 * staged, is the same for all rows of a matrix, wherever they start: a thread may replace its own vectors by those of
 * the next row as soon as it has read them. */
template <class T, bool RESIDENT> struct Share {
    static constexpr int E = Elem<T>::E;
    const T *base;   /* the row's address rounded down to 16 bytes */
    int lead;        /* entries between base and the row's first */
    int n;           /* entries of the row */
    int v0, v1;      /* this block's vectors */
    int first, last; /* this thread's: first, first + 32, ... below last */
    uint4 *stage;

    static __host__ __device__ __forceinline__ int per_block(int cols, int size) { /* vectors of a share, at most */
        return ((cols + 2 * E - 2) / E + size - 1) / size;
    }
    __device__ __forceinline__ void init(const T *row, int cols, unsigned rank, unsigned size, uint4 *smem) {
        lead = (int)((reinterpret_cast<unsigned long long>(row) & 15u) / sizeof(T));
        base = row - lead;
        n = cols;
        const int nvec = (lead + cols + E - 1) / E, per = per_block(cols, (int)size);
        v0 = (int)rank * per;
        v1 = max(v0, min(nvec, v0 + per));
        const int piece = ((per + kWarps - 1) / kWarps + 31) & ~31;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        first = v0 + warp * piece + lane;
        last = min(v1, v0 + (warp + 1) * piece);
        stage = smem;
    }
    __device__ __forceinline__ int entry(int v) const { return v * E - lead; } /* index of a vector's first entry */
    __device__ __forceinline__ bool whole(int v) const { return entry(v) >= 0 && entry(v) + E <= n; }

    __device__ __forceinline__ uint4 from_memory(int v) const {
        return whole(v) ? reinterpret_cast<const uint4 *>(base)[v] : edge<T>(base, v, lead, n);
    }
    /* start the copies of this thread's vectors; wait() before the first get() */
    __device__ __forceinline__ void fetch() const {
#pragma unroll 4
        for (int v = RESIDENT ? first : last; v < last; v += 32) {
            if (whole(v))
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_addr(stage + (v - v0))),
                             "l"(reinterpret_cast<const uint4 *>(base) + v)
                             : "memory");
            else
                stage[v - v0] = edge<T>(base, v, lead, n);
        }
    }
    __device__ __forceinline__ void wait() const {
        if (RESIDENT) asm volatile("cp.async.wait_all;" ::: "memory");
    }
    __device__ __forceinline__ uint4 get(int v) const { return RESIDENT ? stage[v - v0] : from_memory(v); }
};

/* a vector of a result row laid out like the share's row; 16-byte stores where both start at the same place of a
 * 16-byte word */
template <class T, bool R> __device__ __forceinline__ void put(const Share<T, R> &share, T *row, bool same, int v, const uint4 &w) {
    if (same && share.whole(v))
        *reinterpret_cast<uint4 *>(row + share.entry(v)) = w;
    else
        put_edge<T>(row, v, share.lead, share.n, w);
}

/* --------------------------------------------------------- reductions */
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, d));
    return v;
}
__device__ __forceinline__ float warp_min(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = fminf(v, __shfl_xor_sync(~0u, v, d));
    return v;
}
template <class V> __device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
}
template <class V> __device__ __forceinline__ V warp_scan(V v) { /* inclusive */
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const V o = __shfl_up_sync(~0u, v, d);
        if (lane >= d) v += o;
    }
    return v;
}

/* -------------------------------------------------------------- weights */
/* The share of an entry is exp((x - top) / T), top the row's maximum.  It is held as a whole number in units of 2^-43,
 * so that sums do not depend on their order -- on how a row is split over warps and blocks -- and a million entries
 * (kMaxCols) still fit into 64 bits.  Two indices are told apart by a sum: an error of 2^-24 of each of 10^5 like
 * entries would pick the wrong one every few thousand rows.  So 2^y is computed in 64 bits:
 *     64 y = K + r, K whole, |r| <= 1/2;  2^y = 2^(K >> 6) * table[K & 63] * polynomial(r)
 * with the cubic Taylor polynomial of 2^(r / 64), wrong by less than (ln 2 / 128)^4 / 24 < 2^-34.6 of itself: eight
 * 64-bit operations where the library's function takes some twenty.  The table is in shared memory sixteen times, a
 * copy for every lane of a half warp, so that no two lanes meet in a bank. */
constexpr int kUnitLog2 = 43;
constexpr int kTable = 64;
constexpr int kTableCopies = 16;

static __device__ __noinline__ void fill_table(double *table) { /* kTable * kTableCopies; by all threads, a barrier follows */
    const double v = exp2((double)(threadIdx.x % kTable) * (1.0 / kTable));
    for (int i = threadIdx.x / kTable; i < kTableCopies; i += kThreads / kTable) table[(threadIdx.x % kTable) * kTableCopies + i] = v;
}

/* WIDE: scores of 24 bits, whose distance from the maximum takes 64 bits.  That of two 16-bit scores is exact in 32,
 * but for scores nearer to 0 than 2^-16 of the maximum, where it is off by 2^-25 of itself. */
template <bool WIDE> struct Weigh {
    static constexpr double kRound = 6755399441055744.0; /* 1.5 * 2^52: adding it rounds to a whole number */
    float top, least;    /* scores below `least` weigh less than half a unit, or are excluded */
    double c;            /* 64 log2(e) / T */
    const double *table; /* this lane's copy */

    __device__ __forceinline__ Weigh(float maximum, double temperature, const double *shared_table) {
        top = maximum;
        table = shared_table + (threadIdx.x & (kTableCopies - 1));
        c = 64.0 * 1.4426950408889634 / temperature;
        least = fmaxf(-3.402823466e+38f, (float)((double)top - (kUnitLog2 + 2) * 0.69314718055994531 * temperature));
    }
    /* for f >= least; anything below */
    __device__ __forceinline__ u64 of(float f) const {
        constexpr double l = 0.69314718055994531 / kTable;
        const double x = WIDE ? (double)f - (double)top : (double)(f - top);
        const double t = fma(x, c, kRound);
        const int k = __double2loint(t);
        const double r = fma(x, c, kRound - t);
        double m = table[(k & (kTable - 1)) * kTableCopies];
        m = __hiloint2double(__double2hiint(m) + ((k & ~(kTable - 1)) << 14), __double2loint(m));
        const double unit = (double)(1ull << kUnitLog2);
        /* 2^52 makes a unit of 2^-43 the last bit */
        m = fma(m, fma(fma(fma(unit * l * l * l / 6.0, r, unit * l * l / 2.0), r, unit * l), r, unit), 4503599627370496.0);
        return (u64)__double_as_longlong(m) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 weight(float f) const { return f >= least ? of(f) : 0; }
    /* The weight of those of a vector's scores (none below `least`) that `wanted` takes: one after the other where they
     * are few; else all of them side by side, without a branch, which hides the latency of the 64-bit operations. */
    template <int E, class F> __device__ __forceinline__ u64 some(const float (&f)[E], F wanted) const {
        unsigned found = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) found |= (unsigned)(wanted(f[i]) && f[i] >= least) << i;
        u64 sum = 0;
        if (__popc(found) > 2) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const u64 w = of(f[i]);
                sum += (found >> i) & 1u ? w : 0;
            }
        } else {
            for (; found; found &= found - 1) {
                float x = f[0];
#pragma unroll
                for (int i = 1; i < E; ++i)
                    if ((found >> i) & 1u && !(found & ((1u << i) - 1u))) x = f[i];
                sum += of(x);
            }
        }
        return sum;
    }
};

/* ------------------------------------------------------ candidate lists */
/* An entry as one number: larger for larger scores and, among equal ones, for lower indices.  0 is no entry. */
__device__ __forceinline__ u64 entry_of(float f, int index) { return (u64)key_of(f) << 32 | (0xffffffffu - (unsigned)index); }
__device__ __forceinline__ float score_of(u64 e) { return value_of((unsigned)(e >> 32)); }
__device__ __forceinline__ int index_of(u64 e) { return (int)(0xffffffffu - (unsigned)e); }

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
template <class T, bool RESIDENT, bool BY_MASS, class Get>
__device__ Border find_border(const Share<T, RESIDENT> &share, Get get, Level &lv, unsigned size, unsigned klo, unsigned khi,
                              u64 target, const Weigh<sizeof(T) == 4> &weigh, double fraction, unsigned spare) {
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
            get(v, f);
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
template <class T, bool RESIDENT, class Raw>
__device__ void count_bins(const Share<T, RESIDENT> &share, Raw raw, FineBins &bins, const BinOrder &order, const Weigh<sizeof(T) == 4> &weigh, float from,
                           u64 (&coarse)[2]) {
    constexpr int E = Elem<T>::E;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
#pragma unroll
    for (int i = 0; i < kFineBins / kThreads / 4; ++i) *reinterpret_cast<uint4 *>(&bins.count[4 * (t + i * kThreads)]) = make_uint4(0, 0, 0, 0);
    if (t < 2) bins.found[t][1] = ~0ull;
    if (t == 0) bins.n_near = 0;
    __syncthreads();
    for (int v = share.first; v < share.last; v += 32) {
        const uint4 w = raw(v);
        typename Elem<T>::Max best;
        best.add(w);
        if (!(best.get() >= from)) continue;
        float f[E];
        Elem<T>::unpack(w, f);
        unsigned near = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const bool in = f[i] >= from;
            if (in) atomicAdd(&bins.count[order.of(f[i])], 1u);
            near |= (unsigned)(in && order.shared(f[i])) << i;
        }
        if (near) {
            unsigned at = atomicAdd(&bins.n_near, __popc(near));
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (((near >> i) & 1u) && at < kNear) bins.near[at++] = f[i];
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
            Elem<T>::unpack(raw(v), f);
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
template <bool WIDE> __device__ u64 weight_before(FineBins &bins, const BinOrder &order, const Weigh<WIDE> &weigh, const u64 (&coarse)[2], int end) {
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
 * same arguments; `lv` may lie in the place of `bins`. */
template <class T, bool RESIDENT, class Raw, class Get>
__device__ Border border_by_bins(const Share<T, RESIDENT> &share, Raw raw, Get get, FineBins &bins, Level &lv, unsigned size,
                                 const Weigh<sizeof(T) == 4> &weigh, float from, float most, u64 k, double top_p, u64 total, BlockPart &part) {
    constexpr int E = Elem<T>::E;
    constexpr bool EXACT = Elem<T>::kShift == 16; /* a bin that is not shared is one key */
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const unsigned rank = cluster_rank();
    const BinOrder order(most, from);
    u64 coarse[2], own_coarse[2];
    count_bins(share, raw, bins, order, weigh, from, own_coarse);
    if (t < (int)size) peer_store(peer_addr(shared_addr(&bins.shared[rank][0]), t), own_coarse[0], own_coarse[1]);
    cluster_sync(size);
    coarse[0] = coarse[1] = 0;
    for (unsigned r = 0; r < size; ++r) coarse[0] += bins.shared[r][0], coarse[1] += bins.shared[r][1];
    /* every block adds up a slice of the bins of all */
    const int slice = kFineBins / (int)size, per = (slice + kThreads - 1) / kThreads;
    const int bin0 = (int)rank * slice + min(slice, t * per), bin1 = (int)rank * slice + min(slice, t * per + per);
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
        return n ? n * weigh.weight(value_of(key_of_bin<EXACT>(order, bin, high))) : 0;
    };
    /* the first bin up to which the sum of `of` reaches what `goal` makes of the whole sum, or -1; what precedes it.
     * Search 0 and 1 of a call. */
    u64 before = 0;
    unsigned equals = 0;
    auto find = [&](int search, auto of, auto goal) {
        u64 mine = 0;
#pragma unroll 1
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
            k = 0;
            if (!(top_p < 1.0)) return Border{key_of(neg_inf()), 0, 0};
            return find_border<T, RESIDENT, true>(share, get, lv, size, key_of(from), key_of(most), 0, weigh, top_p, 0);
        }
        Border border{key_of_bin<EXACT>(order, bin, false), (unsigned)(k - before), equals};
        if (!EXACT || bin == middle || bin == last)
            border = find_border<T, RESIDENT, false>(share, get, lv, size, order.lowest(bin) << 16, order.highest(bin) << 16 | 0xffffu, k - before, weigh, 0.0, 0);
        if (!(top_p < 1.0)) return border;
        const Border b = find_border<T, RESIDENT, true>(share, get, lv, size, border.key, key_of(most), 0, weigh, top_p, border.equals - border.ties);
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
            const uint4 w = raw(v);
            typename Elem<T>::Max best;
            best.add(w);
            if (!(best.get() > above)) continue;
            float f[E];
            Elem<T>::unpack(w, f);
            more += weigh.template some<E>(f, [&](float x) { return x > above; });
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
    const Border b = find_border<T, RESIDENT, true>(share, get, lv, size, klo, khi, target - before, weigh, 0.0, 0);
    return b.ties != 0xffffffffu ? b : Border{klo - 1, 0, 0};
}

}  // namespace accb_rows
