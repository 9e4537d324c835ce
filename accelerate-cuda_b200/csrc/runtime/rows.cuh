/*
 * rows.cuh -- what the operators over rows of scores (rows.cu) share: element
 * types, a row held on chip by a cluster of blocks, exchanges between the
 * blocks, and exact weights.
 *
 * A row of scores is longer than what the folds over rows see (10^4 to 10^6
 * entries) and has to be looked at several times: for its maximum, its sum of
 * exponentials, the value of its k-th entry, and once more for what is written.
 * So a row belongs to a cluster of 1 to 8 blocks.  Every block copies its
 * share of the row to shared memory once (cp.async, 16 bytes a thread), all
 * passes read that copy, and the blocks tell one another what they found
 * through distributed shared memory.  HBM sees the row once, up to eight
 * blocks' 192 KB; longer rows are read again by every pass (draws from 128
 * rows of 2^20 bf16 338 us, with top_p 0.9 1117).  No scratch memory is used
 * at all: launches on different streams or in captured graphs share nothing.
 *
 * Inside a block every warp owns a contiguous piece of the share, so that
 * sums over warps in order are sums over the row in order; a thread reads the
 * same vectors in every pass, which makes its own copies visible to it
 * without a barrier.
 *
 * What bounds them: not HBM (a copy of 1024 x 131072 bf16 takes 41 us, the
 * operators' single passes over it 15 to 30) but the chain of steps that a
 * row has to take one after the other -- fetch, maximum, sum, exchange, finish
 * -- each of which ends in a barrier of the cluster.  Hence three blocks an
 * SM, so that one computes while others wait, and as little code as possible
 * on the way: a block runs most of it once per row, and waiting for
 * instructions was half the time of the first versions.
 *
 * accelerate-cuda has no counterpart: its folds reduce a row with one block in
 * one pass (Data/Array/Accelerate/CUDA/CodeGen/Reduction.hs:221-367).
 */
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace accb_rows {

struct RowsIn {
    const void *x;
    long long rows, pitch; /* pitch in elements */
    int cols;
};

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
    int in0;
    unsigned in; /* vectors in0 .. in0 + in - 1 of the row lie wholly inside it */
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
        in0 = lead != 0;
        in = (unsigned)max(0, (lead + cols) / E - in0);
        stage = smem;
    }
    __device__ __forceinline__ int vectors() const { return (lead + n + E - 1) / E; } /* of the whole row */
    __device__ __forceinline__ int entry(int v) const { return v * E - lead; } /* index of a vector's first entry */
    __device__ __forceinline__ bool whole(int v) const { return (unsigned)(v - in0) < in; }

    __device__ __forceinline__ uint4 from_memory(int v) const {
        return whole(v) ? reinterpret_cast<const uint4 *>(base)[v] : edge<T>(base, v, lead, n);
    }
    /* start the copies of this thread's vectors; wait() before the first get().  No branch but at the edges of the row,
     * which are at most two vectors of all threads. */
    __device__ __forceinline__ void fetch() const {
        if (!RESIDENT) return;
        const uint4 *from = reinterpret_cast<const uint4 *>(base) + first;
        unsigned to = shared_addr(stage + (first - v0));
        const unsigned i0 = (unsigned)(first - in0);
#pragma unroll 4
        for (int d = 0; d < last - first; d += 32) {
            const int go = i0 + (unsigned)d < in;
            asm volatile(
                "{\n"
                ".reg .pred p;\n"
                "setp.ne.s32 p, %2, 0;\n"
                "@p cp.async.cg.shared.global [%0], [%1], 16;\n"
                "}\n" ::"r"(to + d * 16),
                "l"(from + d), "r"(go)
                : "memory");
        }
        if (in0 && first == 0 && last > 0) stage[0] = edge<T>(base, 0, lead, n);
        const int v = in0 + (int)in;
        if (v >= first && v < last && ((v - first) & 31) == 0) stage[v - v0] = edge<T>(base, v, lead, n);
    }
    __device__ __forceinline__ void wait() const {
        if (RESIDENT) asm volatile("cp.async.wait_all;" ::: "memory");
    }
    __device__ __forceinline__ uint4 get(int v) const { return RESIDENT ? stage[v - v0] : from_memory(v); }
};

/* A vector of a row of which `bits` does not allow all entries: the others are -inf. */
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
/* A vector of a row whose maximum is +inf: its like weigh 1, all others nothing. */
template <class T> __device__ __noinline__ uint4 only_infinite(uint4 w) {
    constexpr int E = Elem<T>::E;
    float f[E];
    Elem<T>::unpack(w, f);
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = f[i] == __uint_as_float(0x7f800000u) ? 0.0f : neg_inf();
    return Elem<T>::pack(f);
}

/* A share as the searches see it.  What changes a staged vector is applied to it once, by apply(); where the row is not
 * staged, whenever it is read. */
template <class T, bool RESIDENT> struct Row : Share<T, RESIDENT> {
    const unsigned *bits = nullptr; /* allowed entries */
    bool infinite = false;
    __device__ __forceinline__ uint4 changed(int v, uint4 w) const {
        if (bits) w = only_allowed<T>(w, this->entry(v), this->n, bits);
        if (infinite) w = only_infinite<T>(w);
        return w;
    }
    __device__ __forceinline__ uint4 raw(int v) const { return RESIDENT ? this->get(v) : changed(v, this->get(v)); }
    /* as floats, a NaN as -inf */
    __device__ __forceinline__ void floats(int v, float *f) const {
        Elem<T>::unpack(raw(v), f);
#pragma unroll
        for (int i = 0; i < Elem<T>::E; ++i) f[i] = not_nan(f[i]);
    }
    /* by all lanes of a warp, which see one another's vectors changed afterwards: gather() reads them */
    __device__ __forceinline__ void apply() const {
        for (int v = RESIDENT ? this->first : this->last; v < this->last; v += 32) this->stage[v - this->v0] = changed(v, this->get(v));
        __syncwarp();
    }
};

/* a vector of a result row laid out like the share's row; 16-byte stores where both start at the same place of a
 * 16-byte word, else entry by entry: the gradient from statistics of 1500 x 100003 fp16 takes 108 us with rows every
 * 100003 in scores and gradient, 101 with every 100032 in both, 365 to 377 with one of each */
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
 *     64 y = x c - N = K + r,  2^y = 2^(K >> 6) * table[K & 63] * polynomial(r),
 * c = 64 log2(e) / T, N the whole number next to top c (which leaves all weights of a row a common factor of at most
 * 2^(1/128)), K whole, |r| <= 1/2; x c is not rounded before N is taken off.  The polynomial is
 * the cubic Taylor one of 2^(r / 64), wrong by less than (ln 2 / 128)^4 / 24 < 2^-34.6 of itself: eight
 * 64-bit operations where the library's function takes some twenty.  The table is in shared memory sixteen times, a
 * copy for every lane of a half warp, so that no two lanes meet in a bank; entry j is stored with j << 14 taken from its
 * upper half, so that adding K << 14 there adds K >> 6 to the exponent. */
constexpr int kUnitLog2 = 43;
constexpr int kTable = 64;
constexpr int kTableCopies = 16;

static __device__ __noinline__ void fill_table(double *table) { /* kTable * kTableCopies; by all threads, a barrier follows */
    double v = exp2((double)(threadIdx.x % kTable) * (1.0 / kTable));
    v = __hiloint2double(__double2hiint(v) - ((threadIdx.x % kTable) << 14), __double2loint(v));
    for (int i = threadIdx.x / kTable; i < kTableCopies; i += kThreads / kTable) table[(threadIdx.x % kTable) * kTableCopies + i] = v;
}

struct Weigh {
    static constexpr double kRound = 6755399441055744.0; /* 1.5 * 2^52: adding it rounds to a whole number */
    float top, least;    /* scores below `least` weigh less than half a unit, or are excluded */
    double c;            /* 64 log2(e) / T */
    double start;        /* kRound less the whole number next to top * c: what that leaves is a factor of all weights */
    const double *table; /* this lane's copy */

    __device__ __forceinline__ Weigh(float maximum, double temperature, const double *shared_table) {
        top = maximum;
        table = shared_table + (threadIdx.x & (kTableCopies - 1));
        c = 64.0 * 1.4426950408889634 / temperature;
        /* so cold that any other score weighs nothing, and would not be told apart: the maxima have one weight each */
        if (!(fabs((double)top * c) < 1125899906842624.0)) c = 0.0;
        start = kRound - rint((double)top * c);
        least = fmaxf(-3.402823466e+38f, (float)((double)top - (kUnitLog2 + 2) * 0.69314718055994531 * temperature));
    }
    /* log of the weight of the maximum, in units */
    __device__ __forceinline__ double log_of_top() const { return fma((double)top, c, start - kRound) * (0.69314718055994531 / kTable); }
    /* for least <= f <= top; anything elsewhere */
    __device__ __forceinline__ u64 of(float f) const { return (u64)__double_as_longlong(above_2_52(f)) & 0xfffffffffffffull; }
    /* 2^52 + the weight */
    __device__ __forceinline__ double above_2_52(float f) const {
        constexpr double l = 0.69314718055994531 / kTable;
        const double x = (double)f, t = fma(x, c, start);
        const int k = __double2loint(t);
        const double r = fma(x, c, start - t);
        double m = table[(k & (kTable - 1)) * kTableCopies];
        m = __hiloint2double(__double2hiint(m) + (k << 14), __double2loint(m));
        const double unit = (double)(1ull << kUnitLog2);
        /* 2^52 makes a unit of 2^-43 the last bit */
        return fma(m, fma(fma(fma(unit * l * l * l / 6.0, r, unit * l * l / 2.0), r, unit * l), r, unit), 4503599627370496.0);
    }
    __device__ __forceinline__ u64 weight(float f) const { return f >= least ? of(f) : 0; }
    /* The weight of those of a vector's scores that are not below `from` (at least `least`): one after the other where
     * they are few; else, or where `most` are said to be, all of them side by side and without a branch, which hides the
     * latency of the 64-bit operations.  Sums of up to 512 weights are exact in a double.  Unless `most`, all lanes of a
     * warp call it together. */
    template <int E> __device__ __forceinline__ double some(const float (&f)[E], float from, bool most) const {
        unsigned found = 0;
        if (!most) {
#pragma unroll
            for (int i = 0; i < E; ++i) found |= (unsigned)(f[i] >= from) << i;
        }
        double sum = 0.0;
        if (most || __any_sync(~0u, __popc(found) > 2)) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const double w = above_2_52(f[i]) - 4503599627370496.0;
                if (f[i] >= from) sum += w;
            }
        } else {
            for (; found; found &= found - 1) {
                float x = f[0];
#pragma unroll
                for (int i = 1; i < E; ++i)
                    if ((found >> i) & 1u && !(found & ((1u << i) - 1u))) x = f[i];
                sum += above_2_52(x) - 4503599627370496.0;
            }
        }
        return sum;
    }
};

}  // namespace accb_rows
