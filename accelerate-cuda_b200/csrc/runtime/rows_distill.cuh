/*
 * rows_distill.cuh -- the divergence of every row from a teacher's best entries, and its gradient (accb_distill_rows,
 * accb_distill_rows_backward).
 */
#pragma once
#include "rows.cuh"

namespace accb_rows {

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
    int first;   /* the first of its index in the list */
};

/* Where the best of the entries not named is less likely than this share of the row's best, the statistics hold the
 * gradient of the others by their own maximum: q, and q times a factor that is a share of 1 / q_r, would leave the range
 * of 32 bits.  Marked by a negative second number; top, -1 / sum, others_top, factor of exp((x - others_top) / tau). */
constexpr float kApart = 2.328306437e-10f; /* 2^-32 */

/* exp((a - b) / tau) for a <= b; inverse = 1 / tau, c = log2(e) / tau.  With k the whole number next to its exponent to
 * base two, 2^k times the Taylor polynomial of degree 9 of x = (a - b) / tau - k ln 2, |x| < 0.347.  64-bit operations are
 * what it waits for, so the terms from x^5 on, 5e-5 at most, are added up in 32 bits: wrong by less than 2^-32 of itself
 * (ten roundings of 2^-24 of 5e-5, and 0.347^10 / 10! = 7e-12, over exp(x) >= 0.7).  For terms that are not one of many:
 * the special function unit's error of 2^-22 of a named entry, which may have most of the row's weight, would be the
 * loss's (1024 x 131072 bf16, loss 0.06: off by 6e-8 root mean square, with these 2e-9, at 531 us a step over 4096 such
 * rows in place of 525). */
__device__ __forceinline__ double exp_below(float a, float b, double inverse, float c) {
    const float y = (a - b) * c;
    const int k = __float2int_rn(y);
    const double x = fma((double)a - (double)b, inverse, (double)k * -0.69314718055994531), x2 = x * x;
    const float s = (float)x, s2 = s * s;
    float rest = fmaf(1.0f / 362880.0f, s, 1.0f / 40320.0f);
    rest = fmaf(rest, s, 1.0f / 5040.0f);
    rest = fmaf(rest, s, 1.0f / 720.0f);
    rest = fmaf(rest, s, 1.0f / 120.0f);
    rest *= s2 * s2 * s;
    const double e = fma(fma(1.0 / 24.0, x2, fma(1.0 / 6.0, x, 0.5)), x2, 1.0 + x) + (double)rest;
    /* a NaN stays one, at k = 0 */
    return y < -1000.0f ? 0.0 : __hiloint2double(__double2hiint(e) + (k << 20), __double2loint(e));
}

/* The row as all its blocks know it. */
struct RowSums {
    float top, others_top;         /* maximum of the row, and of the entries not named (-inf: none) */
    double sum, others_sum, cross; /* sums of exponentials below those maxima; sum of p (teacher's - student's score) / tau */
};

/* Where an index is named twice: not whichever thread came first but the first in the list counts, so that sums are taken
 * in one order.  Returns the largest of the student's scores of this thread's. */
static __device__ __noinline__ float settle_firsts(Named *named, int k) {
    float most = neg_inf();
    for (int j = threadIdx.x; j < k; j += kThreads) {
        Named &n = named[j];
        bool first = n.at >= 0;
        for (int o = 0; o < j && first; ++o) first = named[o].at != n.at;
        n.first = first;
        if (first) most = fmaxf(most, n.z);
    }
    return most;
}

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

/* With x the student's scores, q = softmax(x / tau), p the teacher's probabilities and r what they leave of 1:
 *     loss = sum p (log p - log q) + r (log r - log q_r),  q_r = the sum of q over the entries not named
 *          = sum p (teacher - x) / tau + sum p (lse - shift) + r (log r - log q_r)
 *     d loss / d x = ((sum p + r) q - p) / tau at named entries, (sum p + r - r / q_r) q / tau elsewhere.
 * The named entries leave the staged row before it is summed: q_r is a sum of its own, not a difference of like numbers.
 * Maximum and sum are taken per warp, each by itself, and joined once per row by one warp of every block; the gradient is
 * written from the staged copy everywhere as if no entry were named, then the named ones once more.
 *
 * Loss and gradient of 4096 x 131072 bf16, 64 named, with the rest: 531 us, 3.9 TB/s, 60 % of the copy rate; the special
 * function unit, two exponentials an entry, is busy for 47 % and the row's chain of steps is the rest.  The loss alone of
 * 2048 x 50257 floats: 124 us, half of the copy rate.  The gradient from statistics needs no exchange and is bound by HBM
 * (1024 x 131072 bf16 89 us, 92 % of the copy rate); where rows start anywhere, as 1500 x 100003 fp16 do, 107 us, 84 %.
 * One row per cluster: clusters that stay and fetch the next row in the place of this one, vector by vector behind
 * the gradient pass, took 560 us; 2 blocks an SM the same as 3, blocks of 128, 384, 512 and
 * 1024 threads more.
 *
 * BACKWARD: the statistics are given, and no block needs the others. */
template <class T, bool R, bool BACKWARD> __global__ void __launch_bounds__(kThreads, 3) distill_rows(const __grid_constant__ DistillParams p) {
    constexpr int E = Elem<T>::E;
    extern __shared__ uint4 dynamic[];
    __shared__ double scratch[kWarps];
    __shared__ float warp_top[kWarps];
    __shared__ alignas(16) u64 told[kMaxCluster * kWarps][4];
    __shared__ float4 statistics;
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
    if (!BACKWARD && twice) most_named = settle_firsts(named, p.k);

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
        /* exponents and exponentials of the many in 32 bits, added up by thread and warp in 32 and from there in 64: their
         * errors, 2^-22 of a term, average out (c in two parts brought the loss no closer: 8e-8 off, with one 6e-8, 1.3 large) */
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
                    if (named[j].first) named_sum += exp_below(named[j].z, named_base, inv, c);
                named_sum = warp_sum(named_sum);
            }
            cross = warp_sum(cross);
        }
        const double others = (double)warp_sum(part_a + part_b);
        if (size > 1) cluster_wait();
        if (lane < (int)size) {
            const unsigned to = peer_addr(shared_addr(&told[rank * kWarps + warp][0]), lane);
            peer_store(to, __double_as_longlong(others), __double_as_longlong(named_sum));
            peer_store(to + 16, __double_as_longlong(cross), (u64)__float_as_uint(most) << 32 | __float_as_uint(rest ? most_named : neg_inf()));
        }
        cluster_sync(size);
        if (!grad && rank != 0) return;
        /* one warp adds up what all warps of the row found, and says what the gradient needs */
        if (warp == 0) {
            const int n = (int)size * kWarps;
            RowSums all{neg_inf(), neg_inf(), 0.0, 0.0, 0.0};
            for (int i = lane; i < n; i += 32) {
                all.others_top = fmaxf(all.others_top, __uint_as_float((unsigned)(told[i][3] >> 32)));
                all.top = fmaxf(all.top, __uint_as_float((unsigned)told[i][3]));
            }
            all.others_top = warp_max(all.others_top);
            all.top = rest ? fmaxf(all.others_top, warp_max(all.top)) : all.others_top;
            for (int i = lane; i < n; i += 32) {
                /* a sum that is 0 belongs to no entry; one that is not, at a maximum of -inf, to entries that are NaN */
                const double a = __longlong_as_double((long long)told[i][0]), b = __longlong_as_double((long long)told[i][1]);
                const float at_a = __uint_as_float((unsigned)(told[i][3] >> 32)), at_b = __uint_as_float((unsigned)told[i][3]);
                const double of_a = exp_below(at_a, all.others_top, inv, c), of_b = exp_below(at_b, all.top, inv, c);
                if (a != 0.0) all.others_sum += a * of_a;
                if (b != 0.0) all.sum += b * of_b;
                all.cross += __longlong_as_double((long long)told[i][2]);
            }
            all.others_sum = warp_sum(all.others_sum);
            if (rest) all.sum = warp_sum(all.sum);
            const double down = rest ? exp_below(all.others_top, all.top, inv, c) : 1.0; /* from one maximum to the other */
            if (all.others_sum != 0.0) all.sum += all.others_sum * down;
            const bool excluded = all.top == neg_inf() && all.sum == 0.0; /* by the student, every entry */
            double r = rest && all.others_top > neg_inf() ? fmax(0.0, 1.0 - named_p) : 0.0;
            float4 said = make_float4(all.top, (float)(1.0 / all.sum), (float)(named_p + r), (float)(named_p + r));
            if (r > 0.0 && down >= kApart)
                said.w = (float)(named_p + r - r * (all.sum / all.others_sum / down));
            else if (r > 0.0)
                said = make_float4(all.top, -said.y, all.others_top, (float)((named_p + r) * (double)said.y * down - r / all.others_sum));
            if (excluded) said = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (lane == 0) statistics = said;
            if (rank == 0) {
                all.cross = warp_sum(all.cross) - (named_p != 0.0 ? named_p * shift : 0.0); /* of an infinite shift nothing is named */
                const float loss = excluded ? 0.0f : row_loss(all, named_p, rest ? 1.0 : total, r, inv);
                if (lane == 0) {
                    p.loss[row] = weight * loss;
                    if (p.stats) {
                        float *s = p.stats + row * 4;
                        s[0] = said.x, s[1] = said.y, s[2] = said.z, s[3] = said.w;
                    }
                }
            }
        }
        if (!grad) return;
        __syncthreads();
        top = statistics.x, inverse = statistics.y, at_named = statistics.z, elsewhere = statistics.w;
        if (inverse == 0.0f) { /* the same in every block of the row */
            nothing();
            return;
        }
    }

    /* gradient: elsewhere * q everywhere, then the named entries once more with their own value */
    float g = (float)((double)weight * inv);
    if (BACKWARD && p.upstream) g *= p.upstream[row];
    const bool apart = inverse < 0.0f;
    const float factor = apart ? g * elsewhere : g * elsewhere * inverse, base = apart ? at_named : top;
    const Pair times(factor, factor), less(-base, -base), by(c, c);
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
        const float q = fabsf(inverse) * fast_exp2((named[j].z - top) * c);
        grad[at] = Elem<T>::down(g * (float)((apart ? fmax(named_p, 1.0) : (double)at_named) * q - sum));
    }
}

}  // namespace accb_rows
