/*
 * rows.cu -- operators over rows of scores: the best entries of a row (accb_top_rows), one index drawn from a row
 * (accb_sample_rows), and the divergence of a row from a teacher's best entries with its gradient (accb_distill_rows,
 * accb_distill_rows_backward).
 *
 * They stand beside the folds over rows (fold.cuh): a matrix comes in, every row is reduced.  rows.cuh says how a row
 * is held on chip.
 */
#include <algorithm>
#include <iterator>

#include "common.h"
#include "rows_distill.cuh"
#include "rows_sample.cuh"
#include "rows_top.cuh"

namespace accb_rows {

constexpr size_t kSharedMost = 192u << 10; /* dynamic shared memory a block may ask for (227 KB less what it declares) */
constexpr long long kShareBytes = 68 << 10; /* the share of a row that a block holds at most, if eight blocks do */

/* Blocks per row: as few as hold the row in shares of 68 KB, so that three blocks of an SM overlap one another's phases
 * (fewer and larger, or more and smaller, were slower: rows of 256 KB by 3, 4, 5 blocks 597, 522, 593 us for a training
 * step over 4096); more while rows are too few to give every SM two blocks, as long as a share stays worth a block. */
static int cluster_for(long long rows, long long row_bytes, int sm_count) {
    int size = (int)std::min<long long>(kMaxCluster, (row_bytes + kShareBytes - 1) / kShareBytes);
    while (size < kMaxCluster && rows * (size + 1) <= 2 * sm_count && row_bytes > (8 << 10) * size) ++size;
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

/* an array of elements of `bytes` bytes, or null */
static int check_aligned(accb_context *ctx, const void *ptr, size_t bytes, const char *what, const char *name) {
    return reinterpret_cast<uintptr_t>(ptr) % bytes ? fail(ctx, ACCB_EINVAL, "%s: misaligned pointer to %s", what, name) : ACCB_OK;
}

static RowsIn rows_in(const accb_rows_array *a) { return RowsIn{a->ptr, a->rows, a->pitch, a->cols}; }

/* Whether rows of two matrices of one shape and type share memory; the same memory row by row does not count, nor do
 * matrices side by side in the rows of a larger one. */
static bool overlap(const accb_rows_array *a, const accb_rows_array *b) {
    const long long bytes = (long long)size_of(a->type), row = a->cols * bytes;
    const uintptr_t p = reinterpret_cast<uintptr_t>(a->ptr), q = reinterpret_cast<uintptr_t>(b->ptr);
    const long long p_step = a->rows > 1 ? a->pitch * bytes : row, q_step = a->rows > 1 ? b->pitch * bytes : row;
    if (p + (a->rows - 1) * p_step + row <= q || q + (a->rows - 1) * q_step + row <= p) return false;
    if (p_step != q_step) return true;
    if (p == q) return false;
    const long long apart = (long long)((p < q ? q - p : p - q) % (uintptr_t)p_step);
    return apart < row || p_step - apart < row;
}

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
        auto known = std::find_if(std::begin(ctx->rows_clusters), std::end(ctx->rows_clusters), [&](const accb_context::RowsClusters &c) {
            return c.kernel == (const void *)kernel && c.size == size && c.smem == smem;
        });
        if (known == std::end(ctx->rows_clusters)) {
            int most = 0;
            const int st = check_cuda(ctx, cudaOccupancyMaxActiveClusters(&most, (const void *)kernel, &cfg), name);
            if (st != ACCB_OK) return st;
            known = ctx->rows_clusters + ctx->rows_clusters_next;
            ctx->rows_clusters_next = (ctx->rows_clusters_next + 1) % (int)std::size(ctx->rows_clusters);
            *known = {(const void *)kernel, size, smem, std::max(1, most)};
        }
        clusters = std::min<long long>(clusters, known->most);
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
    TRY(check_aligned(ctx, values, size_of(x->type), "top_rows", "values"));
    TRY(check_aligned(ctx, index, 4, "top_rows", "index"));
    TRY(check_aligned(ctx, lse, 4, "top_rows", "lse"));
    int room = 256;
    while (room < 2 * k) room *= 2;
    const TopParams p{rows_in(x), values, index, lse, temperature, k, room};
    const int size = cluster_for(x->rows, (long long)x->cols * size_of(x->type), ctx->sm_count);
    const size_t fixed = (room + own_places(room, size)) * sizeof(u64);
#define CALL(T) launch_rows(ctx, top_rows<T, true>, top_rows<T, false>, p, x, size, fixed, true, (cudaStream_t)stream, "top_rows")
    return BY_TYPE(x->type, CALL);
#undef CALL
}

int accb_sample_rows(accb_context *ctx, accb_stream stream, const accb_rows_array *x, const uint32_t *allowed, long long allowed_pitch,
                     const float *uniform, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                     int32_t *token, float *logprob) {
    LOCK(ctx);
    TRY(check_rows(ctx, x, "sample_rows"));
    if (allowed && (allowed_pitch < (x->cols + 31) / 32 || allowed_pitch > (1LL << 60) / std::max(1LL, x->rows)))
        return fail(ctx, ACCB_EINVAL, "sample_rows: %lld words of allowed bits for rows of %d entries", allowed_pitch, x->cols);
    if (x->rows == 0) return ACCB_OK;
    if (!uniform || !token) return fail(ctx, ACCB_EINVAL, "sample_rows: null random numbers or result");
    const void *const arrays[] = {allowed, uniform, temperature, top_k, top_p, min_p, token, logprob};
    const char *const names[] = {"allowed", "uniform", "temperature", "top_k", "top_p", "min_p", "token", "logprob"};
    for (int i = 0; i < 8; ++i) TRY(check_aligned(ctx, arrays[i], 4, "sample_rows", names[i]));
    const SampleParams p{rows_in(x), allowed, allowed_pitch, uniform, temperature, top_p, min_p, top_k, token, logprob};
    const int size = cluster_for(x->rows, (long long)x->cols * size_of(x->type), ctx->sm_count);
#define CALL(T)                                                                                                                            \
    (top_k || top_p ? launch_rows(ctx, sample_rows<T, true, true>, sample_rows<T, false, true>, p, x, size, 0, true, (cudaStream_t)stream, "sample_rows") \
                    : launch_rows(ctx, sample_rows<T, true, false>, sample_rows<T, false, false>, p, x, size, 0, true, (cudaStream_t)stream, "sample_rows"))
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
    const void *const arrays[] = {p.index, p.teacher_lse, p.weight, p.upstream, p.loss, p.stats};
    const char *const names[] = {"index", "teacher_lse", "weight", "upstream", "loss", "stats"};
    for (int i = 0; i < 6; ++i) TRY(check_aligned(ctx, arrays[i], 4, what, names[i]));
    TRY(check_aligned(ctx, p.teacher, size_of(p.teacher_type), what, "teacher"));
    if (grad && overlap(student, grad)) return fail(ctx, ACCB_EINVAL, "%s: the gradient overlaps the scores and is not in their place", what);
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
