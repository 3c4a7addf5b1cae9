// lfm_ops.hip -- the C ABI of include/lfm_ops.h: argument checks on the host, then the launchers of ops_common.hpp.
#include <math.h>

#include <algorithm>
#include <string>
#include <vector>

#include "ops_common.hpp"

using namespace lfm::ops;

static thread_local std::string g_ops_err;

static int refuse(int code, const char *msg)
{
    try {
        g_ops_err = msg;
    } catch (...) {  // no exception leaves a C entry point
    }
    return code;
}

static int finish(hipError_t e)
{
    if (e == hipSuccess) return LFM_OK;
    return refuse(e == hipErrorOutOfMemory ? LFM_ENOMEM : LFM_ENODEV, hipGetErrorString(e));
}

extern "C" const char *lfm_ops_last_error(void) { return g_ops_err.c_str(); }

static const int64_t MOST_ROWS = 2147483647;
static const int64_t MOST_SOFTMAX_ROWS = 1 << 27, MOST_SOFTMAX_ITEMS = 1 << 30;  // (launches stay below 2^32 threads)

static int check_type(int32_t dtype, int32_t id_bytes)
{
    if (dtype != LFM_F32 && dtype != LFM_BF16 && dtype != LFM_F16) return refuse(LFM_EINVAL, "dtype must be LFM_F32, LFM_BF16 or LFM_F16");
    if (id_bytes != 4 && id_bytes != 8) return refuse(LFM_EINVAL, "ids must be int32 or int64");
    return LFM_OK;
}

static int check_space(const void *ws, int64_t have, int64_t need)
{
    if (have < need || (need && !ws)) return refuse(LFM_EINVAL, "workspace is smaller than the call needs");
    if ((uintptr_t)ws & 255) return refuse(LFM_EINVAL, "workspace must be 256-byte aligned");
    return LFM_OK;
}

#define OPS_TRY(expr)                  \
    do {                               \
        const int rc_ = (expr);        \
        if (rc_ != LFM_OK) return rc_; \
    } while (0)

static int check_softmax_sizes(int64_t rows, int64_t vocab, int32_t d, int32_t dtype)
{
    OPS_TRY(check_type(dtype, 4));
    if (rows < 0 || rows > MOST_SOFTMAX_ROWS) return refuse(LFM_EINVAL, "rows out of range");
    if (vocab < 1 || vocab > MOST_SOFTMAX_ITEMS) return refuse(LFM_EINVAL, "the vocabulary is empty or too large");
    if (d < 1) return refuse(LFM_EINVAL, "d must be positive");
    if (d > LFM_MAX_COMPONENTS) return refuse(LFM_EUNSUPPORTED, "d is beyond LFM_MAX_COMPONENTS");
    return LFM_OK;
}

extern "C" int lfm_ops_softmax_workspace(int64_t rows, int64_t vocab, int32_t d, int32_t dtype, int32_t grad, int64_t *bytes)
{
    if (!bytes) return refuse(LFM_EINVAL, "null pointer");
    OPS_TRY(check_softmax_sizes(rows, vocab, d, dtype));
    *bytes = softmax_workspace(rows, vocab, d, dtype, grad != 0);
    return LFM_OK;
}

static int run_softmax(const lfm_softmax_args *a, bool grad, void *ws, int64_t ws_bytes, void *stream)
{
    if (!a) return refuse(LFM_EINVAL, "null arguments");
    OPS_TRY(check_softmax_sizes(a->rows, a->vocab, a->d, a->dtype));
    OPS_TRY(check_type(a->dtype, a->id_bytes));
    if (a->hidden_stride < a->d || a->table_stride < a->d) return refuse(LFM_EINVAL, "a row stride is smaller than d");
    if (!a->table || (a->rows && (!a->hidden || !a->targets || !a->loss || !a->lse))) return refuse(LFM_EINVAL, "null pointer");
    if (grad && (!a->d_table || (a->rows && !a->d_hidden))) return refuse(LFM_EINVAL, "null gradient pointer");
    OPS_TRY(check_space(ws, ws_bytes, softmax_workspace(a->rows, a->vocab, a->d, a->dtype, grad)));
    return finish(softmax_loss(*a, grad, ws, (hipStream_t)stream));
}

extern "C" int lfm_ops_softmax_loss(const lfm_softmax_args *args, void *ws, int64_t ws_bytes, void *stream)
{
    return run_softmax(args, false, ws, ws_bytes, stream);
}

extern "C" int lfm_ops_softmax_loss_grad(const lfm_softmax_args *args, void *ws, int64_t ws_bytes, void *stream)
{
    return run_softmax(args, true, ws, ws_bytes, stream);
}

static int check_lookup(const lfm_lookup_args *a)
{
    if (!a) return refuse(LFM_EINVAL, "null arguments");
    OPS_TRY(check_type(a->dtype, a->id_bytes));
    if (a->rows < 0 || a->rows > MOST_ROWS || a->nnz < 0 || a->nnz > MOST_ROWS - 4096) return refuse(LFM_EINVAL, "rows or ids out of range");
    if (a->vocab < 1 || a->vocab > MOST_ROWS) return refuse(LFM_EINVAL, "the vocabulary is empty or too large");
    if (a->d < 1 || a->d > 65536) return refuse(LFM_EINVAL, "d out of range");
    if (!a->indptr && a->nnz != a->rows) return refuse(LFM_EINVAL, "without indptr there is one id per row");
    if (!a->indptr && a->values) return refuse(LFM_EINVAL, "values need an indptr");
    if (a->indptr && !a->rows && a->nnz) return refuse(LFM_EINVAL, "ids without a row");
    if (a->nnz && !a->ids) return refuse(LFM_EINVAL, "null ids");
    return LFM_OK;
}

extern "C" int lfm_ops_embedding_lookup(const lfm_lookup_args *a, void *stream)
{
    OPS_TRY(check_lookup(a));
    if (a->table_stride < a->d) return refuse(LFM_EINVAL, "a row stride is smaller than d");
    if (!a->table || (a->rows && !a->out)) return refuse(LFM_EINVAL, "null pointer");
    return finish(embedding_lookup(*a, (hipStream_t)stream));
}

extern "C" int lfm_ops_embedding_grad_workspace(int64_t rows, int64_t vocab, int64_t nnz, int32_t d, int32_t bags, int64_t *bytes)
{
    if (!bytes) return refuse(LFM_EINVAL, "null pointer");
    if (rows < 0 || rows > MOST_ROWS || nnz < 0 || nnz > MOST_ROWS - 4096 || vocab < 1 || vocab > MOST_ROWS || d < 1 || d > 65536)
        return refuse(LFM_EINVAL, "sizes out of range");
    *bytes = embedding_grad_workspace(rows, vocab, nnz, d, bags != 0);
    return LFM_OK;
}

extern "C" int lfm_ops_embedding_lookup_grad(const lfm_lookup_args *a, void *ws, int64_t ws_bytes, void *stream)
{
    OPS_TRY(check_lookup(a));
    if (a->d_out_stride < a->d) return refuse(LFM_EINVAL, "a row stride is smaller than d");
    if (!a->out || (a->rows && !a->d_out)) return refuse(LFM_EINVAL, "null pointer");
    if ((uintptr_t)a->out & 15) return refuse(LFM_EINVAL, "the gradient must be 16-byte aligned");
    OPS_TRY(check_space(ws, ws_bytes, embedding_grad_workspace(a->rows, a->vocab, a->nnz, a->d, a->indptr != nullptr)));
    return finish(embedding_grad(*a, ws, (hipStream_t)stream));
}

static int check_clip(int64_t n, const int64_t *counts)
{
    if (n < 0 || n > (1 << 20) || (n && !counts)) return refuse(LFM_EINVAL, "number of tensors out of range");
    for (int64_t i = 0; i < n; ++i)
        if (counts[i] < 0 || counts[i] > (int64_t)1 << 36) return refuse(LFM_EINVAL, "a tensor's size is out of range");
    return LFM_OK;
}

// Tensors are read and written at the same time by many blocks: an output may be its own input and nothing else.
static int check_overlap(int64_t n, const void *const *x, void *const *out, const int64_t *counts, const int32_t *dtypes)
{
    struct Span {
        uintptr_t begin, end;
        bool written;
    };
    try {
        std::vector<Span> spans;
        spans.reserve((size_t)n * 2);
        for (int64_t i = 0; i < n; ++i) {
            if (!counts[i]) continue;
            const uintptr_t bytes = (uintptr_t)counts[i] * (uintptr_t)dtype_bytes(dtypes[i]), to = (uintptr_t)out[i], from = (uintptr_t)x[i];
            spans.push_back({to, to + bytes, true});
            if (from != to) spans.push_back({from, from + bytes, false});
        }
        std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.begin < b.begin; });
        uintptr_t any = 0, written = 0;  // where the spans so far end
        for (const Span &s : spans) {
            if (s.begin < written || (s.written && s.begin < any)) return refuse(LFM_EINVAL, "a tensor that is written overlaps another one");
            any = std::max(any, s.end);
            if (s.written) written = std::max(written, s.end);
        }
    } catch (...) {
        return refuse(LFM_ENOMEM, "out of host memory");
    }
    return LFM_OK;
}

extern "C" int lfm_ops_clip_workspace(int64_t n_tensors, const int64_t *counts, int64_t *bytes)
{
    if (!bytes) return refuse(LFM_EINVAL, "null pointer");
    OPS_TRY(check_clip(n_tensors, counts));
    *bytes = clip_workspace(n_tensors, counts);
    return LFM_OK;
}

extern "C" int lfm_ops_clip_global_norm(int64_t n_tensors, const void *const *x, void *const *out, const int64_t *counts,
                                        const int32_t *dtypes, double max_norm, float *norm, void *ws, int64_t ws_bytes,
                                        void *stream)
{
    OPS_TRY(check_clip(n_tensors, counts));
    if (!norm || (n_tensors && (!x || !dtypes))) return refuse(LFM_EINVAL, "null pointer");
    if (out && !(max_norm >= 0.0)) return refuse(LFM_EINVAL, "max_norm must not be negative");
    for (int64_t i = 0; i < n_tensors; ++i) {
        OPS_TRY(check_type(dtypes[i], 4));
        if (counts[i] && (!x[i] || (out && !out[i]))) return refuse(LFM_EINVAL, "null tensor");
    }
    if (out) OPS_TRY(check_overlap(n_tensors, x, out, counts, dtypes));
    OPS_TRY(check_space(ws, ws_bytes, clip_workspace(n_tensors, counts)));
    return finish(clip_global_norm(n_tensors, x, out, counts, dtypes, max_norm, norm, ws, (hipStream_t)stream));
}
