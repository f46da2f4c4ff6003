// extern "C" entry points declared in include/ntops.h: argument validation on the host, then the launches on the caller's
// stream.  Nothing here allocates, frees or synchronises.
#include "ops_common.h"

namespace ntfp8 {

int64_t layer_norm_most_cols(int dtype);
int layer_norm_blocks(int dtype, int64_t rows, int64_t cols);
int run_layer_norm_forward(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride, const void* weight, const void* bias,
                           int w_dtype, float eps, void* y, float* mean, float* rstd, hipStream_t st);
int run_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride,
                            const void* weight, int w_dtype, const float* mean, const float* rstd, void* dx, void* dweight, void* dbias,
                            float* scratch, hipStream_t st);
bool adamw_within_reach(const ntops_adamw_tensor* tensors, int count);
int run_adamw(const ntops_adamw_tensor* tensors, int count, const ntops_adamw_options& o, hipStream_t st);
int run_adamw_unpack(const void* codes, const float* scale, int64_t n, float* out, hipStream_t st);
int64_t head_piece(int64_t vocab);
int64_t head_workspace(const ntops_linear_cross_entropy_desc& d);
int run_head(const ntops_linear_cross_entropy_desc& d, hipStream_t st);
int run_scale(const ntops_scale_tensor* t, int count, int x_dtype, const float* factor, int out_dtype, hipStream_t st);

namespace {

constexpr int64_t kMostElements = (int64_t)1 << 46;

bool dtype_ok(int d) { return d == NTFP8_F32 || d == NTFP8_F16 || d == NTFP8_BF16; }
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
bool overlap(const void* a, int64_t an, const void* b, int64_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + (uintptr_t)bn && y < x + (uintptr_t)an;
}
// bytes from the first element of `rows` rows to the last, `stride` elements apart
int64_t span(int64_t rows, int64_t cols, int64_t stride, int dtype) { return ((rows - 1) * stride + cols) * size_of(dtype); }
bool rows_ok(int64_t rows, int64_t cols, int64_t stride) {
    return rows > 0 && cols > 0 && rows <= 0x7fffffff && stride >= cols && stride <= kMostElements / rows;
}

int check_norm(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride, int w_dtype) {
    if (!x) return NTFP8_ERR_NULL;
    if (!dtype_ok(x_dtype) || (w_dtype != NTFP8_F32 && w_dtype != x_dtype)) return NTFP8_ERR_ENUM;
    if (!rows_ok(rows, cols, x_stride)) return NTFP8_ERR_SIZE;
    if (cols > layer_norm_most_cols(x_dtype)) return NTFP8_ERR_UNSUPPORTED;
    return aligned(x, size_of(x_dtype)) ? NTFP8_OK : NTFP8_ERR_ALIGN;
}

int check_head(const ntops_linear_cross_entropy_desc& d) {
    // sizes first: the workspace depends on them alone
    if (d.x_dtype != NTFP8_BF16 && d.x_dtype != NTFP8_F16) return NTFP8_ERR_ENUM;
    constexpr int64_t kMost = (int64_t)1 << 22;   // (and so in head.hip)
    if (d.tokens <= 0 || d.hidden <= 0 || d.vocab <= 0 || d.tokens > ((int64_t)1 << 30) || d.hidden > kMost || d.vocab > kMost) return NTFP8_ERR_SIZE;
    if (!rows_ok(d.tokens, d.hidden, d.x_stride) || !rows_ok(d.vocab, d.hidden, d.weight_stride)) return NTFP8_ERR_SIZE;
    if ((d.dx || d.dweight) && d.grad_dtype != d.x_dtype && d.grad_dtype != NTFP8_F32) return NTFP8_ERR_ENUM;
    return NTFP8_OK;
}

}  // namespace
}  // namespace ntfp8

using namespace ntfp8;

extern "C" {

int ntops_layer_norm_forward(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride, const void* weight,
                             const void* bias, int w_dtype, float eps, void* y, float* mean, float* rstd, void* stream) {
    if (!y || (mean == nullptr) != (rstd == nullptr)) return NTFP8_ERR_NULL;
    if (const int rc = check_norm(x, x_dtype, rows, cols, x_stride, w_dtype)) return rc;
    if (!aligned(weight, size_of(w_dtype)) || !aligned(bias, size_of(w_dtype)) || !aligned(y, size_of(x_dtype)) || !aligned(mean, 4) || !aligned(rstd, 4))
        return NTFP8_ERR_ALIGN;
    const int64_t yb = rows * cols * size_of(x_dtype), wb = cols * size_of(w_dtype);
    if (overlap(x, span(rows, cols, x_stride, x_dtype), y, yb) || overlap(weight, wb, y, yb) || overlap(bias, wb, y, yb)) return NTFP8_ERR_ALIAS;
    return run_layer_norm_forward(x, x_dtype, rows, cols, x_stride, weight, bias, w_dtype, eps, y, mean, rstd, static_cast<hipStream_t>(stream));
}

int64_t ntops_layer_norm_scratch(int x_dtype, int64_t rows, int64_t cols) {
    if (!dtype_ok(x_dtype) || rows <= 0 || cols <= 0 || cols > layer_norm_most_cols(x_dtype)) return 0;
    return (int64_t)layer_norm_blocks(x_dtype, rows, cols) * 2 * cols * 4;
}

int ntops_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride,
                              const void* weight, int w_dtype, const float* mean, const float* rstd, void* dx, void* dweight,
                              void* dbias, void* scratch, void* stream) {
    if (!dy || !mean || !rstd || (!dx && !dweight && !dbias) || ((dweight || dbias) && !scratch)) return NTFP8_ERR_NULL;
    if (const int rc = check_norm(x, x_dtype, rows, cols, x_stride, w_dtype)) return rc;
    if (!rows_ok(rows, cols, dy_stride)) return NTFP8_ERR_SIZE;
    const size_t xs = size_of(x_dtype), wsz = size_of(w_dtype);
    if (!aligned(dy, xs) || !aligned(weight, wsz) || !aligned(dx, xs) || !aligned(dweight, wsz) || !aligned(dbias, wsz) || !aligned(mean, 4) ||
        !aligned(rstd, 4) || !aligned(scratch, 16))
        return NTFP8_ERR_ALIGN;
    const int64_t db = rows * cols * (int64_t)xs;
    if (overlap(x, span(rows, cols, x_stride, x_dtype), dx, db) || overlap(dy, span(rows, cols, dy_stride, x_dtype), dx, db)) return NTFP8_ERR_ALIAS;
    return run_layer_norm_backward(dy, dy_stride, x, x_dtype, rows, cols, x_stride, weight, w_dtype, mean, rstd, dx, dweight, dbias,
                                   static_cast<float*>(scratch), static_cast<hipStream_t>(stream));
}

int ntops_adamw_check(const ntops_adamw_tensor* tensors, int count, const ntops_adamw_options* options) {
    if (!options || (count > 0 && !tensors)) return NTFP8_ERR_NULL;
    const ntops_adamw_options& o = *options;
    if (count < 0 || o.step < 1) return NTFP8_ERR_SIZE;
    if (!dtype_ok(o.param_dtype) || !dtype_ok(o.grad_dtype) || (o.bits != 8 && o.bits != 32)) return NTFP8_ERR_ENUM;
    if (!(o.beta1 >= 0.0 && o.beta1 < 1.0) || !(o.beta2 >= 0.0 && o.beta2 < 1.0) || !(o.eps >= 0.0) || !(o.lr == o.lr) || !(o.weight_decay == o.weight_decay))
        return NTFP8_ERR_UNSUPPORTED;
    if (!aligned(o.grad_scale, 4)) return NTFP8_ERR_ALIGN;
    for (int i = 0; i < count; ++i) {
        const ntops_adamw_tensor& t = tensors[i];
        if (t.n < 0 || t.n > kMostElements) return NTFP8_ERR_SIZE;
        if (t.n == 0) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (o.bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale))) return NTFP8_ERR_NULL;
        if (t.copy && !dtype_ok(o.copy_dtype)) return NTFP8_ERR_ENUM;
        const size_t ss = o.bits == 8 ? 1 : 4;
        if (!aligned(t.param, size_of(o.param_dtype)) || !aligned(t.grad, size_of(o.grad_dtype)) || !aligned(t.exp_avg, ss) || !aligned(t.exp_avg_sq, ss) ||
            (t.copy && !aligned(t.copy, size_of(o.copy_dtype))) || !aligned(t.exp_avg_scale, 4) || !aligned(t.exp_avg_sq_scale, 4))
            return NTFP8_ERR_ALIGN;
        const int64_t pb = t.n * size_of(o.param_dtype), gb = t.n * size_of(o.grad_dtype), sb = t.n * (int64_t)ss, cb = t.n * size_of(o.copy_dtype);
        if (overlap(t.param, pb, t.grad, gb) || overlap(t.param, pb, t.exp_avg, sb) || overlap(t.param, pb, t.exp_avg_sq, sb) ||
            overlap(t.exp_avg, sb, t.exp_avg_sq, sb) || overlap(t.grad, gb, t.exp_avg, sb) || overlap(t.grad, gb, t.exp_avg_sq, sb) ||
            overlap(t.copy, cb, t.param, pb) || overlap(t.copy, cb, t.grad, gb) || overlap(t.copy, cb, t.exp_avg, sb) || overlap(t.copy, cb, t.exp_avg_sq, sb))
            return NTFP8_ERR_ALIAS;
    }
    return adamw_within_reach(tensors, count) ? NTFP8_OK : NTFP8_ERR_UNSUPPORTED;
}

int ntops_adamw(const ntops_adamw_tensor* tensors, int count, const ntops_adamw_options* options, void* stream) {
    if (const int rc = ntops_adamw_check(tensors, count, options)) return rc;
    return run_adamw(tensors, count, *options, static_cast<hipStream_t>(stream));
}

int ntops_adamw_unpack(const void* codes, const float* scale, int64_t n, float* out, void* stream) {
    if (!codes || !scale || !out) return NTFP8_ERR_NULL;
    if (n <= 0 || n > kMostElements) return NTFP8_ERR_SIZE;
    if (!aligned(scale, 4) || !aligned(out, 4)) return NTFP8_ERR_ALIGN;
    if (overlap(codes, n, out, 4 * n)) return NTFP8_ERR_ALIAS;
    return run_adamw_unpack(codes, scale, n, out, static_cast<hipStream_t>(stream));
}

int64_t ntops_linear_cross_entropy_piece(int64_t vocab) { return vocab > 0 && vocab <= ((int64_t)1 << 22) ? head_piece(vocab) : 0; }

int64_t ntops_linear_cross_entropy_workspace(const ntops_linear_cross_entropy_desc* d) {
    return d && check_head(*d) == NTFP8_OK ? head_workspace(*d) : 0;
}

int ntops_linear_cross_entropy(const ntops_linear_cross_entropy_desc* d, void* stream) {
    if (!d || !d->x || !d->weight || !d->labels || !d->losses || !d->workspace) return NTFP8_ERR_NULL;
    if (const int rc = check_head(*d)) return rc;
    if (d->dweight && d->grad_dtype != NTFP8_F32 && d->tokens > head_piece(d->vocab)) return NTFP8_ERR_UNSUPPORTED;
    if (!aligned(d->x, 2) || !aligned(d->weight, 2) || !aligned(d->labels, 8) || !aligned(d->losses, 4) || !aligned(d->loss, 4) || !aligned(d->dx, 16) ||
        !aligned(d->dweight, 16) || !aligned(d->workspace, 256))
        return NTFP8_ERR_ALIGN;
    struct Range {
        const void* p;
        int64_t bytes;
    };
    const int64_t gs = size_of(d->grad_dtype == NTFP8_F32 ? NTFP8_F32 : d->x_dtype);
    const Range in[] = {{d->x, span(d->tokens, d->hidden, d->x_stride, d->x_dtype)}, {d->weight, span(d->vocab, d->hidden, d->weight_stride, d->x_dtype)}, {d->labels, 8 * d->tokens}};
    const Range out[] = {{d->losses, 4 * d->tokens}, {d->loss, 4}, {d->dx, d->tokens * d->hidden * gs}, {d->dweight, d->vocab * d->hidden * gs}, {d->workspace, head_workspace(*d)}};
    for (int i = 0; i < 5; ++i) {
        for (const Range& r : in)
            if (overlap(r.p, r.bytes, out[i].p, out[i].bytes)) return NTFP8_ERR_ALIAS;
        for (int j = 0; j < i; ++j)
            if (overlap(out[j].p, out[j].bytes, out[i].p, out[i].bytes)) return NTFP8_ERR_ALIAS;
    }
    return run_head(*d, static_cast<hipStream_t>(stream));
}

int ntops_scale(const ntops_scale_tensor* tensors, int count, int x_dtype, const float* factor, int out_dtype, void* stream) {
    if (!factor || (count > 0 && !tensors)) return NTFP8_ERR_NULL;
    if (!dtype_ok(x_dtype) || !dtype_ok(out_dtype)) return NTFP8_ERR_ENUM;
    if (count < 0) return NTFP8_ERR_SIZE;
    if (!aligned(factor, 4)) return NTFP8_ERR_ALIGN;
    for (int i = 0; i < count; ++i) {
        const ntops_scale_tensor& t = tensors[i];
        if (!t.x || !t.out) return NTFP8_ERR_NULL;
        if (t.n <= 0 || t.n > kMostElements) return NTFP8_ERR_SIZE;
        if (!aligned(t.x, size_of(x_dtype)) || !aligned(t.out, size_of(out_dtype))) return NTFP8_ERR_ALIGN;
        if ((t.x != t.out || x_dtype != out_dtype) && overlap(t.x, t.n * size_of(x_dtype), t.out, t.n * size_of(out_dtype))) return NTFP8_ERR_ALIAS;
    }
    return run_scale(tensors, count, x_dtype, factor, out_dtype, static_cast<hipStream_t>(stream));
}

}  // extern "C"
