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
int64_t rms_norm_most_cols(int dtype);
int rms_norm_blocks(int dtype, int64_t rows, int64_t cols, bool full);
int run_rms_norm_forward(const ntops_rms_norm_desc& d, hipStream_t st);
int run_rms_norm_backward(const ntops_rms_norm_desc& d, const ntops_rms_norm_grads& g, hipStream_t st);
int run_rotary(const ntops_rotary_desc& d, hipStream_t st);
bool attention_fits(const ntops_attention_desc& d);
int64_t attention_workspace(const ntops_attention_desc& d, bool backward);
int64_t attention_plan(const ntops_attention_desc& d);
int run_attention_forward(const ntops_attention_desc& d, hipStream_t st);
int run_attention_backward(const ntops_attention_desc& d, hipStream_t st);
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

struct Range {
    const void* p;
    int64_t bytes;
};
// whether an output lies over an input, or over another output
template <size_t I, size_t O>
bool collide(const Range (&in)[I], const Range (&out)[O]) {
    for (size_t i = 0; i < O; ++i) {
        for (const Range& r : in)
            if (overlap(r.p, r.bytes, out[i].p, out[i].bytes)) return true;
        for (size_t j = 0; j < i; ++j)
            if (overlap(out[j].p, out[j].bytes, out[i].p, out[i].bytes)) return true;
    }
    return false;
}

int check_rms_norm(const ntops_rms_norm_desc& d) {
    if (!dtype_ok(d.x_dtype) || (d.residual_dtype != NTFP8_F32 && d.residual_dtype != d.x_dtype) || (d.w_dtype != NTFP8_F32 && d.w_dtype != d.x_dtype) ||
        d.gate_kind < NTOPS_GATE_NONE || d.gate_kind > NTOPS_GATE_ELEMENT)
        return NTFP8_ERR_ENUM;
    if (!rows_ok(d.rows, d.cols, d.x_stride) || (d.residual && !rows_ok(d.rows, d.cols, d.residual_stride)) ||
        (d.gate_kind == NTOPS_GATE_ELEMENT && !rows_ok(d.rows, d.cols, d.gate_stride)))
        return NTFP8_ERR_SIZE;
    if (d.cols > rms_norm_most_cols(d.x_dtype) || !(d.eps >= 0.0f) || !(d.residual_scale == d.residual_scale)) return NTFP8_ERR_UNSUPPORTED;
    if (d.gate_kind != NTOPS_GATE_NONE && !d.gate) return NTFP8_ERR_NULL;
    const size_t xs = size_of(d.x_dtype), rs = size_of(d.residual_dtype), ws = size_of(d.w_dtype);
    if (!aligned(d.x, xs) || !aligned(d.residual, rs) || !aligned(d.gate, d.gate_kind == NTOPS_GATE_ELEMENT ? xs : ws) || !aligned(d.weight, ws) ||
        !aligned(d.post_weight, ws) || !aligned(d.y, xs) || !aligned(d.h, rs) || !aligned(d.first, 4) || !aligned(d.second, 4))
        return NTFP8_ERR_ALIGN;
    return NTFP8_OK;
}

// elements between a tensor's first and behind its last
int64_t reach(int64_t rows, int64_t stride, int64_t heads, int64_t head, int64_t dim) { return (rows - 1) * stride + (heads - 1) * head + dim; }

int check_rotary(const ntops_rotary_desc& d) {
    if (!dtype_ok(d.dtype) || (d.position_bits != 32 && d.position_bits != 64)) return NTFP8_ERR_ENUM;
    if (d.heads < 0 || d.kv_heads < 0 || (d.heads > 0 && (!d.q || !d.q_out)) || (d.kv_heads > 0 && (!d.k || !d.k_out)) || !d.positions || !d.frequencies) return NTFP8_ERR_NULL;
    const int64_t heads = (int64_t)d.heads + d.kv_heads;
    if (d.tokens <= 0 || d.tokens > 0x7fffffff || heads < 1 || heads > 16384 || d.head_dim < 1 || d.pairs < 1 || d.pairs > d.head_dim / 2 || d.position_count < 1) return NTFP8_ERR_SIZE;
    constexpr int64_t kMost = (int64_t)1 << 31;   // elements from token to token and from head to head
    for (const int64_t v : {d.q_stride, d.q_head, d.k_stride, d.k_head})
        if (v < 0 || v > kMost) return NTFP8_ERR_SIZE;
    if ((d.heads && d.q_stride > kMostElements / d.tokens) || (d.kv_heads && d.k_stride > kMostElements / d.tokens)) return NTFP8_ERR_SIZE;
    if (d.head_dim > 2048 || !(d.scale == d.scale)) return NTFP8_ERR_UNSUPPORTED;
    const size_t s = size_of(d.dtype);
    if (!aligned(d.q, s) || !aligned(d.k, s) || !aligned(d.q_out, s) || !aligned(d.k_out, s) || !aligned(d.positions, d.position_bits / 8) || !aligned(d.frequencies, 8))
        return NTFP8_ERR_ALIGN;
    const int64_t b = (int64_t)s;
    const Range in[] = {{d.heads ? d.q : nullptr, reach(d.tokens, d.q_stride, d.heads, d.q_head, d.head_dim) * b},
                        {d.kv_heads ? d.k : nullptr, reach(d.tokens, d.k_stride, d.kv_heads, d.k_head, d.head_dim) * b},
                        {d.positions, std::min(d.position_count, d.tokens) * d.position_bits / 8},
                        {d.frequencies, 8 * (int64_t)d.pairs}};
    const Range out[] = {{d.heads ? d.q_out : nullptr, d.tokens * d.heads * d.head_dim * b}, {d.kv_heads ? d.k_out : nullptr, d.tokens * d.kv_heads * d.head_dim * b}};
    return collide(in, out) ? NTFP8_ERR_ALIAS : NTFP8_OK;
}

int check_attention_sizes(const ntops_attention_desc& d) {
    if (d.dtype != NTFP8_BF16 && d.dtype != NTFP8_F16) return NTFP8_ERR_ENUM;
    constexpr int64_t kMost = (int64_t)1 << 27;
    if (d.heads < 1 || d.kv_heads < 1 || d.heads % d.kv_heads != 0 || d.head_dim < 8 || d.sequences < 1 || d.sequences > kMost || d.q_rows < 1 || d.k_rows < 0 ||
        d.q_rows > kMost / d.heads || d.k_rows > kMost / d.kv_heads)
        return NTFP8_ERR_SIZE;
    if ((d.cu_q == nullptr) != (d.cu_k == nullptr)) return NTFP8_ERR_NULL;
    if (!d.cu_q && (d.q_rows % d.sequences != 0 || d.k_rows % d.sequences != 0)) return NTFP8_ERR_SIZE;
    if (d.head_dim > 128 || d.head_dim % 8 != 0) return NTFP8_ERR_UNSUPPORTED;
    return attention_fits(d) ? NTFP8_OK : NTFP8_ERR_SIZE;
}

int check_attention(const ntops_attention_desc& d) {
    if (const int rc = check_attention_sizes(d)) return rc;
    if (!d.q || (d.k_rows > 0 && (!d.k || !d.v)) || !d.out || !d.workspace) return NTFP8_ERR_NULL;
    if (!(d.scale >= 1e-30f) || d.scale > 1e30f) return NTFP8_ERR_UNSUPPORTED;
    // (64 rows of a tile lie within 2^31 bytes)
    for (const int64_t v : {d.q_stride, d.k_stride, d.v_stride, d.do_stride})
        if (v < 0 || v > ((int64_t)1 << 24) || v % 8 != 0) return NTFP8_ERR_SIZE;
    for (const int64_t v : {d.q_head, d.k_head, d.v_head, d.do_head, d.q_batch, d.k_batch, d.v_batch, d.do_batch})
        if (v < 0 || v > kMostElements || v % 8 != 0) return NTFP8_ERR_SIZE;
    // (where they are used, all heads and sequences together lie within that too)
    const int64_t most = kMostElements / d.heads, most_kv = kMostElements / d.kv_heads, most_batch = d.cu_q ? kMostElements : kMostElements / d.sequences;
    if (d.q_head > most || d.k_head > most_kv || d.v_head > most_kv || (d.dout && d.do_head > most) || d.q_batch > most_batch || d.k_batch > most_batch || d.v_batch > most_batch ||
        (d.dout && d.do_batch > most_batch))
        return NTFP8_ERR_SIZE;
    for (const void* p : {d.q, d.k, d.v, d.dout, (const void*)d.out, (const void*)d.dq, (const void*)d.dk, (const void*)d.dv})
        if (!aligned(p, 16)) return NTFP8_ERR_ALIGN;
    return aligned(d.lse, 4) && aligned(d.cu_q, 4) && aligned(d.cu_k, 4) && aligned(d.workspace, 256) && aligned(d.plan, 256) && aligned(d.out_low, 8) ? NTFP8_OK : NTFP8_ERR_ALIGN;
}
// bytes of a tensor of a call, from its first element on
int64_t attention_reach(const ntops_attention_desc& d, int64_t rows, int64_t heads, int64_t stride, int64_t head, int64_t batch) {
    if (rows == 0) return 0;
    const int64_t each = d.cu_q ? rows : rows / d.sequences;
    return 2 * (reach(each, stride, heads, head, d.head_dim) + (d.cu_q ? 0 : (d.sequences - 1) * batch));
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
    const int64_t gs = size_of(d->grad_dtype == NTFP8_F32 ? NTFP8_F32 : d->x_dtype);
    const Range in[] = {{d->x, span(d->tokens, d->hidden, d->x_stride, d->x_dtype)}, {d->weight, span(d->vocab, d->hidden, d->weight_stride, d->x_dtype)}, {d->labels, 8 * d->tokens}};
    const Range out[] = {{d->losses, 4 * d->tokens}, {d->loss, 4}, {d->dx, d->tokens * d->hidden * gs}, {d->dweight, d->vocab * d->hidden * gs}, {d->workspace, head_workspace(*d)}};
    if (collide(in, out)) return NTFP8_ERR_ALIAS;
    return run_head(*d, static_cast<hipStream_t>(stream));
}

int ntops_rms_norm_forward(const ntops_rms_norm_desc* d, void* stream) {
    if (!d || !d->x || !d->y || (d->residual == nullptr) != (d->h == nullptr)) return NTFP8_ERR_NULL;
    if (d->residual ? (d->second == nullptr && d->first != nullptr) : (d->post_weight || d->gate_kind != NTOPS_GATE_NONE)) return NTFP8_ERR_NULL;
    if (d->second && d->post_weight && !d->first) return NTFP8_ERR_NULL;
    if (const int rc = check_rms_norm(*d)) return rc;
    if (!d->residual && d->residual_dtype != d->x_dtype) return NTFP8_ERR_ENUM;
    const int64_t n = d->rows * d->cols, xs = size_of(d->x_dtype), rs = size_of(d->residual_dtype), wb = d->cols * size_of(d->w_dtype);
    const bool element = d->gate_kind == NTOPS_GATE_ELEMENT;
    const Range in[] = {{d->x, span(d->rows, d->cols, d->x_stride, d->x_dtype)},
                        {d->residual, span(d->rows, d->cols, d->residual_stride, d->residual_dtype)},
                        {d->gate_kind ? d->gate : nullptr, element ? span(d->rows, d->cols, d->gate_stride, d->x_dtype) : wb},
                        {d->weight, wb},
                        {d->post_weight, wb}};
    const Range out[] = {{d->y, n * xs}, {d->h, n * rs}, {d->first, 4 * d->rows}, {d->second, 4 * d->rows}};
    if (collide(in, out)) return NTFP8_ERR_ALIAS;
    return run_rms_norm_forward(*d, static_cast<hipStream_t>(stream));
}

int64_t ntops_rms_norm_scratch(const ntops_rms_norm_desc* d) {
    if (!d || check_rms_norm(*d) != NTFP8_OK) return 0;
    const bool full = d->post_weight || d->gate_kind;
    return (int64_t)rms_norm_blocks(d->x_dtype, d->rows, d->cols, full) * (full ? 3 : 1) * d->cols * 4;
}

int ntops_rms_norm_backward(const ntops_rms_norm_desc* d, const ntops_rms_norm_grads* g, void* stream) {
    if (!d || !g || !d->x || !d->second || (d->post_weight && !d->first) || (!g->dy && !g->dh)) return NTFP8_ERR_NULL;
    if (!d->h && (d->post_weight || d->gate_kind != NTOPS_GATE_NONE || g->dh || g->dresidual)) return NTFP8_ERR_NULL;
    if ((g->dweight && !d->weight) || (g->dpost_weight && !d->post_weight) || (g->dgate && d->gate_kind == NTOPS_GATE_NONE)) return NTFP8_ERR_NULL;
    if (!g->dx && !g->dresidual && !g->dgate && !g->dweight && !g->dpost_weight) return NTFP8_ERR_NULL;
    if ((g->dweight || g->dpost_weight || (g->dgate && d->gate_kind == NTOPS_GATE_CHANNEL)) && !g->scratch) return NTFP8_ERR_NULL;
    if (const int rc = check_rms_norm(*d)) return rc;
    if (!d->h && d->residual_dtype != d->x_dtype) return NTFP8_ERR_ENUM;
    if ((g->dy && !rows_ok(d->rows, d->cols, g->dy_stride)) || (g->dh && !rows_ok(d->rows, d->cols, g->dh_stride))) return NTFP8_ERR_SIZE;
    const bool element = d->gate_kind == NTOPS_GATE_ELEMENT;
    const size_t xs = size_of(d->x_dtype), rs = size_of(d->residual_dtype), ws = size_of(d->w_dtype);
    if (!aligned(g->dy, xs) || !aligned(g->dh, rs) || !aligned(g->dx, xs) || !aligned(g->dresidual, rs) || !aligned(g->dgate, element ? xs : ws) || !aligned(g->dweight, ws) ||
        !aligned(g->dpost_weight, ws) || !aligned(g->scratch, 16))
        return NTFP8_ERR_ALIGN;
    const int64_t n = d->rows * d->cols, wb = d->cols * (int64_t)ws;
    const Range in[] = {{d->x, span(d->rows, d->cols, d->x_stride, d->x_dtype)},
                        {d->h, n * (int64_t)rs},
                        {d->gate_kind ? d->gate : nullptr, element ? span(d->rows, d->cols, d->gate_stride, d->x_dtype) : wb},
                        {d->weight, wb},
                        {d->post_weight, wb},
                        {d->first, 4 * d->rows},
                        {d->second, 4 * d->rows},
                        {g->dy, span(d->rows, d->cols, g->dy_stride, d->x_dtype)},
                        {g->dh, span(d->rows, d->cols, g->dh_stride, d->residual_dtype)}};
    const Range out[] = {{g->dx, n * (int64_t)xs}, {g->dresidual, n * (int64_t)rs}, {g->dgate, element ? n * (int64_t)xs : wb}, {g->dweight, wb}, {g->dpost_weight, wb},
                         {g->scratch, g->scratch ? ntops_rms_norm_scratch(d) : 0}};
    if (collide(in, out)) return NTFP8_ERR_ALIAS;
    return run_rms_norm_backward(*d, *g, static_cast<hipStream_t>(stream));
}

int ntops_rotary(const ntops_rotary_desc* d, void* stream) {
    if (!d) return NTFP8_ERR_NULL;
    if (const int rc = check_rotary(*d)) return rc;
    return run_rotary(*d, static_cast<hipStream_t>(stream));
}

int64_t ntops_attention_workspace(const ntops_attention_desc* d, int backward) {
    return d && check_attention_sizes(*d) == NTFP8_OK ? std::max<int64_t>(256, attention_workspace(*d, backward != 0)) : 0;
}

int64_t ntops_attention_plan(const ntops_attention_desc* d) { return d && check_attention_sizes(*d) == NTFP8_OK ? attention_plan(*d) : 0; }

int ntops_attention_forward(const ntops_attention_desc* d, void* stream) {
    if (!d) return NTFP8_ERR_NULL;
    if (const int rc = check_attention(*d)) return rc;
    const int64_t cu = d->cu_q ? 4 * (d->sequences + 1) : 0;
    const Range in[] = {{d->q, attention_reach(*d, d->q_rows, d->heads, d->q_stride, d->q_head, d->q_batch)},
                        {d->k, attention_reach(*d, d->k_rows, d->kv_heads, d->k_stride, d->k_head, d->k_batch)},
                        {d->v, attention_reach(*d, d->k_rows, d->kv_heads, d->v_stride, d->v_head, d->v_batch)},
                        {d->cu_q, cu},
                        {d->cu_k, cu}};
    const Range out[] = {{d->out, 2 * d->q_rows * d->heads * d->head_dim}, {d->lse, 4 * d->q_rows * d->heads}, {d->workspace, attention_workspace(*d, false)},
                         {d->plan, attention_plan(*d)},
                         {d->out_low, d->q_rows * d->heads * d->head_dim}};
    if (collide(in, out)) return NTFP8_ERR_ALIAS;
    return run_attention_forward(*d, static_cast<hipStream_t>(stream));
}

int ntops_attention_backward(const ntops_attention_desc* d, void* stream) {
    if (!d || !d->dout || !d->lse || (!d->dq && !d->dk && !d->dv)) return NTFP8_ERR_NULL;
    if (const int rc = check_attention(*d)) return rc;
    const int64_t cu = d->cu_q ? 4 * (d->sequences + 1) : 0, qb = 2 * d->q_rows * d->heads * d->head_dim, kb = 2 * d->k_rows * d->kv_heads * d->head_dim;
    const Range in[] = {{d->q, attention_reach(*d, d->q_rows, d->heads, d->q_stride, d->q_head, d->q_batch)},
                        {d->k, attention_reach(*d, d->k_rows, d->kv_heads, d->k_stride, d->k_head, d->k_batch)},
                        {d->v, attention_reach(*d, d->k_rows, d->kv_heads, d->v_stride, d->v_head, d->v_batch)},
                        {d->dout, attention_reach(*d, d->q_rows, d->heads, d->do_stride, d->do_head, d->do_batch)},
                        {d->out, qb},
                        {d->lse, 4 * d->q_rows * d->heads},
                        {d->plan, attention_plan(*d)},
                        {d->out_low, d->q_rows * d->heads * d->head_dim},
                        {d->cu_q, cu},
                        {d->cu_k, cu}};
    const Range out[] = {{d->dq, qb}, {d->dk, kb}, {d->dv, kb}, {d->workspace, attention_workspace(*d, true)}};
    if (collide(in, out)) return NTFP8_ERR_ALIAS;
    return run_attention_backward(*d, static_cast<hipStream_t>(stream));
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
