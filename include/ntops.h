/* ntops — C ABI of the operators that stand beside the FP8 linears in a training step (MI355X, gfx950): layer
 * normalisation, the vocabulary projection with its softmax cross entropy, and AdamW over many tensors.  They live in the
 * same library as the entry points of ntfp8.h and follow its conventions: device pointers owned by the caller, nothing
 * allocated, freed or synchronised, argument errors returned as NTFP8_ERR_* before anything is launched, element types
 * NTFP8_F32 / NTFP8_F16 / NTFP8_BF16, `stream` a hipStream_t.  Row strides are in elements. */
#ifndef NTOPS_H
#define NTOPS_H

#include "ntfp8.h"

#ifdef __cplusplus
extern "C" {
#endif

/* y = (x - mean) * rstd * weight + bias over the last dimension of x [rows, cols] (rows `x_stride` elements apart; y is
 * dense), rstd = 1 / sqrt(var + eps), all in fp32 with one rounding to the type of x.  weight and bias [cols] of type
 * w_dtype (fp32, or the type of x) may each be NULL; mean and rstd [rows] fp32 may both be NULL (no backward pass follows).
 * cols <= 16384 for fp32 x, 32768 for 16-bit x (NTFP8_ERR_UNSUPPORTED beyond). */
int ntops_layer_norm_forward(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride, const void* weight,
                             const void* bias, int w_dtype, float eps, void* y, float* mean, float* rstd, void* stream);

/* Gradients of the above from dy [rows, cols] (rows dy_stride apart, type of x).  dx (dense, type of x), dweight and dbias
 * (type w_dtype) may each be NULL; the sums over rows are made in fp32 within a workgroup and in 64 bits over them,
 * in an order that depends on the sizes alone.
 * `scratch`: ntops_layer_norm_scratch(...) bytes, 16-byte aligned; may be NULL where neither dweight nor dbias is asked for. */
int64_t ntops_layer_norm_scratch(int x_dtype, int64_t rows, int64_t cols);
int ntops_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride,
                              const void* weight, int w_dtype, const float* mean, const float* rstd, void* dx, void* dweight,
                              void* dbias, void* scratch, void* stream);

/* One AdamW step over `count` tensors, all of one set of types:
 *   g = grad * *grad_scale;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2;
 *   param = param (1 - lr weight_decay) - lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 * in fp32, every operation rounded by itself; the new value is rounded once to the type of param, and, by itself, to copy_dtype
 * into `copy` where one is given.  bits 32: exp_avg and exp_avg_sq are fp32 m and v.  bits 8: exp_avg holds E4M3 codes of m and exp_avg_sq
 * those of sqrt(v); every NTOPS_ADAMW_BLOCK elements (counted from the tensor's start, the last block may be short) share a
 * scale (value = code / scale), the power of two that brings the largest finite magnitude of the block into (224, 448]; codes are
 * rounded stochastically with 16 bits hashed from the element's index and `seed`, a root above zero never to zero, and a value
 * that is not finite becomes NaN, at no cost to its neighbours.  The parameters move by the moments before they are rounded.
 * Tensors must not overlap, and lie below 2^48 (NTFP8_ERR_UNSUPPORTED).  An empty tensor (n = 0) is passed over. */
#define NTOPS_ADAMW_BLOCK 256
typedef struct ntops_adamw_tensor {
    void* param;
    const void* grad;
    void* exp_avg;
    void* exp_avg_sq;
    void* copy;                /* NULL: none */
    float* exp_avg_scale;      /* bits 8: [ceil(n / NTOPS_ADAMW_BLOCK)] */
    float* exp_avg_sq_scale;
    int64_t n;
} ntops_adamw_tensor;
typedef struct ntops_adamw_options {
    double lr, beta1, beta2, eps, weight_decay;
    int64_t step;              /* >= 1 */
    int param_dtype, grad_dtype, copy_dtype, bits;
    uint32_t seed;             /* bits 8 */
    const float* grad_scale;   /* device scalar, NULL: 1 */
} ntops_adamw_options;
int ntops_adamw(const ntops_adamw_tensor* tensors, int count, const ntops_adamw_options* options, void* stream);
/* What ntops_adamw would say of these arguments, without a launch: for a caller whose step is several calls (types differ), of
 * which none should be made if one is refused. */
int ntops_adamw_check(const ntops_adamw_tensor* tensors, int count, const ntops_adamw_options* options);

/* out = fp32 of what E4M3 codes and block scales as above stand for */
int ntops_adamw_unpack(const void* codes, const float* scale, int64_t n, float* out, void* stream);

/* Softmax cross entropy of the logits x weight^T under int64 labels, the logits never in memory as such.
 *   x [tokens, hidden], weight [vocab, hidden], both of x_dtype (NTFP8_BF16 or NTFP8_F16), rows x_stride / weight_stride
 *   elements apart (any number; more than 2^22, or no multiple of 8: a copy in the workspace); labels [tokens].  hidden and vocab
 *   at most 2^22.  Products on the matrix cores with fp32 sums, the softmax's maxima and sums in fp32.
 * Outputs: losses [tokens] fp32 = logsumexp - logit of the label, 0 where the label is ignore_index, NaN where it is outside
 * [0, vocab).  loss (may be NULL): their sum, divided by the number of labels that are not ignored if `mean` (0 if all
 * are).  Gradients of `loss` (dx and dweight both NULL: none are made; each may be NULL by itself): dx [tokens, hidden]
 * dense, dweight [vocab, hidden] dense, each of x_dtype, or fp32 (grad_dtype NTFP8_F32).
 * workspace: ntops_linear_cross_entropy_workspace(...) bytes, aligned to 256 (2 bytes a logit of a piece and 4 an element of dx,
 * at most 2 GiB of each, and copies of x and, if need be, weight).  Tokens beyond ntops_linear_cross_entropy_piece(vocab) at a
 * time go through it in pieces; dweight of type fp32 then collects the pieces, and a 16-bit dweight needs all tokens in
 * one piece (NTFP8_ERR_UNSUPPORTED otherwise: take fp32). */
typedef struct ntops_linear_cross_entropy_desc {
    const void* x;
    const void* weight;
    const int64_t* labels;
    int64_t tokens, hidden, vocab, x_stride, weight_stride, ignore_index;
    int x_dtype, mean, grad_dtype;
    float* losses;
    float* loss;
    void* dx;
    void* dweight;
    void* workspace;
} ntops_linear_cross_entropy_desc;
int64_t ntops_linear_cross_entropy_piece(int64_t vocab);
int64_t ntops_linear_cross_entropy_workspace(const ntops_linear_cross_entropy_desc* d);
int ntops_linear_cross_entropy(const ntops_linear_cross_entropy_desc* d, void* stream);

/* out = out_dtype(x * *factor) for `count` tensors of n elements of x_dtype; out may be x (same type): then nothing is read or
 * written where *factor is 1.  What a backward pass does with the gradient that reaches a loss. */
typedef struct ntops_scale_tensor {
    const void* x;
    void* out;
    int64_t n;
} ntops_scale_tensor;
int ntops_scale(const ntops_scale_tensor* tensors, int count, int x_dtype, const float* factor, int out_dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* NTOPS_H */
