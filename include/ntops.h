/* ntops — C ABI of the operators that stand beside the FP8 linears in a training step (MI355X, gfx950): layer
 * normalisation, the norms around a block with its gate and residual, rotary positions, attention, the vocabulary projection with
 * its softmax cross entropy, and AdamW over many tensors.  They live in the same library as the entry points of ntfp8.h and follow its conventions: device pointers owned by the caller, nothing
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

/* Root-mean-square norms around a block, over rows of `cols` elements (16384 at most of a 16-bit x, 8192 of fp32):
 *   p = x / rms(x) * post_weight, or x where post_weight is NULL;  rms(x) = root(mean(x^2) + eps)
 *   h = residual_scale * residual + gate * p, rounded to residual_dtype;  y = h / rms(h) * weight of the rounded h, rounded to x_dtype
 * in fp32.  residual NULL: the norm alone, y = x / rms(x) * weight, without post_weight, gate and h.  x, y: x_dtype; residual, h:
 * residual_dtype (fp32, or x_dtype); weight, post_weight [cols] (each may be NULL) and a channel's gate [cols]: w_dtype (fp32, or x_dtype).
 * gate_kind NTOPS_GATE_NONE, NTOPS_GATE_CHANNEL, or NTOPS_GATE_ELEMENT (a gate of x_dtype for every element, rows gate_stride apart).
 * y and h are dense; rows of x and residual lie x_stride and residual_stride elements apart.  first and second [rows] fp32 receive 1 / rms
 * of x (where post_weight is given) and of h for a backward pass; both NULL if none follows. */
#define NTOPS_GATE_NONE 0
#define NTOPS_GATE_CHANNEL 1
#define NTOPS_GATE_ELEMENT 2
typedef struct ntops_rms_norm_desc {
    const void* x;
    const void* residual;
    const void* gate;
    const void* weight;
    const void* post_weight;
    int64_t rows, cols, x_stride, residual_stride, gate_stride;
    int x_dtype, residual_dtype, w_dtype, gate_kind;
    float eps, residual_scale;
    void* y;
    void* h;
    float* first;
    float* second;
} ntops_rms_norm_desc;
int ntops_rms_norm_forward(const ntops_rms_norm_desc* d, void* stream);

/* Gradients of the above from dy (type of x) and dh (type of h), either of which may be NULL (nothing arrives there), rows dy_stride and
 * dh_stride apart.  Of the desc: x, gate, weights, h (NULL: there was no residual), first, second, strides, types, eps and
 * residual_scale; y and residual are not read.  dx (dense, type of x), dresidual (dense, type of h), dweight, dpost_weight (w_dtype) and dgate (as the
 * gate; dense) may each be NULL.  Sums over rows are made in fp32 within a workgroup and in 64 bits over them, in an order that
 * depends on the sizes alone.  scratch: ntops_rms_norm_scratch(...) bytes, 16-byte aligned, for the gradients that are such sums. */
typedef struct ntops_rms_norm_grads {
    const void* dy;
    const void* dh;
    int64_t dy_stride, dh_stride;
    void* dx;
    void* dresidual;
    void* dgate;
    void* dweight;
    void* dpost_weight;
    void* scratch;
} ntops_rms_norm_grads;
int64_t ntops_rms_norm_scratch(const ntops_rms_norm_desc* d);
int ntops_rms_norm_backward(const ntops_rms_norm_desc* d, const ntops_rms_norm_grads* g, void* stream);

/* Rotary positions: the first 2 * pairs elements of every head of q and k are turned, pair i by angle = position * frequencies[i]:
 *   (a, b) -> (a cos - b sin, b cos + a sin) * scale;  `inverse`: by -angle (what a backward pass does with the gradients)
 * a and b lie side by side (`interleaved`) or `pairs` elements apart; elements behind 2 * pairs are copied.  Angles are made in 64 bits, sines,
 * cosines and products in fp32.  q [tokens][heads][head_dim] with q_stride elements between tokens and q_head between heads, k likewise; k (or q) may be NULL
 * with kv_heads (heads) 0.  q_out and k_out are dense.  Token t is at positions[t mod position_count] (int32 or int64, by
 * position_bits).  head_dim <= 2048, heads + kv_heads <= 16384. */
typedef struct ntops_rotary_desc {
    const void* q;
    const void* k;
    void* q_out;
    void* k_out;
    int64_t tokens, q_stride, q_head, k_stride, k_head;
    int heads, kv_heads, head_dim, pairs, dtype;
    const void* positions;
    int64_t position_count;
    int position_bits;
    const double* frequencies;   /* [pairs] radians a position */
    int interleaved, inverse;
    float scale;
} ntops_rotary_desc;
int ntops_rotary(const ntops_rotary_desc* d, void* stream);

/* Attention: out = softmax(scale q k^T) v, a head of q each; heads of q share those of k and v (heads a multiple of kv_heads, head h
 * reads kv head h / (heads / kv_heads)).  Rows of tokens: q [q_rows][heads][head_dim], k and v [k_rows][kv_heads][head_dim], elements
 * between rows q_stride, k_stride, v_stride, between heads q_head, k_head, v_head, all multiples of 8, on 16-byte boundaries.
 * Sequences: packed, sequence s being rows cu_q[s] .. cu_q[s + 1] - 1 of q and cu_k[s] .. cu_k[s + 1] - 1 of k and v (device
 * memory, int32 [sequences + 1], not decreasing; offsets outside the rows that there are count as the nearest inside); or cu_q and cu_k NULL, `sequences` of equal
 * lengths q_rows / sequences and k_rows / sequences, q_batch, k_batch, v_batch elements apart.
 * causal: row i of a sequence of n queries and m keys sees the keys 0 .. m - n + i, so that the last rows of both belong together.  A
 * row that sees no key, and a row of q that belongs to no sequence, is 0, and so are its gradients; what is in rows of k and v
 * that a row does not see, NaN say, does not reach it.  A row whose keys all score minus infinity is 0 / 0: it and its gradients are NaN.
 * head_dim <= 128, a multiple of 8; scale 1e-30 to 1e30; dtype NTFP8_BF16 or NTFP8_F16.  Scores, maxima, sums and outputs are fp32 until the one rounding of
 * out; the softmax's numerators are rounded to dtype for the product with v.  out is dense; lse [heads][q_rows] fp32 (minus the logarithm of a row's
 * sum of exponentials, over scale) is what a backward pass needs, NULL if none follows.  q_rows * heads and k_rows * kv_heads at most 2^27.
 * out_low (as out, a byte an element, aligned to 8; may be NULL): what a forward call's rounding of out left out, 8 more bits of
 * significand, with which a backward call's dq and dk lose less.
 * workspace: ntops_attention_workspace(d, backward) bytes, aligned to 256.  plan (packed sequences, may be NULL): ntops_attention_plan(d) bytes,
 * aligned to 256, that a forward call fills and the backward call of the same sizes and offsets reads; without it each makes its own (in its
 * workspace, which is the larger for it).
 * Backward: dq, dk, dv (dense, dtype, each may be NULL) from dout (do_stride, do_head, do_batch, with the limits of q's) and the q, k, v, out and lse of the forward call.
 * The same inputs give the same bits.  fp16: p and ds are kept with powers of two on them, ds with one a call, from the largest finite dout and v, so that gradients
 * below its normal range survive that are no more than 2^28 below 2 head_dim times these. */
typedef struct ntops_attention_desc {
    const void* q;
    const void* k;
    const void* v;
    int64_t q_stride, k_stride, v_stride, q_head, k_head, v_head, q_batch, k_batch, v_batch;
    const int32_t* cu_q;
    const int32_t* cu_k;
    int64_t sequences, q_rows, k_rows;
    int heads, kv_heads, head_dim, dtype, causal;
    float scale;
    void* out;
    uint8_t* out_low;
    float* lse;
    void* workspace;
    void* plan;
    const void* dout;
    int64_t do_stride, do_head, do_batch;
    void* dq;
    void* dk;
    void* dv;
} ntops_attention_desc;
int64_t ntops_attention_workspace(const ntops_attention_desc* d, int backward);
int64_t ntops_attention_plan(const ntops_attention_desc* d);
int ntops_attention_forward(const ntops_attention_desc* d, void* stream);
int ntops_attention_backward(const ntops_attention_desc* d, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* NTOPS_H */
