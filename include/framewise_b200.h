/* framewise_b200.h -- C ABI of the operators of framewise training on B200 (sm_100a): output layer with
 * softmax cross entropy, label embedding, scores of labels off logits, AdamW, Muon.  They follow an alignment or a
 * label sequence: a network is trained on one class per frame (the (B,T) result of fbw_b200_viterbi) or on label
 * sequences.
 * No counterpart in the reference, which ends at the losses on log probabilities.
 *
 * All pointers are DEVICE pointers unless a comment says host.  Sizes are 64-bit.  No call allocates
 * device memory, synchronises, or keeps anything of a call for the next one; calls enqueue work on the
 * given stream and may be captured into a CUDA graph.  Buffers called `saved` and `work` must be 256-byte
 * aligned, grad_table 16-byte; other tensors need the alignment of their element type only.
 *
 * Positions.  Activations and labels are (B,T) padded batches.  A position (b,t) counts if
 * t < seq_lens[b] (all t where seq_lens is NULL) and its label is not `ignore_index`.  Nothing is read of
 * the activations and gradients of positions that do not count: they may hold NaN.  A position that counts
 * with a label outside [0, V) cannot be refused without reading it on the host: its results, and the
 * gradients that it takes part in, are NaN. */
#ifndef FRAMEWISE_B200_H
#define FRAMEWISE_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st* framewise_b200_stream_t;

/* Status codes (0 = success). */
enum {
    FRAMEWISE_B200_OK           = 0,
    FRAMEWISE_B200_BAD_ARGUMENT = 1, /* null pointer, negative dimension, size past a limit, misaligned buffer */
    FRAMEWISE_B200_WORKSPACE    = 2, /* caller-provided buffer too small                                      */
    FRAMEWISE_B200_CUDA_ERROR   = 3, /* a CUDA call failed (see cudaGetLastError)                             */
    FRAMEWISE_B200_TENSOR_MAP   = 4, /* the driver made no tensor map (or has no call for it)                 */
    FRAMEWISE_B200_OVERLAP      = 5  /* what is written is given twice, or overlaps something else of the call */
};

enum { FRAMEWISE_B200_F32 = 0, FRAMEWISE_B200_BF16 = 1 };

/* Sizes and types of one call of the cross entropy.  B*T, V and D below 2^31. */
typedef struct {
    int64_t B, T, V, D;
    int64_t hidden_stride_b, hidden_stride_t; /* in elements; the last dimension of `hidden` is dense */
    int64_t ignore_index;
    int32_t dtype;     /* of hidden, weight, bias and their gradients */
    int32_t labels64;  /* targets are int64 (else int32)              */
    int32_t has_bias;
    int32_t train;     /* the backward pass will follow               */
    int32_t copy_weight; /* bf16: nonzero where `weight` is not 16-byte aligned or D is no multiple of 8
                            (it is then copied into `saved`); f32: ignored */
} framewise_b200_ce_shape;

/* Output layer and softmax cross entropy: for z = hidden . weight^T + bias,
 *     loss[b,t] = log sum_v exp z[v] - z[target],  0 at positions that do not count.
 * The logits are never held: a tile of them lives in tensor memory, and per row a running maximum and sum.
 * Products of bf16 inputs are exact and summed in 32 bits; f32 inputs are split into three bf16 parts
 * (24 bits), whose six leading products are summed in 32 bits.
 * hidden (B,T,D), weight (V,D) dense, bias (V), targets (B,T) dense, loss (B,T) f32.
 * `saved`: kept by the caller from the forward to the backward pass; `work`: scratch of one call.
 * The weight must not change between the two passes. */
int framewise_b200_ce_bytes(const framewise_b200_ce_shape* shape, size_t* saved_bytes,
                            size_t* forward_work_bytes, size_t* backward_work_bytes);
int framewise_b200_ce_forward(const framewise_b200_ce_shape* shape, const void* hidden, const void* weight,
                              const void* bias, const void* targets, const int32_t* seq_lens, float* loss,
                              void* saved, size_t saved_bytes, void* work, size_t work_bytes,
                              framewise_b200_stream_t stream);

/* Its gradients, for the incoming gradient `grad_loss` (B,T) f32 with the given strides (0 allowed):
 *     q = grad_loss (softmax(z) - onehot(target));  grad_hidden = q . weight,  grad_weight = q^T . hidden,
 *     grad_bias = sum of q.
 * The logits are computed again, q is held for some thousand rows at a time: in bf16 for bf16 inputs (8 bits of
 * each value, as the gradients themselves have, which are then some 1.4 times as far from exact ones as their own rounding;
 * 16 bits for up to 256 positions), in three bf16 parts for f32.  Outputs are dense; a NULL output is not computed.  Sums
 * are formed in a fixed order: equal calls give equal bits. */
int framewise_b200_ce_backward(const framewise_b200_ce_shape* shape, const void* weight,
                               const float* grad_loss, int64_t grad_stride_b, int64_t grad_stride_t,
                               void* grad_hidden, void* grad_weight, void* grad_bias,
                               const void* saved, size_t saved_bytes, void* work, size_t work_bytes,
                               framewise_b200_stream_t stream);

/* Scaled embedding: out[b,t,:] = scale * table[label[b,t],:], zeros at positions that do not count.
 * table (V,D) dense, labels (B,T) dense, out (B,T,D) dense, both of `dtype`; the product is formed in 32 bits
 * and rounded once. */
int framewise_b200_embed_forward(int64_t B, int64_t T, int64_t V, int64_t D, int32_t dtype, int32_t labels64,
                                 int64_t ignore_index, float scale, const void* table, const void* labels,
                                 const int32_t* seq_lens, void* out, framewise_b200_stream_t stream);

/* Its gradient: grad_table[v,:] = scale * sum of grad_out[b,t,:] over the positions with label v, added in
 * 32 bits in the order of the positions (in pieces of a fixed size), rounded once; equal calls give equal
 * bits.  grad_out (B,T,D) with strides in elements (0 allowed), its last dimension dense. */
size_t framewise_b200_embed_bytes(int64_t B, int64_t T, int64_t V, int64_t D);
int framewise_b200_embed_backward(int64_t B, int64_t T, int64_t V, int64_t D, int32_t dtype, int32_t labels64,
                                  int64_t ignore_index, float scale, const void* grad_out,
                                  int64_t grad_stride_b, int64_t grad_stride_t, const void* labels,
                                  const int32_t* seq_lens, void* grad_table, void* work, size_t work_bytes,
                                  framewise_b200_stream_t stream);

/* One tensor of an AdamW step.  `exp_avg` and `exp_avg_sq` point to n floats (state_bits 32) or to n codes of
 * 8 bits (int8, uint8) with one f32 step per block of FRAMEWISE_B200_STATE_BLOCK values.  `master`: n floats, or NULL
 * where the parameter itself is f32 (or is to be updated without a copy in 32 bits). */
#define FRAMEWISE_B200_STATE_BLOCK 256
typedef struct {
    void*       param;
    const void* grad;
    float*      master;
    void*       exp_avg;
    void*       exp_avg_sq;
    float*      exp_avg_steps;
    float*      exp_avg_sq_steps;
    int64_t     n;
} framewise_b200_tensor;

/* A step of AdamW over `count` tensors (HOST array), in few launches:
 *     m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
 *     x = x (1 - lr weight_decay) - m lr / (1 - beta1^step) / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 * in 32 bits, x being the master copy where there is one (the parameter is then x rounded once).
 * 8-bit states: a code c and its block's step k stand for c |c| k; the codes of the first moment are -127..127,
 * those of the ROOT of the second 0..255, at least 1 where the root is not zero.  A block's step is its largest
 * magnitude / 127^2 (255^2), zero where that is below 2^-120; a block with an infinity or a NaN stands for it
 * throughout.  Where both betas are 0.98 at most, the root of |value| / k is rounded to the nearest whole number; where one
 * is above, an offset is added first, for such codes would hardly ever follow a moment that shrinks.  For value i of its
 * tensor at step s: ((i a + s b) mod 2^32 >> 9) 2^-23 - 1/2 with a, b = 2447445413, 3242174889 for the first moment and
 * 3242174889, 2447445413 for the second.  The sum, rounded to f32, is rounded to the nearest whole number and limited
 * to 0..127 (255). */
int framewise_b200_adamw(const framewise_b200_tensor* tensors, int64_t count, int32_t dtype,
                         int32_t state_bits, double lr, double beta1, double beta2, double eps,
                         double weight_decay, int64_t step, framewise_b200_stream_t stream);

/* The same step; but where a parameter is not its master copy rounded, the program has changed it since (a model loaded,
 * weights clipped), and the copy starts from the parameter's value.  Parameters without a copy: as above. */
int framewise_b200_adamw_follow(const framewise_b200_tensor* tensors, int64_t count, int32_t dtype,
                                int32_t state_bits, double lr, double beta1, double beta2, double eps,
                                double weight_decay, int64_t step, framewise_b200_stream_t stream);

/* 8-bit states to the values that they stand for: the codes in exp_avg / exp_avg_sq to f32 in param / master
 * (the second moment itself, not its root); other fields are ignored. */
int framewise_b200_adamw_decode(const framewise_b200_tensor* tensors, int64_t count, framewise_b200_stream_t stream);

/* Sizes and types of one call on distributions over V classes that are in memory.  B*T below 2^31, V below 2^27. */
typedef struct {
    int64_t B, T, V;
    int64_t logits_stride_b, logits_stride_t; /* in elements; the last dimension of `logits` is dense */
    int64_t ignore_index;
    int32_t dtype;    /* of logits and their gradient          */
    int32_t labels64; /* labels and top_labels are int64 (else int32) */
    int32_t top;      /* alternatives: 0 .. min(V, 32)         */
} framewise_b200_scores_shape;

/* For z = logits[b,t,:] and log p = z - log sum_v exp z[v]:
 *     log_probs[b,t] = log p[label];  entropy[b,t] = - sum_v p log p  (classes of z = -inf add nothing);
 *     top_labels[b,t,:], top_log_probs[b,t,:]: the `top` largest of z in falling order (equal ones by their index; NaN is the
 *     largest) and their log p.
 * Positions that do not count: 0, and `ignore_index` as labels.  A row of -inf alone: log probabilities -inf, entropy 0.
 * A row with NaN or +inf: NaN.  logits (B,T,V), labels (B,T) dense, outputs dense, f32.  `kept`: 16 B T bytes, 16-byte
 * aligned, for the backward pass, or NULL. */
int framewise_b200_scores_forward(const framewise_b200_scores_shape* shape, const void* logits, const void* labels,
                                  const int32_t* seq_lens, float* log_probs, float* entropy, float* top_log_probs,
                                  void* top_labels, void* kept, framewise_b200_stream_t stream);

/* Incoming gradients, f32, with strides in elements (0 allowed); NULL: none. */
typedef struct {
    const float* log_probs;
    const float* entropy;
    const float* top_log_probs;
    int64_t log_probs_stride_b, log_probs_stride_t, entropy_stride_b, entropy_stride_t;
    int64_t top_stride_b, top_stride_t, top_stride_k;
} framewise_b200_scores_grads;

/* grad_logits (B,T,V) dense: g (onehot(label) - p) - g_H p (log p + entropy) + sum_j g_j (onehot(top_labels[j]) - p), in 32
 * bits, rounded once; zeros at positions that do not count and in rows of -inf alone. */
int framewise_b200_scores_backward(const framewise_b200_scores_shape* shape, const void* logits, const void* labels,
                                   const int32_t* seq_lens, const void* top_labels, const void* kept,
                                   const framewise_b200_scores_grads* grads, void* grad_logits,
                                   framewise_b200_stream_t stream);

/* Orthogonalisation by Newton-Schulz products.  For X = x / max(|x|, eps) (Frobenius norm; matrices with more rows than
 * columns lie transposed) and each of `steps` triples (a, b, c) of `coefficients` (HOST array of 3 steps values):
 *     A = X X^T;  X = a X + (b A + c A A) X
 * X is held in 32 bits; the products' operands are rounded to 11 bits for bf16 matrices (22 for A = X X^T where the shorter side is at most
 * 128), to 22 for f32 ones, the sums are formed in 32 bits in a fixed order: equal calls give equal bits.  `count` dense matrices
 * of rows x cols one after another, out likewise (may be x).  eps: any positive number.  A matrix with NaN or an infinity becomes
 * NaN; zeros stay zeros.  Coefficients that let a singular value grow past 10^6 are refused.  The result of _bytes is 0 for sizes
 * past the limits. */
size_t framewise_b200_orthogonalize_bytes(int64_t count, int64_t rows, int64_t cols, int32_t dtype);
int framewise_b200_orthogonalize(int64_t count, int64_t rows, int64_t cols, int32_t dtype, const void* x, void* out,
                                 const double* coefficients, int32_t steps, double eps, void* work, size_t work_bytes,
                                 framewise_b200_stream_t stream);

/* One matrix of a Muon step: param and grad of rows x cols (`dtype`), momentum (f32), dense; master: f32, or NULL. */
typedef struct {
    void*       param;
    const void* grad;
    float*      momentum;
    float*      master;
    int64_t     rows, cols;
} framewise_b200_matrix;

/* A step of Muon over `count` matrices (HOST array):
 *     v = v + (g - v) (1 - beta);   u = nesterov ? g + (v - g) beta : v;   o = u orthogonalised as above
 *     x = x (1 - lr weight_decay) - lr s o,   s = sqrt(max(1, rows / cols)), or match_rms: 0.2 sqrt(max(rows, cols))
 * x being the master copy where there is one (the parameter is then x rounded once); follow: a copy of which its parameter
 * is not the rounded value starts from the parameter.  What is written (params, momentum, masters) overlaps nothing else of the
 * call; gradients may be shared.  Matrices of up to 128 x 256 (either way round) take a launch for every 24 of them; the others go
 * together, 256 of them and two gigabytes of scratch at most at a time, through a chain of 3 steps + 2 launches and one for every 24 of
 * them. */
size_t framewise_b200_muon_bytes(const framewise_b200_matrix* matrices, int64_t count, int32_t dtype);
int framewise_b200_muon(const framewise_b200_matrix* matrices, int64_t count, int32_t dtype, double lr, double beta,
                        int32_t nesterov, double weight_decay, int32_t match_rms, const double* coefficients,
                        int32_t steps, double eps, int32_t follow, void* work, size_t work_bytes,
                        framewise_b200_stream_t stream);

/* Number of kernels of this library launched by this process so far. */
int64_t framewise_b200_launch_count(void);

/* Text for a status code (static storage). */
const char* framewise_b200_status_string(int status);

#ifdef __cplusplus
}
#endif
#endif /* FRAMEWISE_B200_H */
