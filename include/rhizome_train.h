/*
 * rhizome_train.h -- C ABI of the training operators in librhizome_gdr.so:
 * the backward passes of the Local block's mixer (rhizome_gdr.h has the
 * forward ones) and layer norm.
 *
 * Conventions are rhizome_gdr.h's: plain pointers and sizes, row-major tensors
 * in caller-owned device memory, everything validated before the GPU is
 * touched, launches ordered on `stream` and asynchronous to the host, no
 * allocation, results deterministic (no atomics).  Nothing is kept between
 * calls, so that a call can be captured into a graph; calls that may run at
 * the same time need a workspace each.
 */
#ifndef RHIZOME_TRAIN_H
#define RHIZOME_TRAIN_H

#include "rhizome_gdr.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Backward pass of rhz_gdr_prefill, for training on the GPU: the gradients of
 * a scalar with respect to q, k, v, the gates, beta and the initial state,
 * from grad_o and grad_final_state, its gradients with respect to o and the
 * final state.  Nothing of the forward call is kept: the inputs are given
 * again and the states recomputed.  The reference names this adjoint
 * (docs/kernels.md:16) without implementing it.
 *
 * In 64-token chunks on MFMA, as the CHUNKED prefill: bf16 tensors as fp16
 * operands, scaled by powers of two, with fp32 accumulation and fp32 states;
 * fp32 tensors in fp32 throughout, accurate where beta |k|^2 <= 2 and alpha <= 1.
 *
 * A bf16 head whose inputs leave the prefill's domain (a key row with |k|^2 >
 * 1.03125, a beta or alpha outside [0, 1], a value that is not finite, q, k, v
 * and grad_o included) or whose values leave fp16's range on the way is computed
 * in fp32 in the same call, by one workgroup: 2.4 us a token at d_k = d_v = 128,
 * 3.9 at d_v = 256.  4 x 4096 tokens of 16 heads at d = 128 take 10 ms with one
 * such head or all, 0.5 ms without and 1.8 ms as fp32 tensors, which is how to
 * pass inputs that leave the domain often.
 *
 * A bf16 call's errors are of bf16's rounding or near it, taken of the largest
 * terms that a gradient is summed from.  Where these cancel, what remains has
 * fewer digits: keys all alike with beta = 0.9 leave grad_v 2 % off, and grad_gate
 * and grad_initial_state, small differences then, off by up to their own size.
 * Values of a chunk share powers of two, so that those of 2^-14 of its largest and
 * less lose digits: a grad_o row among others 10^5 times larger, or what a chunk
 * makes of a state that its decays shrink by more than that.  fp32 tensors have
 * neither loss.
 *
 * grad_gate is the gradient of the gate as it is given: of g, or of alpha
 * (RHZ_GATE_ALPHA; finite at alpha = 0 too).  grad_q, grad_k, grad_v,
 * grad_gate and grad_beta have the dtype of q; grad_initial_state is fp32, with
 * a bf16 call's error all the same.  Rows of a pack outside every sequence are
 * left as they were.  No output overlaps an input, the workspace or another
 * output. */
typedef struct rhz_gdr_prefill_backward_args {
    int32_t batch;   /* dense: B;  packed: number of sequences N (>= 1) */
    int32_t seq_len; /* dense: T;  packed: total tokens in the pack (>= 0) */
    int32_t heads;   /* H >= 1 */
    int32_t d_k;     /* 1..128 */
    int32_t d_v;     /* 1..1024 */
    int32_t dtype;     /* rhz_dtype of q, k, v, grad_o and of the gradients */
    int32_t gate_kind; /* rhz_gate */
    const void* q;      /* [tokens, H, d_k], as for rhz_gdr_prefill */
    const void* k;
    const void* v;      /* [tokens, H, d_v] */
    const float* gate;  /* [tokens, H] */
    const float* beta;  /* [tokens, H] */
    const void* grad_o; /* [tokens, H, d_v] */
    const int32_t* cu_seqlens;     /* device [N+1], or NULL (dense), as for rhz_gdr_prefill */
    const float* initial_state;    /* [batch, H, d_v, d_k], or NULL for zeros */
    const float* grad_final_state; /* [batch, H, d_v, d_k], or NULL for zeros */
    void* grad_q;       /* [tokens, H, d_k] out */
    void* grad_k;       /* [tokens, H, d_k] out */
    void* grad_v;       /* [tokens, H, d_v] out */
    void* grad_gate;    /* [tokens, H] out */
    void* grad_beta;    /* [tokens, H] out */
    float* grad_initial_state; /* [batch, H, d_v, d_k] out, or NULL */
    void* workspace;    /* device scratch, 256-byte aligned */
    size_t workspace_bytes;
} rhz_gdr_prefill_backward_args;

/* Bytes of device workspace rhz_gdr_prefill_backward needs for these arguments
 * (cu_seqlens tells a pack; no other pointer is read): per chunk of 64 tokens
 * and head the states on its either side and what the scans hand on, at d_k =
 * d_v = 128 some 115 KiB for bf16 and 227 for fp32.  Two calls that may run at
 * the same time need a workspace each. */
rhz_status rhz_gdr_prefill_backward_workspace_size(const rhz_gdr_prefill_backward_args* args,
                                                   size_t* bytes);

rhz_status rhz_gdr_prefill_backward(const rhz_gdr_prefill_backward_args* args, void* stream);

/* Backward pass of rhz_gdr_conv_prepare, the Local block's prologue: from the
 * gradients of its outputs q, k, v, beta and g (as rhz_gdr_prefill_backward
 * gives them for RHZ_GATE_LOG_ALPHA) and of the final conv state, those of x,
 * the weights, the bias, the logits, a_log and the initial conv state.  The
 * forward call's inputs are given again and the convolution formed again, in
 * fp32.  The same shapes as the forward call (else RHZ_ERR_UNSUPPORTED).  Rows
 * of a pack outside every sequence are left as they were and add nothing.  No
 * output overlaps an input, the workspace or another output. */
typedef struct rhz_gdr_conv_prepare_backward_args {
    int32_t batch;    /* dense: B;  packed: number of sequences N (>= 1) */
    int32_t seq_len;  /* dense: T;  packed: total tokens (>= 0) */
    int32_t heads;    /* H >= 1 */
    int32_t d_k;      /* >= 1 */
    int32_t d_v;      /* >= 1 */
    int32_t dtype;    /* rhz_dtype of x, of grad_q .. grad_g and of grad_x */
    float q_scale;    /* as in the forward call; must be finite */
    const void* x;              /* [tokens, C], C = H (2 d_k + d_v) */
    const float* weight;        /* [C, 4] */
    const float* bias;          /* [C], or NULL for zero */
    const int32_t* cu_seqlens;  /* [N+1] or NULL (dense) */
    const float* initial_state; /* [batch, C, 3], or NULL for zeros */
    const float* beta_logit;    /* [tokens, H] */
    const float* alpha_logit;   /* [tokens, H] */
    const float* a_log;         /* [H] */
    const void* grad_q;         /* [tokens, H, d_k] */
    const void* grad_k;         /* [tokens, H, d_k] */
    const void* grad_v;         /* [tokens, H, d_v] */
    const void* grad_beta;      /* [tokens, H] */
    const void* grad_g;         /* [tokens, H] */
    const float* grad_final_state; /* [batch, C, 3], or NULL for zeros */
    void* grad_x;               /* [tokens, C] out */
    float* grad_weight;         /* [C, 4] out */
    float* grad_bias;           /* [C] out, or NULL */
    float* grad_beta_logit;     /* [tokens, H] out */
    float* grad_alpha_logit;    /* [tokens, H] out */
    float* grad_a_log;          /* [H] out */
    float* grad_initial_state;  /* [batch, C, 3] out, or NULL */
    void* workspace;            /* device scratch, 256-byte aligned */
    size_t workspace_bytes;
} rhz_gdr_conv_prepare_backward_args;

rhz_status rhz_gdr_conv_prepare_backward_workspace_size(const rhz_gdr_conv_prepare_backward_args* args,
                                                        size_t* bytes);

rhz_status rhz_gdr_conv_prepare_backward(const rhz_gdr_conv_prepare_backward_args* args, void* stream);

/* Layer norm of every row of `dim` values: y = (x - mean) / sqrt(variance +
 * eps) * weight + bias, the variance from the centred values, in fp32.  y may
 * be x itself; else it overlaps no input. */
typedef struct rhz_layernorm_args {
    int32_t rows;     /* >= 0 */
    int32_t dim;      /* 1..8192 */
    int32_t dtype;    /* rhz_dtype of x and y */
    float eps;        /* >= 0 */
    const void* x;        /* [rows, dim] */
    const float* weight;  /* [dim] */
    const float* bias;    /* [dim], or NULL for zero */
    void* y;              /* [rows, dim] */
} rhz_layernorm_args;

rhz_status rhz_layernorm(const rhz_layernorm_args* args, void* stream);

/* Backward pass of a row norm, rhz_layernorm or rhz_rmsnorm_heads: from grad_y
 * and the forward call's x, grad_x and the sums over the rows for the weights
 * (rhz_rmsnorm_heads's scale) and for layer norm's bias.  Statistics and sums
 * in fp32.  No output overlaps an input, the workspace or another output. */
typedef struct rhz_norm_backward_args {
    int32_t rows;     /* >= 0 */
    int32_t dim;      /* 1..8192 */
    int32_t dtype;    /* rhz_dtype of grad_y, x and grad_x */
    float eps;        /* as in the forward call */
    const void* grad_y;   /* [rows, dim] */
    const void* x;        /* [rows, dim] */
    const float* weight;  /* [dim]: layer norm's weight, or RMSNorm's scale */
    void* grad_x;         /* [rows, dim] out */
    float* grad_weight;   /* [dim] out */
    float* grad_bias;     /* [dim] out, or NULL; NULL for RMSNorm */
    void* workspace;      /* device scratch, 256-byte aligned */
    size_t workspace_bytes;
} rhz_norm_backward_args;

/* Bytes of workspace of either of the two calls below: at most 4 KiB per
 * column. */
rhz_status rhz_norm_backward_workspace_size(const rhz_norm_backward_args* args, size_t* bytes);

rhz_status rhz_layernorm_backward(const rhz_norm_backward_args* args, void* stream);

rhz_status rhz_rmsnorm_heads_backward(const rhz_norm_backward_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* RHIZOME_TRAIN_H */
