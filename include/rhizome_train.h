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
 * operands, scaled tile by tile by powers of two, with fp32 accumulation and
 * fp32 states; fp32 tensors in fp32 throughout.  A bf16 head whose inputs
 * leave the prefill's domain (a key row with |k|^2 > 1.03125, a beta or alpha
 * outside [0, 1], a value that is not finite, q, k, v and grad_o included) is
 * computed in fp32 in the same call, several times slower.  fp32 tensors are
 * accurate where beta |k|^2 <= 2 and alpha <= 1.
 *
 * grad_gate is the gradient of the gate as it is given: of g, or of alpha
 * (RHZ_GATE_ALPHA; finite at alpha = 0 too).  grad_q, grad_k, grad_v,
 * grad_gate and grad_beta have the dtype of q: a bf16 call's gate gradients
 * are sums of products of 11-bit operands, whose error is that of bf16's
 * rounding or near it.  grad_initial_state is fp32, with the same error in a
 * bf16 call.  Rows of a pack outside every sequence are left as they were.
 * No output overlaps an input, the workspace or another output. */
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
 * and head some 1280 bytes per padded d_k and d_v at d_k = d_v (160 KiB at 128
 * for bf16, 320 for fp32).  Two calls that may run at the same time need a
 * workspace each. */
rhz_status rhz_gdr_prefill_backward_workspace_size(const rhz_gdr_prefill_backward_args* args,
                                                   size_t* bytes);

rhz_status rhz_gdr_prefill_backward(const rhz_gdr_prefill_backward_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* RHIZOME_TRAIN_H */
