/*
 * rhizome_attention.h -- C ABI of the Global block's latent attention in
 * librhizome_gdr.so: rotary positions, the paged cache of latents with its
 * writer and its reader of a sequence's last positions, and the prefill with
 * its backward pass.
 *
 * A token has one latent c_t (d_c values) and one rotary key r_t (d_r values)
 * for all heads.  Expanded, head h has the key [k_t,h | r_t] and the value
 * v_t,h, both projections of c_t; absorbed, its query is projected instead and
 * meets the latent itself, which is key and value at once:
 *
 *     scores  s = scale * q . [k | r]     or   scale * q . [c | r]
 *     o = softmax(s) v                    or   softmax(s) c
 *
 * The reference has both on the CPU (crates/ops/src/attention.rs:7-70,
 * 164-219, 226-300).  A query that sees no key has an output of zeros and a
 * logarithm of -infinity.  What a query does not see has no part in its
 * result, whatever it holds: infinities and NaN stay with those who see them.
 *
 * Conventions are rhizome_gdr.h's: plain pointers and sizes, row-major tensors
 * in caller-owned device memory, everything validated before the GPU is
 * touched, launches ordered on `stream` and asynchronous to the host, no
 * allocation, results deterministic (no atomics) and batch-invariant: a
 * sequence's results do not depend on what else is in the call.  Nothing is
 * kept between calls, so that a call can be captured into a graph; calls that
 * may run at the same time need a workspace each.  Strides are in elements.
 */
#ifndef RHIZOME_ATTENTION_H
#define RHIZOME_ATTENTION_H

#include "rhizome_gdr.h"

#ifdef __cplusplus
extern "C" {
#endif

/* How rotary frequencies are stretched for contexts beyond the trained length. */
typedef enum rhz_rope_scaling {
    RHZ_ROPE_PLAIN = 0,   /* theta^(-2i/dim) */
    RHZ_ROPE_LINEAR = 1,  /* every frequency divided by factor */
    RHZ_ROPE_BY_PARTS = 2 /* pairs that turn more than `fast` times over the trained length keep
                             their frequency, those below `slow` turns are divided by factor,
                             those between are mixed linearly in their turns; the rotated values
                             are multiplied by 0.1 ln(factor) + 1 */
} rhz_rope_scaling;

typedef struct rhz_rope_frequency_args {
    int32_t dim;     /* rotated channels, even, 2..1024 */
    int32_t scaling; /* rhz_rope_scaling */
    double theta;    /* base, > 1 */
    double factor;   /* >= 1; LINEAR and BY_PARTS */
    double trained_length; /* >= 1; BY_PARTS */
    double fast;     /* BY_PARTS: turns, fast > slow >= 0 */
    double slow;
} rhz_rope_frequency_args;

/* The table of a rotary embedding, on the host: turns[i], i < dim / 2, is pair
 * i's turns per position (its frequency over 2 pi), which the calls below take
 * in device memory, and *magnitude what its rotated values are multiplied by. */
rhz_status rhz_rope_frequencies(const rhz_rope_frequency_args* args, double* turns, float* magnitude);

/* Rotary positions (elementwise.rs has the reference's): the channels
 * [offset, offset + rot) of every head in pairs (a, b), turned by the angle
 * 2 pi turns[i] position:
 *     (a, b) := magnitude (a cos - b sin, a sin + b cos)
 * Pairs are (i, i + rot / 2), or (2 i, 2 i + 1) when interleaved.  inverse: by
 * the negative angle, which is the backward pass (grad_x from grad_y).  Angles
 * are reduced in 64 bits, so that every 32-bit position is exact to fp32.  The
 * other channels are copied; y may be x itself, with its strides (they are
 * left alone then), else the two ranges of memory do not overlap. */
typedef struct rhz_rope_args {
    int32_t tokens;      /* >= 0 */
    int32_t heads;       /* >= 1 */
    int32_t dim;         /* channels of a head */
    int32_t offset;      /* first rotated channel */
    int32_t rot;         /* rotated channels, even, 2..1024 */
    int32_t dtype;       /* rhz_dtype of x and y */
    int32_t interleaved; /* 0 or 1 */
    int32_t inverse;     /* 0 or 1 */
    float magnitude;     /* finite */
    int64_t x_token_stride, x_head_stride;
    int64_t y_token_stride, y_head_stride;
    const void* x;            /* [tokens, heads, dim] */
    const int32_t* positions; /* [tokens] */
    const double* turns;      /* [rot / 2] */
    void* y;
} rhz_rope_args;

rhz_status rhz_rope(const rhz_rope_args* args, void* stream);

/* New tokens into a paged cache (LatentCache, attention.rs:7-70).  Row of the
 * cache of position p of sequence b:
 *     page_table[b][p / page_size] * page_size + p % page_size
 * and it receives [c | r]: the latent, RMS-normalised and scaled where
 * norm_scale is given, and the rotary key, turned by p where turns are given.
 * The new tokens are the last ones of each sequence, positions
 * lengths[b] - n_b .. lengths[b] - 1.  A token whose position is negative or
 * beyond the table, or whose page is outside the cache, is left out; a page
 * that two tokens of one call write holds either's rows. */
typedef struct rhz_latent_append_args {
    int32_t batch;     /* sequences, >= 1 */
    int32_t seq_len;   /* dense: new tokens of every sequence;  packed: of all */
    int32_t d_c;       /* 1..4096 */
    int32_t d_r;       /* >= 0, even where turns are given, <= 1024 */
    int32_t page_size; /* >= 1 */
    int32_t num_pages; /* pages of the cache, >= 1 */
    int32_t max_pages; /* columns of the page table, >= 1 */
    int32_t dtype;     /* rhz_dtype of latent, k_rope and cache */
    int32_t interleaved;
    float magnitude;   /* finite */
    float eps;         /* >= 0 */
    int64_t latent_stride; /* of a token, >= 0 */
    int64_t k_rope_stride; /* likewise */
    const void* latent;        /* [tokens, d_c] */
    const void* k_rope;        /* [tokens, d_r], or NULL where d_r is 0 */
    const int32_t* cu_seqlens; /* device [batch + 1], or NULL (dense) */
    const int32_t* lengths;    /* [batch], the new tokens included */
    const int32_t* page_table; /* [batch, max_pages] */
    const double* turns;       /* [d_r / 2], or NULL */
    const float* norm_scale;   /* [d_c], or NULL */
    void* cache;               /* [num_pages, page_size, d_c + d_r] */
} rhz_latent_append_args;

rhz_status rhz_latent_append(const rhz_latent_append_args* args, void* stream);

/* Attention of the last `steps` positions of every sequence over its cached
 * latents, absorbed (mla_decode, attention.rs:226-300): query i of sequence b
 * sees positions 0 .. lengths[b] - steps + i.  Positions beyond the table, or
 * from 2^31 - 4097 on, and pages outside the cache hold no keys.  A sequence is
 * split over workgroups by its own length alone and joined in order.  bf16 on
 * bf16 matrix instructions with fp32 accumulation, the weights rounded to bf16
 * before they meet the latents; fp32 in fp32. */
typedef struct rhz_latent_decode_args {
    int32_t batch;     /* >= 1 */
    int32_t steps;     /* 1..RHZ_MULTISTEP_MAX */
    int32_t heads;     /* 1..1024 */
    int32_t d_c;       /* 1..512 */
    int32_t d_r;       /* 0..64 */
    int32_t page_size; /* >= 1 */
    int32_t num_pages; /* >= 1 */
    int32_t max_pages; /* >= 1 */
    int32_t dtype;     /* rhz_dtype of q, cache and o */
    float scale;       /* > 0, finite */
    const void* q;             /* [batch, steps, heads, d_c + d_r] */
    const void* cache;         /* [num_pages, page_size, d_c + d_r] */
    const int32_t* page_table; /* [batch, max_pages] */
    const int32_t* lengths;    /* [batch] */
    void* o;                   /* [batch, steps, heads, d_c] out */
    float* lse;                /* [batch, steps, heads] out: ln sum exp s; or NULL */
    void* workspace;           /* device scratch, 256-byte aligned */
    size_t workspace_bytes;
} rhz_latent_decode_args;

/* Bytes of workspace of the call (no pointer is read): for each sequence's
 * splits, as many as its page table has room for, an fp32 copy of its rows of o. */
rhz_status rhz_latent_decode_workspace_size(const rhz_latent_decode_args* args, size_t* bytes);

rhz_status rhz_latent_decode(const rhz_latent_decode_args* args, void* stream);

/* Attention over keys and values expanded from the latents (mla_prefill,
 * attention.rs:164-219): head h of key j is [k_j,h | k_rope_j].  Causal: the
 * last query of a sequence sees all of its keys, the one before it all but the
 * last, and so on, so that queries that continue a cached context bring its
 * keys along.  bf16 on bf16 matrix instructions with fp32 accumulation, the
 * weights rounded to bf16 before they meet the values; fp32 in fp32.  Tokens of
 * q, k, v and k_rope are at most 2^22 elements apart. */
typedef struct rhz_latent_prefill_args {
    int32_t batch;     /* sequences, >= 1 */
    int32_t seq_len;   /* queries: dense: of every sequence;  packed: of all */
    int32_t seq_len_k; /* keys, likewise */
    int32_t heads;     /* >= 1 */
    int32_t d_n;       /* >= 1 */
    int32_t d_r;       /* >= 0; d_n + d_r <= 192 */
    int32_t d_v;       /* 1..128 */
    int32_t dtype;     /* rhz_dtype of q, k, k_rope, v and o */
    int32_t causal;    /* 0 or 1 */
    float scale;       /* > 0, finite */
    int64_t q_token_stride, q_head_stride; /* all >= 0 */
    int64_t k_token_stride, k_head_stride;
    int64_t v_token_stride, v_head_stride;
    int64_t k_rope_stride;
    const void* q;      /* [queries, H, d_n + d_r] */
    const void* k;      /* [keys, H, d_n] */
    const void* v;      /* [keys, H, d_v] */
    const void* k_rope; /* [keys, d_r], or NULL where d_r is 0 */
    const int32_t* cu_seqlens;   /* device [batch + 1], or NULL (dense) */
    const int32_t* cu_seqlens_k; /* device [batch + 1], or NULL: cu_seqlens */
    void* o;            /* [queries, H, d_v] out */
    float* lse;         /* [queries, H] out, fp32: ln sum exp s */
} rhz_latent_prefill_args;

rhz_status rhz_latent_prefill(const rhz_latent_prefill_args* args, void* stream);

/* Backward pass of rhz_latent_prefill: `forward` is that call's arguments, its
 * o and lse read here as it wrote them, and grad_o (and grad_lse) the gradients
 * of its outputs.  The gradients are contiguous, of q's dtype; grad_k_rope is
 * summed over the heads in fp32 and rounded once.  In bf16 the weights, and their
 * gradients, are rounded to bf16 before the products that sum them.  Rows of a
 * pack outside every sequence are left as they were.  No output overlaps an
 * input, the workspace or another output. */
typedef struct rhz_latent_prefill_backward_args {
    rhz_latent_prefill_args forward;
    const void* grad_o;    /* [queries, H, d_v] */
    const float* grad_lse; /* [queries, H], or NULL for zeros */
    void* grad_q;          /* [queries, H, d_n + d_r] out */
    void* grad_k;          /* [keys, H, d_n] out */
    void* grad_v;          /* [keys, H, d_v] out */
    void* grad_k_rope;     /* [keys, d_r] out, or NULL where d_r is 0 */
    void* workspace;       /* device scratch, 256-byte aligned */
    size_t workspace_bytes;
} rhz_latent_prefill_backward_args;

/* Bytes of workspace: two floats for each query and head, and d_r for each key
 * and head (no pointer is read). */
rhz_status rhz_latent_prefill_backward_workspace_size(const rhz_latent_prefill_backward_args* args, size_t* bytes);

rhz_status rhz_latent_prefill_backward(const rhz_latent_prefill_backward_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* RHIZOME_ATTENTION_H */
