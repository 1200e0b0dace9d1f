/*
 * m2d_seq.h -- C ABI of the sequence operators next to the wavefront scan: linear attention with a decay per head,
 * group normalisation with an activation on channels-last tensors, clipping by the global norm of many tensors.
 *
 * Conventions are those of m2d_scan.h: device pointers, memory owned by the caller, asynchronous on `stream` (of the
 * current device), status codes, re-entrant, nothing kept between calls.  Strides are in elements.
 */
#ifndef M2D_SEQ_H
#define M2D_SEQ_H

#include "m2d_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- linear attention -------------------------------------------------------------------------------------------
 * Per sequence b and head h, with a state S (K,V):
 *     S_t = exp(g_t) S_{t-1} + k_t v_t^T,      o_t = scale * q_t^T S_t.
 * q and k have G heads, each shared by H / G neighbouring heads of v.  g = log_decay, fp32, at most 0 (-inf forgets
 * everything before the token; a positive value grows the state and is not checked for).
 *
 * State, its gradient and that of the decay are fp32 whatever the tensors' type.  bf16 tensors with K and V of up to 128 in whole
 * 16-byte pieces, 16-byte aligned and with such strides, take a form on the tensor cores (tcgen05), all others, and d_q and d_k
 * where the decay's gradient is wanted, one for any size and with more exact products.  With the former, products of values below 1e-17
 * or above 1e17 may lose bits or range where decays sum to about 65 in 128 tokens (pairs' weights are products of factors of up to 2^48).
 * Long sequences of few heads are cut into segments whose states the workspace holds; the workspace queries read the
 * sizes, G, dtype and, for the backward pass, whether d_log_decay is given, and need no other pointer.  B * H up to 2^24, T below
 * 2^31 - 2048.
 * A wait inside the tensor-core form that gives up makes its rows NaN, or the state that its CTA was to leave for other rows, and so
 * those; it shows in m2d_take_wait_failure().
 */
#define M2D_ATTN_MAX_DIM 256      /* K and V, each */

typedef struct m2d_attn_tensor {
    const void *data;              /* (B, T, heads, dim), neighbours along dim */
    int64_t batch, token, head;    /* strides of the other three */
} m2d_attn_tensor;

typedef struct m2d_attn_desc {
    uint32_t struct_bytes;         /* = sizeof(m2d_attn_desc) */
    int32_t dtype;                 /* m2d_dtype of q, k, v, o and their gradients */
    int32_t B, T, H, G, K, V;      /* G divides H */
    uint32_t flags;                /* 0, or the test hook */
    float scale;
    m2d_attn_tensor q, k, v;       /* the latter with H heads */
    const float *log_decay;        /* log_decay[b * g_batch + t * g_token + h * g_head] */
    int64_t g_batch, g_token, g_head;
    const int32_t *lengths;        /* (B) tokens of each sequence, clamped to 0 ... T, or NULL: T.  Rows behind a
                                      sequence's last are not read (they may hold anything); outputs there are zero */
    const float *state;            /* (B,H,K,V) dense: the state before the first token, or NULL: zero */
    float *state_out;              /* (B,H,K,V) dense: the state after the last one, or NULL       [fwd] */
    void *o;                       /* (B,T,H,V) dense                                              [fwd] */
    /* backward */
    m2d_attn_tensor d_o;           /* (B,T,H,V) */
    const float *d_state_out;      /* (B,H,K,V) dense, or NULL: zero */
    void *d_q, *d_k, *d_v;         /* (B,T,G,K), (B,T,G,K), (B,T,H,V) dense */
    float *d_log_decay;            /* (B,T,H) dense, or NULL: not wanted */
    float *d_state;                /* (B,H,K,V) dense, or NULL: not wanted */
    void *workspace;               /* scratch, 256-byte aligned */
    uint64_t workspace_bytes;
} m2d_attn_desc;

/*
 * Test hook, rejected with M2D_ERR_FLAGS unless the environment variable M2D_TEST_HOOKS is 1: in the first CTA of every launch of
 * the tcgen05 form that computes segments' states the first wait that does not succeed at once gives up.  Nothing faults or
 * hangs; the launch ends as after a wait that ran out.
 */
#define M2D_ATTN_TEST_GIVE_UP 0x100u

uint64_t m2d_attn_fwd_workspace(const m2d_attn_desc *desc);
uint64_t m2d_attn_bwd_workspace(const m2d_attn_desc *desc);
int m2d_attn_fwd(const m2d_attn_desc *desc, void *stream);
int m2d_attn_bwd(const m2d_attn_desc *desc, void *stream);

/*
 * One token for every sequence: T = 1, `state` is read and `state_out` written; they may be the same array.  Both are
 * (B,H,K,V) with dense (K,V) and the strides given here.  lengths and the backward's fields are ignored; no workspace.
 */
int m2d_attn_step(const m2d_attn_desc *desc, int64_t state_batch, int64_t state_head, void *stream);

/* ---- group normalisation ----------------------------------------------------------------------------------------
 * x (N,S,C), channels last: y = act((x - mean) * rstd * weight + bias), mean and variance over S and the C / groups
 * channels of a group.  Value and slope of act at an infinity are their limits.  C up to 2^29, N * groups below 2^31.  A slower form
 * takes tensors that are not 16-byte aligned or whose rows are not whole 16-byte pieces, images (S > 1) with rows of more than 4 KB,
 * and S = 1 with groups of more than 512 bytes or not of whole pieces.  The backward pass's workspace query reads whether d_weight is
 * given.
 */
typedef enum { M2D_ACT_NONE = 0, M2D_ACT_SILU = 1, M2D_ACT_GELU = 2 /* erf form */ } m2d_act;

typedef struct m2d_norm_desc {
    uint32_t struct_bytes;         /* = sizeof(m2d_norm_desc) */
    int32_t dtype;                 /* m2d_dtype of x, y, d_y, d_x */
    int64_t N, S;
    int32_t C, groups, act;
    int32_t params_f32;            /* weight and bias (and their gradients) are fp32, else of `dtype` */
    float eps;
    const void *x;                 /* dense */
    const void *weight, *bias;     /* (C), or NULL: one and zero */
    void *y;                       /*                                            [fwd] */
    float *stats;                  /* (N,groups,2): mean, rstd; written by fwd (NULL: not wanted), read by bwd */
    const void *d_y;               /*                                            [bwd] */
    void *d_x;
    void *d_weight, *d_bias;       /* (C), or both NULL */
    void *workspace;               /* scratch, 256-byte aligned */
    uint64_t workspace_bytes;
} m2d_norm_desc;

uint64_t m2d_norm_fwd_workspace(const m2d_norm_desc *desc);
uint64_t m2d_norm_bwd_workspace(const m2d_norm_desc *desc);
int m2d_norm_fwd(const m2d_norm_desc *desc, void *stream);
int m2d_norm_bwd(const m2d_norm_desc *desc, void *stream);

/* ---- clipping by the global norm --------------------------------------------------------------------------------
 * norm = sqrt(sum of squares over all tensors); every tensor is multiplied by min(1, max_norm / (norm + 1e-6)).  The
 * tensors must not overlap.  Squares are taken in fp32: a value beyond 1.8e19 makes the norm infinite.
 */
typedef struct m2d_clip_tensor {
    void *data;                    /* aligned to its elements */
    int64_t elements;              /* at least 0 */
    int32_t dtype;                 /* m2d_dtype */
} m2d_clip_tensor;

uint64_t m2d_clip_workspace(const m2d_clip_tensor *tensors, int32_t count);
int m2d_clip_grad_norm(const m2d_clip_tensor *tensors, int32_t count, float max_norm, float *norm, void *workspace,
                       uint64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* M2D_SEQ_H */
