/*
 * d2p_amd_training.h -- C ABI of what stands around the attention layer in the training of a
 * sequence encoder on MI355X (gfx950): token embedding, the residual stream's norms, gradient
 * norm and clipping.  No counterpart in the reference, whose callers bring finished scores.
 *
 * The conventions are those of d2p_amd.h and d2p_amd_encoder.h (element types D2P_FLOAT32,
 * D2P_FLOAT16, D2P_BFLOAT16): device pointers to caller-owned buffers, scratch memory from the
 * caller (*_workspace_bytes), kernels enqueued on `stream` without synchronising, 0 on success
 * and non-zero on failure with the message in d2p_last_error().  Base pointers are aligned to
 * their element, workspaces and a residual norm's statistics are aligned to 16 bytes.  Results do
 * not depend on the order in which workgroups run.
 */
#ifndef D2P_AMD_TRAINING_H
#define D2P_AMD_TRAINING_H

#include "d2p_amd_encoder.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Strides of a [batch, row, feature] tensor that is only read, in elements; features are
 * adjacent. */
typedef struct {
    long long batch, row;
} d2p_row_strides;

/* ---- token embedding ------------------------------------------------------------------
 * For token t = tokens[b, l] of the first lengths[b] of each sequence:
 *   out[b, l] = scale * weight[t],        zeros for t = padding and past lengths[b]
 *   dweight[v] = scale * sum of grad[b, l] over all b, l whose token is v (zeros: none)
 * A token outside [0, V) comes back NaN, as do all rows of a sequence whose length is not
 * within 0 and L; neither adds to dweight. */
typedef struct {
    int weight_dtype;           /* of weight and dweight */
    int dtype;                  /* of out and grad: weight_dtype, or 16 bits beside float32 */
    int B, L;                   /* B * L below 2^31 */
    int V, D;                   /* V from 1, below 2^31 - 1; D from 8 to 2^20 */
    const void* tokens;         /* [B, L] contiguous, on the device */
    int token_bytes;            /* 4 or 8: int32 or int64 */
    const int* lengths;         /* int32 [B] on the device, or null for L each */
    long long padding;          /* a token, or -1 for none */
    float scale;
    d2p_row_strides grad;       /* backward only */
} d2p_token_embedding_params;

/* weight [V, D] and out [B, L, D], contiguous. */
int d2p_token_embedding(const d2p_token_embedding_params* p, const void* weight, void* out,
                        void* stream);

/* Workspace bytes of d2p_token_embedding_backward. */
size_t d2p_token_embedding_backward_workspace_bytes(const d2p_token_embedding_params* p);

/* dweight [V, D] contiguous, written whole; sums in float32 in a fixed order. */
int d2p_token_embedding_backward(const d2p_token_embedding_params* p, const void* grad,
                                 void* dweight, void* workspace, size_t workspace_bytes,
                                 void* stream);

/* ---- residual stream ------------------------------------------------------------------
 * Between two blocks of a residual network, for each row of D features, y being the first
 * block's output and x the stream that went round it:
 *   z = N(y; post_weight, post_bias)      (y itself for D2P_NORM_NONE)
 *   h = residual_scale * x + scale * gate * z
 *   n = N(h; weight, bias)                the next block's input
 *   N(v; w, b) = w v / sqrt(mean(v^2) + eps) + b                       (D2P_NORM_RMS)
 *              = w (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps) + b   (D2P_NORM_LAYER)
 * n is formed from h before h is rounded to its type.  Without y: h = x, and only n is
 * written.  All is computed in float32: a row whose sum of squares (a layer norm's: around its
 * mean) is infinite there has N = b. */
#define D2P_NORM_NONE 0
#define D2P_NORM_RMS 1
#define D2P_NORM_LAYER 2

/* What a gate's number is for: [D], [B, 1, D] or [B, L, D]. */
#define D2P_GATE_NONE 0
#define D2P_GATE_FEATURE 1
#define D2P_GATE_SEQUENCE 2
#define D2P_GATE_TOKEN 3

/* A learned vector [D], contiguous, or null. */
typedef struct {
    const void* data;
    int dtype;
} d2p_vector;

typedef struct {
    int dtype;                  /* of x, h and their gradients */
    int block_dtype;            /* of y, n and their gradients: dtype, or 16 bits beside float32 */
    int B, L, D;                /* D from 8 to 8192 */
    int with_y;                 /* 0: no block yet */
    d2p_row_strides x, y;
    d2p_row_strides dh, dn;     /* of the results' gradients (backward only) */
    int norm, post_norm;        /* D2P_NORM_* */
    d2p_vector weight, bias, post_weight, post_bias;    /* null: ones, zeros */
    int gate_kind;              /* D2P_GATE_* */
    const void* gate;
    int gate_dtype;
    d2p_row_strides gate_strides;   /* the ones of what the gate is for */
    float scale, residual_scale, eps;
} d2p_residual_norm_params;

/* h (null without y) and n (null for D2P_NORM_NONE) [B, L, D], contiguous; stats [B, L, 4]
 * float32, for the backward pass, or null: mean and 1 / sqrt(...) of n's norm and of z's. */
int d2p_residual_norm(const d2p_residual_norm_params* p, const void* x, const void* y, void* h,
                      void* n, float* stats, void* stream);

/* Workspace bytes of d2p_residual_norm_backward. */
size_t d2p_residual_norm_backward_workspace_bytes(const d2p_residual_norm_params* p);

/* Gradients from dh = dL/dh and dn = dL/dn (one may be null: zeros).  stream_in, null where n has
 * no norm or no gradient: h as the forward pass wrote it if it is float32; x, with its strides, if
 * it has 16 bits (h is formed from x and y again then, unrounded) or if there is no y.  y: null
 * where it is needed for neither that, nor its own norm, nor the gate's gradient.  dx, dy [B, L, D]
 * and dgate (of the gate's sizes), contiguous, in their inputs' types; dweight .. dpost_bias [D] in
 * theirs.  Null: not wanted; dx, and dy where there is a y, always are, but dy may be null where it
 * equals dx (no gate, no post_norm, equal scales and types). */
int d2p_residual_norm_backward(const d2p_residual_norm_params* p, const void* dh, const void* dn,
                               const void* stream_in, const void* y, const float* stats, void* dx,
                               void* dy, void* dgate, void* dweight, void* dbias,
                               void* dpost_weight, void* dpost_bias, void* workspace,
                               size_t workspace_bytes, void* stream);

/* ---- gradient norm and clipping -------------------------------------------------------- */

/* One of the tensors that a norm is taken over: n adjacent numbers.  The list is read before
 * the call returns. */
typedef struct {
    const void* src;
    void* dst;                  /* d2p_clip_by_norm only; src itself, or apart from every src and
                                   every other dst */
    long long n;
    int dtype;
} d2p_tensor;

/* Workspace bytes of both for `count` tensors. */
size_t d2p_global_norm_workspace_bytes(int count);

/* norm = sqrt(sum of the squares of all numbers of all tensors), summed in float64. */
int d2p_global_norm(const d2p_tensor* tensors, int count, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream);

/* dst = c src, c = 1 where norm <= max_norm, max_norm / norm otherwise (NaN for a NaN, 0 for an
 * infinite norm, whose infinities then become NaN).  max_norm is not negative. */
int d2p_clip_by_norm(const d2p_tensor* tensors, int count, double max_norm, float* norm,
                     void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* D2P_AMD_TRAINING_H */
