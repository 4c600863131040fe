/*
 * d2p_amd_encoder.h -- C ABI of the sequence-encoder operators on MI355X (gfx950): the
 * attention layer whose embeddings a caller multiplies into the score matrices that the
 * alignment entry points of d2p_amd.h take.  No counterpart in the reference, whose callers
 * bring finished scores.
 *
 * The conventions are those of d2p_amd.h: device pointers to caller-owned buffers, scratch
 * memory from the caller (*_workspace_bytes), kernels enqueued on `stream` without
 * synchronising, 0 on success and non-zero on failure with the message in d2p_last_error().
 * Results do not depend on the order in which workgroups run: no entry point adds with
 * floating-point atomics.
 */
#ifndef D2P_AMD_ENCODER_H
#define D2P_AMD_ENCODER_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations. */
#define D2P_FLOAT32 0
#define D2P_FLOAT16 1
#define D2P_BFLOAT16 2

/* Strides of a [batch, row, head, feature] tensor, in elements; features are adjacent.
 * Each is a multiple of 16 bytes' worth of elements (a base pointer is a multiple of 16
 * bytes too), row >= D where there is more than one row, and 128 rows span less than 2 GiB. */
typedef struct {
    long long batch, row, head;
} d2p_strides;

/* One attention call.  For batch element b, query head h (reading key head h * Hkv / Hq),
 * query i < nq and key j < nk, (nq, nk) = lengths[b] or (Lq, Lk):
 *   at_i = i + nk - nq where causal (the last query sits on the last key), i otherwise
 *   s_ij = scale q_i . k_j + bias[buckets[clip(j - at_i, -R, R) + R], h]
 *   p_i  = softmax of s_i over j (causal: over j <= at_i); zeros if there is no such j
 *   o_i  = sum_j p_ij d_ij v_j,  d_ij = 0 or 256 / (256 - drop)
 * Rows i >= nq of the result and of every gradient are zero.  Nothing at or past nq or nk
 * is used, whatever it holds, nor the bias of a distance that only such rows have.
 * Dropout: byte j % 4 of word i % 4 of Philox4x32 with 7 rounds (J. Salmon, M. Moraes,
 * R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) on the counter
 * (j / 4, i / 4, b Hq + h, 0) and the key (low, high word of the seed) keeps the pair if it
 * is at least drop.  Nothing of the mask is stored: the backward pass draws it again. */
typedef struct {
    int dtype;                 /* of q, k, v, out and their gradients */
    int B, Lq, Lk, Hq, Hkv;    /* Hq a multiple of Hkv */
    int D;                     /* features of a head: a multiple of 8, 8 to 128 */
    d2p_strides q, k, v, grad; /* grad: of the result's gradient (backward only) */
    const int* lengths;        /* int32 [B, 2] on the device, or null for (Lq, Lk) each; the
                                  outputs of an element whose lengths are not within 0 and
                                  (Lq, Lk) are NaN */
    int causal;
    float scale;               /* positive */
    const void* bias;          /* [num_buckets, Hq] or null for none */
    int bias_dtype;            /* D2P_FLOAT32 or dtype */
    int num_buckets;
    const int* buckets;        /* int32 [2 R + 1] on the device: the bucket of each clipped
                                  distance; one outside [0, num_buckets) makes its bias NaN */
    int max_distance;          /* R, 0 to 1024 */
    int drop;                  /* probability of dropping a pair in 256ths, 0 to 255 */
    unsigned long long seed;   /* the generator's key ... */
    const long long* seed_ptr; /* ... or, if not null, where it lies on the device */
} d2p_attention_params;

/* Workspace bytes of d2p_attention_forward (0: none needed). */
size_t d2p_attention_workspace_bytes(const d2p_attention_params* p);

/* out [B, Lq, Hq, D] (contiguous) and stats [2, B, Hq, Lq] float32: for each row a value m
 * near the largest s_ij log2 e (-inf for a row without keys), and log2 of the sum of
 * 2^(s_ij log2 e - m).  Two numbers, so that a row whose every bias is the type's lowest
 * value keeps its sum. */
int d2p_attention_forward(const d2p_attention_params* p, const void* q, const void* k,
                          const void* v, void* out, float* stats, void* workspace,
                          size_t workspace_bytes, void* stream);

/* Workspace bytes of d2p_attention_backward. */
size_t d2p_attention_backward_workspace_bytes(const d2p_attention_params* p);

/* Gradients from grad = dL/dout (strides p->grad), the forward's inputs, out and stats; the
 * probabilities are computed again.  dq [B, Lq, Hq, D], dk and dv [B, Lk, Hkv, D], all
 * contiguous; dbias [num_buckets, Hq] of bias_dtype, or null if it is not wanted. */
int d2p_attention_backward(const d2p_attention_params* p, const void* grad, const void* q,
                           const void* k, const void* v, const void* out, const float* stats,
                           void* dq, void* dk, void* dv, void* dbias, void* workspace,
                           size_t workspace_bytes, void* stream);

/* One call of the norm and rotation of queries and keys.  For each row x of D features
 *   n = w x / sqrt(mean(x^2) + eps)
 * and the first R features of n turn by the angles t of their position: the pair (a, c) is
 * (m, m + R / 2), or (2 m, 2 m + 1) where interleaved, m < R / 2, and
 *   y_a = n_a cos t_m - n_c sin t_m,  y_c = n_c cos t_m + n_a sin t_m.
 * The features past R are n. */
typedef struct {
    int dtype;                  /* of q, k, their results and gradients */
    int B, L, Hq, Hkv;          /* Hkv may be 0 */
    int D, R;                   /* D as for attention; R even, 0 to D */
    d2p_strides q, k;           /* of the inputs; last-feature stride 1, no alignment asked */
    d2p_strides gq, gk;         /* of the results' gradients (backward only) */
    const float *q_weight, *k_weight;   /* [D] float32 each, or null for ones */
    const float *cos, *sin;     /* [table_rows, R / 2] float32 */
    long long table_rows;
    const int* positions;       /* int32 [B, L] on the device, or null for 0 .. L - 1; the rows
                                   of a position outside the table are NaN */
    float eps;
    int interleaved;
} d2p_qk_norm_rope_params;

/* q_out [B, L, Hq, D], k_out [B, L, Hkv, D], contiguous. */
int d2p_qk_norm_rope(const d2p_qk_norm_rope_params* p, const void* q, const void* k,
                     void* q_out, void* k_out, void* stream);

/* Workspace bytes of d2p_qk_norm_rope_backward. */
size_t d2p_qk_norm_rope_backward_workspace_bytes(const d2p_qk_norm_rope_params* p);

/* dq, dk contiguous as q_out, k_out; dq_weight, dk_weight [D] float32 (null: not wanted). */
int d2p_qk_norm_rope_backward(const d2p_qk_norm_rope_params* p, const void* gq, const void* gk,
                              const void* q, const void* k, void* dq, void* dk,
                              float* dq_weight, float* dk_weight, void* workspace,
                              size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* D2P_AMD_ENCODER_H */
