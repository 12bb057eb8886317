/*
 * cc1d_gdr.h — C ABI of the gated delta rule kernels of libcc1d.so (B200, sm_100a).
 *
 * Same rules as cc1d.h: plain parameter blocks, element strides, launches on the current device
 * and the given stream, no allocation, no synchronisation, int status codes.
 */
#ifndef CC1D_GDR_H_
#define CC1D_GDR_H_

#include "cc1d.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------------
 * Gated delta rule: the sequence mixer whose q, k and v the convolution produces (no
 * counterpart in the reference).  Per sequence and value head, with a state S of
 * (dim_k, dim_v) fp32 and a_t = exp(g_t):
 *
 *   S_t = a_t S_{t-1} + k_t (beta_t (v_t - a_t S_{t-1}^T k_t))^T      o_t = scale * S_t^T q_t
 *
 * Value head h uses key head h / (heads_v / heads_k).  g = -inf forgets the state.  g is meant to be
 * at most 0: where positive ones add up to more than 88 over 64 tokens, e^sum leaves fp32 and the
 * tokens behind are NaN.  A token whose values are infinite or NaN, or whose products leave fp32, gives
 * NaN to the outputs of itself and of those behind it in its sequence and head (in the dim_v columns it
 * touches), to none before.  In the backward a v that is not finite gives NaN to the gradients of q, k, g
 * and beta from its token on, to none before, and not to dv and dinitial_states; any other value that is
 * not finite may give NaN to all gradients of its sequence and head.
 * All sums and the state are fp32.  The tensor-core products split their fp32 factors into bf16
 * pieces: three (24 bits) of the state, of every factor of fp32 inputs and in the backward; two
 * (2^-17) of the chunk's U, P and of the correction (T - I) R in the forward of 16-bit types, whose
 * output is rounded to 16 bits (its last state is then off by up to 2e-6, of fp32 inputs by 2e-7).
 *
 * Sequences: `batch` rows of `seqlen` tokens, or (cu_seqlens != NULL) batch == 1 and nseq packed
 * sequences, sequence s owning tokens [cu_seqlens[s], cu_seqlens[s+1]) of the seqlen tokens;
 * tokens before cu_seqlens[0] and at or after cu_seqlens[nseq] get zero outputs and gradients.
 * cu_seqlens is non-decreasing and its last entry is at most seqlen (entries outside [0, seqlen] are
 * clamped).
 * State rows: r = state_indices ? state_indices[n] : n for sequence (row) n.  A row at or
 * above state_rows counts as a negative index.  No two sequences may name the same row of
 * final_states.
 * A sequence starts from initial_states[r] where that is given and has_initial_state is NULL or
 * has_initial_state[n] != 0, else from zeros; final_states[r], when given, gets its last state
 * and may alias initial_states.  With a negative index it starts from zeros and stores nothing
 * (cc1d_gdr_update: a padded row: zero output, no state touched).
 * A state row is [heads_v][dim_k][dim_v], the last two dense; pointers 16-byte aligned, strides
 * multiples of 4.
 * ------------------------------------------------------------------------- */
typedef struct cc1d_gdr_params {
    int32_t itype;            /* cc1d_dtype of q, k, v, out                     */
    int32_t gtype, btype;     /* cc1d_dtype of g, of beta                       */
    float scale;
    int64_t batch, seqlen, nseq;
    int64_t heads_k, heads_v, dim_k, dim_v;

    const void *q;            /* (batch, seqlen, heads_k, dim_k), dim stride 1  */
    int64_t q_batch_stride, q_l_stride, q_h_stride;
    const void *k;
    int64_t k_batch_stride, k_l_stride, k_h_stride;
    const void *v;            /* (batch, seqlen, heads_v, dim_v), dim stride 1  */
    int64_t v_batch_stride, v_l_stride, v_h_stride;
    const void *g;            /* (batch, seqlen, heads_v)                       */
    int64_t g_batch_stride, g_l_stride, g_h_stride;
    const void *beta;         /* (batch, seqlen, heads_v)                       */
    int64_t beta_batch_stride, beta_l_stride, beta_h_stride;
    void *out;                /* (batch, seqlen, heads_v, dim_v), dim stride 1  */
    int64_t out_batch_stride, out_l_stride, out_h_stride;

    const int32_t *cu_seqlens;          /* (nseq + 1,) or NULL                  */
    const int32_t *state_indices;       /* (sequences,) or NULL                 */
    const uint8_t *has_initial_state;   /* (sequences,) 0/1 or NULL             */
    int64_t state_rows;                 /* rows of initial_states and final_states */
    const float *initial_states;
    int64_t initial_states_batch_stride, initial_states_h_stride;
    float *final_states;
    int64_t final_states_batch_stride, final_states_h_stride;

    void *workspace;          /* cc1d_gdr_fwd: >= cc1d_gdr_fwd_workspace_bytes(), 16-byte aligned; NULL when that is 0 */
    size_t workspace_bytes;
} cc1d_gdr_params;

/* Forward over whole sequences, in chunks of 64 tokens.  q, k, v, out: 16-byte aligned, strides
 * of 16-byte multiples.  Nothing in the workspace has to start at zero. */
size_t cc1d_gdr_fwd_workspace_bytes(const cc1d_gdr_params *p);
int cc1d_gdr_fwd(const cc1d_gdr_params *p, cc1d_stream_t stream);

/* Gradients of the forward.  `fwd` describes the forward call (out, final_states and its
 * workspace are not read); dout has the shape of out, with strides; dfinal_states, (sequences,
 * heads_v, dim_k, dim_v) dense, or NULL.  All gradients are dense in the shapes of what they
 * belong to, dq, dk, dv in itype, dg in gtype, dbeta in btype; dinitial_states is (sequences,
 * heads_v, dim_k, dim_v) fp32 or NULL.  dq and dk are summed over the value heads of a key head
 * in a fixed order: results are bitwise reproducible. */
typedef struct cc1d_gdr_bwd_params {
    cc1d_gdr_params fwd;
    const void *dout;
    int64_t dout_batch_stride, dout_l_stride, dout_h_stride;
    const float *dfinal_states;
    void *dq, *dk, *dv, *dg, *dbeta;
    float *dinitial_states;
    void *workspace;          /* >= cc1d_gdr_bwd_workspace_bytes(), 16-byte aligned */
    size_t workspace_bytes;
} cc1d_gdr_bwd_params;

size_t cc1d_gdr_bwd_workspace_bytes(const cc1d_gdr_bwd_params *p);
int cc1d_gdr_bwd(const cc1d_gdr_bwd_params *p, cc1d_stream_t stream);

/* Decode step: `seqlen` tokens (one, or a few drafted ones) for each of `batch` rows, the state
 * row read from and written back to final_states in place.  initial_states, cu_seqlens, nseq and
 * has_initial_state are not read.  Any strides of q, k, v, g, beta, out but the last. */
int cc1d_gdr_update(const cc1d_gdr_params *p, cc1d_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* CC1D_GDR_H_ */
