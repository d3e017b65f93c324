/*
 * cgdr_recurrence.h -- C ABI of the token-by-token recurrences of linear
 * recurrent layers on B200 (sm_100a), next to the chunked gated delta rule
 * (cgdr_gdr.h):
 *
 *   cgdrRecurrentGatedDeltaRule       the gated delta rule for serving: few
 *                                     tokens a sequence, on a pool of states;
 *   cgdrGatedLinearRecurrence         the diagonal recurrence
 *                                     h_t = exp(g_t) h_{t-1} + x_t over whole
 *                                     sequences, and its backward pass;
 *   cgdrGatedLinearRecurrenceStep     the same for one token a row, on a
 *                                     pool of states.
 *
 * None of them needs a workspace, so each is one call: it checks its
 * arguments (no device work on failure) and enqueues one kernel on `stream`.
 * The stream's device must be current.  Tensors that may be NULL are named;
 * a tensor whose `data` is NULL counts as absent.
 *
 * Pools of states.  state_indices [B] (int32 or int64, contiguous) names the
 * row of the pool that each sequence owns.  A negative index marks a padded
 * row: no state is read or written for it and its outputs are zero.  An
 * index past the pool, or one that an earlier row of the call has already
 * named, is an error: that row is treated as padding and the device status
 * says so.  NULL: row b owns state b.  `device_status` (int32 on the device,
 * may be NULL) receives 0 or the CGDR_DEVICE_* bits below in stream order.
 */
#ifndef CGDR_RECURRENCE_H_
#define CGDR_RECURRENCE_H_

#include "cgdr_fwd_h.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CGDR_DEVICE_BAD_STATE_INDEX 0x4 /* an index past the pool, or named twice */

/* The gated delta rule, token by token.  Per sequence and value head, with
 * S [Dv, Dk] the sequence's state in the pool:
 *     S = S exp(g_t)
 *     S = S + beta_t (v_t - S k_t) k_t^T
 *     o_t = scale S q_t
 * Layout (TND, that of cgdrChunkGatedDeltaRule, whose finalState is a pool):
 *     query, key   [T, Nk, Dk]   bf16, fp16 or fp32
 *     value, out   [T, Nv, Dv]   the same type
 *     beta         [T, Nv]       the same type, or fp32
 *     g            [T, Nv]       fp32 per-token log gate (NULL: no gate)
 *     state        [S, Nv, Dv, Dk]  fp32 or bf16, updated in place
 *     actual_seq_lengths [B]     int32 tokens of each sequence, contiguous
 *                                (NULL: one token each, T == B)
 * with Nv a multiple of Nk and Dk <= 256.  Innermost dimensions are
 * contiguous, other strides free; widths and strides that are multiples of
 * 16 bytes are read in 16-byte pieces.  The state is held in fp32 from the
 * first token of a call to the last and rounded once to its own type when it
 * is written back.  scale <= 0 selects Dk ** -0.5.  Lengths that are negative
 * or exceed T are cut to what T holds and flagged BAD_VARLEN; rows of `out`
 * behind the last sequence are zero.  T == 0 or B == 0 does nothing. */
cgdrStatus cgdrRecurrentGatedDeltaRule(
    const cgdrTensor* query, const cgdrTensor* key, const cgdrTensor* value, const cgdrTensor* beta,
    const cgdrTensor* state, const cgdrTensor* actual_seq_lengths, const cgdrTensor* g,
    const cgdrTensor* state_indices, float scale, const cgdrTensor* out, int32_t* device_status, void* stream);

/* Tokens between two of the states that the forward pass saves for the
 * backward pass (chunk_states). */
#define CGDR_RECURRENCE_CHUNK 128

/* h_t = exp(g_t) h_{t-1} + x_t, channel by channel, out_t = h_t.
 *     x, out         [B, T, D]  bf16, fp16 or fp32
 *     g              [B, T, D]  log decay (<= 0; -inf forgets), x's type or fp32
 *     initial_state  [N, D]     fp32 (NULL: zeros)
 *     final_state    [N, D]     fp32 (may be NULL)
 *     cu_seqlens     [N+1]      int64 from 0, non-decreasing, contiguous
 *                               (NULL: every batch row is one sequence, N = B);
 *                               needs B == 1
 *     chunk_states   [B, ceil(T/128), D]  fp32, contiguous: the state
 *                               before each 128-token chunk (NULL unless a backward
 *                               pass follows)
 * T and D are below 2^30, N below 2^16, and rows less than 2^25 elements
 * apart.  Innermost dimensions are contiguous; rows of 16-byte multiples are
 * read by TMA, others by smaller copies.  Rows of `out` behind the last
 * sequence are zero.  The state is held in fp32; out is rounded once.  An empty sequence's final state is its initial
 * state. */
cgdrStatus cgdrGatedLinearRecurrence(
    const cgdrTensor* x, const cgdrTensor* g, const cgdrTensor* initial_state, const cgdrTensor* cu_seqlens,
    const cgdrTensor* out, const cgdrTensor* final_state, const cgdrTensor* chunk_states, void* stream);

/* The gradients of the above.  d_out [B, T, D] has x's type, d_final_state
 * [N, D] is fp32; either may be NULL (zero), not both.
 *     dh_t = d_out_t + exp(g_{t+1}) dh_{t+1}    (d_final_state joins the last)
 *     dx_t = dh_t,  dg_t = dh_t exp(g_t) h_{t-1},  d_initial_state = exp(g_1) dh_1
 * dx has x's type, dg g's, d_initial_state is fp32; each may be NULL.  h is
 * recomputed in fp32 from x, g and chunk_states. */
cgdrStatus cgdrGatedLinearRecurrenceBackward(
    const cgdrTensor* x, const cgdrTensor* g, const cgdrTensor* initial_state, const cgdrTensor* cu_seqlens,
    const cgdrTensor* chunk_states, const cgdrTensor* d_out, const cgdrTensor* d_final_state, const cgdrTensor* dx,
    const cgdrTensor* dg, const cgdrTensor* d_initial_state, void* stream);

/* One token a row on a pool of states: state[i_b] = exp(g_b) state[i_b] + x_b,
 * out_b = state[i_b].  x, g, out [B, D] (types as above), state [S, D] fp32,
 * updated in place. */
cgdrStatus cgdrGatedLinearRecurrenceStep(
    const cgdrTensor* x, const cgdrTensor* g, const cgdrTensor* state, const cgdrTensor* state_indices,
    const cgdrTensor* out, int32_t* device_status, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CGDR_RECURRENCE_H_ */
