/*
 * dynconv_layer.h -- C ABI of the operators that stand behind the short
 * convolutions in a layer (libdynconv.so, with dynconv.h): linear attention
 * with a decay for each head, in its form for whole sequences and its form for
 * single tokens; the gated delta rule in both forms; the group norm of their
 * heads with an activation or a gate; the norms around a block with its gate,
 * its residual scale and the residual sum; and the lowrank convolutions' form
 * for single tokens.  The reference has none of these.
 *
 * Conventions are those of dynconv.h (device pointers, int64 sizes, a status
 * of DC_OK or below, no allocation, no synchronisation, kernels only, on
 * `stream` of the current device, deterministic results), and:
 *   - strides are host arrays of int64 in elements; the last axis is contiguous;
 *   - states and decays are float32 whatever `dtype` is; sums, states and norms
 *     are held in float32.
 */
#ifndef DYNCONV_LAYER_H_
#define DYNCONV_LAYER_H_

#include <stdint.h>

#include "dynconv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest head dimensions of linear attention. */
#define DC_LA_MAX_DIM 256

/* Linear attention with a decay for each head: with g = exp(log_decay[h]),
 *     S_t = g S_{t-1} + k_t^T v_t,    o_t = scale * q_t S_t
 * from S_{-1} = initial_state (NULL: zero).
 *   q, k [B, H, T, K], v, o [B, H, T, V] with strides (batch, head, row) each;
 *   log_decay [H], initial_state, final_state [B, H, K, V] float32 (final_state
 *   NULL: not wanted; it may be initial_state);
 *   lengths [B] int32 or NULL: sequence b has lengths[b] (clamped to 0 .. T)
 *   tokens; rows past them are not used, whatever they hold, their outputs are
 *   zero and the state is the one after the last token.
 * T may be 0.  Both calls need a workspace of dc_linear_attention_ws_bytes
 * bytes (0: none), 16-byte aligned; bwd: 0 the forward, 1 the backward, 2 the
 * backward that is given the forward's workspace. */
int64_t dc_linear_attention_ws_bytes(int64_t B, int64_t H, int64_t T, int64_t K, int64_t V, int dtype, int bwd);
int dc_linear_attention_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                            const void* v, const int64_t* v_strides, const float* log_decay,
                            const float* initial_state, const int32_t* lengths, void* o, const int64_t* o_strides,
                            float* final_state, void* workspace, int64_t ws_bytes, int64_t B, int64_t H, int64_t T,
                            int64_t K, int64_t V, float scale, int dtype, void* stream);

/* Gradients of dc_linear_attention_fwd: dq, dk, dv from d_o [B, H, T, V] and
 * d_final_state [B, H, K, V] (NULL: zero), and d_initial_state (NULL: not
 * wanted).  Rows past a sequence's length get zero.  fwd_workspace is NULL or the
 * workspace of the forward of the same inputs, as that call left it: it holds
 * the states that the backward would form again (trusted, not checked). */
int dc_linear_attention_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                            const void* v, const int64_t* v_strides, const float* log_decay,
                            const float* initial_state, const int32_t* lengths, const void* d_o,
                            const int64_t* do_strides, const float* d_final_state, void* dq,
                            const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                            const int64_t* dv_strides, float* d_initial_state, const void* fwd_workspace,
                            void* workspace, int64_t ws_bytes, int64_t B, int64_t H, int64_t T, int64_t K, int64_t V, float scale, int dtype,
                            void* stream);

/* One token of each of B sequences: q, k [B, H, K], v [B, H, V] with strides
 * (batch, head), o [B, H, V] contiguous; state [slots, H, K, V] float32,
 * updated in place.  slot_ids [B] int32 names the row of each sequence (NULL:
 * sequence b has row b, B <= slots); an id outside 0 .. slots-1 takes no part:
 * its o is zero and no state changes.  Ids inside are distinct. */
int dc_linear_attention_step(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                             const void* v, const int64_t* v_strides, const float* log_decay, float* state,
                             const int32_t* slot_ids, void* o, int64_t B, int64_t H, int64_t K, int64_t V,
                             int64_t slots, float scale, int dtype, void* stream);

/* Flags of the gated delta rule. */
typedef enum dc_delta_flags {
  DC_DELTA_NORMALIZE = 1, /* the rows of q and k are divided by sqrt(|row|^2 + eps) */
  DC_DELTA_PRECISE = 2,   /* bf16, fp16: products as good as float32's, for the results that are float32 */
  DC_DELTA_KEEP = 4       /* a backward follows, with the forward's workspace: the forward keeps its states for it there where
                             they take no more than twice the memory of q, k, v and o */
} dc_delta_flags;

/* The gated delta rule: with a = exp(log_decay_t), b = beta_t, for each sequence and head,
 *     S' = a S_{t-1},   u = b (v_t - k_t S'),   S_t = S' + k_t^T u,   o_t = scale * q_t S_t
 * from S_{-1} = initial_state (NULL: zero).
 *   q, k [B, Hk, T, K], v, o [B, H, T, V], log_decay, beta [B, H, T], with strides (batch, head, row) each, those of
 *   log_decay and beta for the whole of their axes; Hk divides H, and head h reads q and k of head h / (H / Hk);
 *   log_decay <= 0 (-inf forgets at once), beta and log_decay in gate_dtype: dtype or float32;
 *   initial_state, final_state, lengths as in dc_linear_attention_fwd, but the two states are not the same memory
 *   (refused), which segments of a sequence read and write side by side.
 * B * H * T is at most 2^40.  Values are finite: one that is not reaches its head's outputs from the start of its chunk of
 * up to 64 tokens on (rows past the lengths may hold anything).  T may be 0.  Both calls need a workspace of
 * dc_delta_rule_ws_bytes bytes (0: none), 16-byte aligned; bwd: 0 the forward, 1 the backward, 2 the backward that is given
 * the forward's workspace (of the same flags). */
int64_t dc_delta_rule_ws_bytes(int64_t B, int64_t Hk, int64_t H, int64_t T, int64_t K, int64_t V, int dtype, int flags,
                               int bwd);
int dc_delta_rule_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                      const int64_t* v_strides, const void* log_decay, const int64_t* log_decay_strides,
                      const void* beta, const int64_t* beta_strides, const float* initial_state, const int32_t* lengths,
                      void* o, const int64_t* o_strides, float* final_state, void* workspace, int64_t ws_bytes,
                      int64_t B, int64_t Hk, int64_t H, int64_t T, int64_t K, int64_t V, float scale, float eps,
                      int dtype, int gate_dtype, int flags, void* stream);

/* Gradients of dc_delta_rule_fwd: dq, dk, dv, dlog_decay, dbeta from d_o and d_final_state (NULL: zero), and
 * d_initial_state (NULL: not wanted; not d_final_state's memory).  Rows past a sequence's length get zero.  fwd_workspace
 * is NULL or the workspace of the forward of the same inputs, as that call left it (trusted, not checked). */
int dc_delta_rule_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                      const int64_t* v_strides, const void* log_decay, const int64_t* log_decay_strides,
                      const void* beta, const int64_t* beta_strides, const float* initial_state, const int32_t* lengths,
                      const void* d_o, const int64_t* do_strides, const float* d_final_state, void* dq,
                      const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                      const int64_t* dv_strides, void* dlog_decay, const int64_t* dlog_decay_strides, void* dbeta,
                      const int64_t* dbeta_strides, float* d_initial_state, const void* fwd_workspace, void* workspace,
                      int64_t ws_bytes, int64_t B, int64_t Hk, int64_t H, int64_t T, int64_t K, int64_t V, float scale,
                      float eps, int dtype, int gate_dtype, int flags, void* stream);

/* One token of each of B sequences: q, k [B, Hk, K], v [B, H, V], log_decay, beta [B, H] with strides (batch, head),
 * o [B, H, V] contiguous; state and slot_ids as in dc_linear_attention_step. */
int dc_delta_rule_step(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                       const int64_t* v_strides, const void* log_decay, const int64_t* log_decay_strides,
                       const void* beta, const int64_t* beta_strides, float* state, const int32_t* slot_ids, void* o,
                       int64_t B, int64_t Hk, int64_t H, int64_t K, int64_t V, int64_t slots, float scale, float eps,
                       int dtype, int gate_dtype, int flags, void* stream);

/* Activations of dc_group_norm_fwd / _bwd (the first two) and of dc_residual_norm_fwd / _bwd. */
typedef enum dc_activation { DC_ACT_NONE = 0, DC_ACT_SILU = 1, DC_ACT_SIGMOID = 2 } dc_activation;

/* Group norm over the channels of each row: x, y, gate [M, D] contiguous, in
 * `groups` groups of D / groups neighbouring channels,
 *     u = (x - mean) / sqrt(var + eps) * weight + bias,
 *     y = u * act(gate)  with a gate,   y = act(u)  without (gate NULL)
 * (biased variance).  weight, bias [D] or NULL (1, 0), both in param_dtype:
 * dtype or float32. */
int dc_group_norm_fwd(const void* x, const void* weight, const void* bias, const void* gate, void* y, int64_t M,
                      int64_t D, int64_t groups, float eps, int activation, int dtype, int param_dtype, void* stream);

/* dx, dgate (with a gate), dweight, dbias (NULL: not wanted) from dy. */
int64_t dc_group_norm_bwd_ws_bytes(int64_t M, int64_t D, int64_t groups, int dtype);
int dc_group_norm_bwd(const void* x, const void* weight, const void* bias, const void* gate, const void* dy, void* dx,
                      void* dgate, void* dweight, void* dbias, void* workspace, int64_t ws_bytes, int64_t M, int64_t D,
                      int64_t groups, float eps, int activation, int dtype, int param_dtype, void* stream);

/* Largest rows of the residual norm. */
#define DC_RN_MAX_DIM 8192

/* The norms around a block, its gate, its residual scale and the residual sum, row by row of [M, D]:
 *     u = branch / sqrt(mean(branch^2) + eps) * branch_weight,    h = x + constant * scale * act(gate) * u,
 *     y = h / sqrt(mean(h^2) + eps) * weight
 * x, h contiguous in x_dtype: dtype or float32 (h is rounded to it before its norm); branch, gate (or NULL: no factor),
 * y contiguous in dtype; weight, branch_weight, scale [D] or NULL (1), all in param_dtype: dtype or float32. */
int dc_residual_norm_fwd(const void* x, const void* branch, const void* weight, const void* branch_weight,
                         const void* gate, const void* scale, void* y, void* h, int64_t M, int64_t D, float constant,
                         float eps, int activation, int dtype, int x_dtype, int param_dtype, void* stream);

/* dx (in x_dtype), dbranch, dgate (with a gate), dweight, dbranch_weight, dscale (NULL: not wanted) from dy and dh
 * (either NULL: zero) and the forward's h. */
int64_t dc_residual_norm_bwd_ws_bytes(int64_t M, int64_t D, int dtype);
int dc_residual_norm_bwd(const void* h, const void* branch, const void* weight, const void* branch_weight,
                         const void* gate, const void* scale, const void* dy, const void* dh, void* dx, void* dbranch,
                         void* dgate, void* dweight, void* dbranch_weight, void* dscale, void* workspace,
                         int64_t ws_bytes, int64_t M, int64_t D, float constant, float eps, int activation, int dtype,
                         int x_dtype, int param_dtype, void* stream);

/* One token of each of N sequences through G lowrank convolutions of one shape
 * (the single-token form of dc_lowrank_fwd_grouped): with x_0 = x[n] and x_w
 * the token w steps back, from `state` (its last row is w = 1),
 *     y[g] = sum_w (z[g] U[g][:, w] + static_w[g][w]) * x_w   (+ x_0 if residual)
 *   x [N, G*D] with rows x_ld apart, z[g] [N, R], U[g] [R, W*D], static_w[g]
 *   [W, D] (or static_w NULL), y[g] [N, D];
 *   state [slots, W-1, G*D] contiguous, of x's type, the last W-1 inputs,
 *   oldest first; it drops its oldest row and takes x[n] behind the others.
 * slot_ids as in dc_linear_attention_step. */
int dc_lowrank_step_grouped(int64_t G, const void* x, int64_t x_ld, const void* const* z, const void* const* U,
                            const void* const* static_w, void* state, const int32_t* slot_ids, void* const* y,
                            int64_t N, int64_t D, int64_t R, int64_t W, int64_t slots, int dtype, int residual,
                            void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DYNCONV_LAYER_H_ */
