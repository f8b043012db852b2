/*
 * dynconv_layer.h -- C ABI of the operators that stand behind the short
 * convolutions in a layer (libdynconv.so, with dynconv.h): linear attention
 * with a decay for each head, in its form for whole sequences and its form for
 * single tokens; the group norm of its heads with an activation or a gate; and
 * the lowrank convolutions' form for single tokens.  The reference has none of
 * these.
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

/* Activations of dc_group_norm_fwd / _bwd. */
typedef enum dc_activation { DC_ACT_NONE = 0, DC_ACT_SILU = 1 } dc_activation;

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
