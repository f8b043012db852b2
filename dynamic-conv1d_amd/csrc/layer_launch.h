// Internal host-side launch interface between the C ABI of dynconv_layer.h
// (layer_capi.hip) and its kernels.  Not part of the public ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dc_launch.h"

namespace dc {

// Workgroups of one launch: a grid's work-items along an axis are counted in 32 bits.
constexpr int64_t most_workgroups(int threads) { return 0xFFFFFFFFll / threads; }

// ------------------------------------------------------- linear attention
// One pass of the chunked operator over B x H sequences of one head each:
//     S_t = g S_{t-1} + skv k_t^T v_t,    o_t = so q_t S_t
// in the order of time, or (rev) against it; q, k have K channels, v, o have V.
// The forward is one such pass, the backward three (linattn.hip).
struct LaPass {
  const void *q, *k, *v;
  void* o;
  int64_t qs[3], ks[3], vs[3], os[3];  // strides (batch, head, row), elements
  // states [B, H, rows, cols]: element (a, n) of the pass's K x V state is at
  // a * s_row + n * s_col of its (batch, head)
  const float* s_in;  // state before the first token of the pass (null: zero)
  float* s_out;       // state after its last token (null: not wanted)
  int64_t s_row, s_col;
  int K, V;
  int rev;
  float so, skv;
};
constexpr int kLaMaxPasses = 3;
struct LaProblem {
  LaPass pass[kLaMaxPasses];
  int npass;
  const float* log_decay;
  const int32_t* lengths;  // null: all T
  int64_t B, H, T;
  int dtype;
  void* ws;
  const float* fwd_states;  // backward: the states before each segment that the forward left in its workspace (null: none)
  hipStream_t stream;
};
int64_t la_ws_bytes(const LaProblem& p, bool fwd_states);  // fwd_states: whether the backward will be given them
hipError_t la_run(const LaProblem& p);

struct LaStep {
  const void *q, *k, *v;
  int64_t qs[2], ks[2], vs[2];
  const float* log_decay;
  float* state;
  const int32_t* slot_ids;
  void* o;
  int64_t B, H, K, V, slots;
  int64_t bh0;  // first head of a launch (all of them: as many launches as it takes)
  float scale;
  int dtype;
  hipStream_t stream;
};
hipError_t la_step(const LaStep& p);

// ------------------------------------------------------- gated delta rule
struct DrProblem {
  const void *q, *k, *v, *g, *b;  // g: log_decay, b: beta
  int64_t qs[3], ks[3], vs[3], gs[3], bs[3];  // strides (batch, head, row), elements
  const float* s_in;
  const int32_t* lengths;
  void* o;
  int64_t os[3];
  float* s_out;
  // backward
  const void* d_o;
  int64_t dos[3];
  const float* ds_in;  // the final state's gradient
  void *dq, *dk, *dv, *dg, *db;
  int64_t dqs[3], dks[3], dvs[3], dgs[3], dbs[3];
  float* ds_out;  // the initial state's
  const void* fwd_ws;
  void* ws;
  int64_t B, Hk, H, T, K, V;
  float scale, eps;
  int dtype, gdtype, normalize, precise, keep;
  hipStream_t stream;
};
int64_t dr_ws_bytes(const DrProblem& p, int bwd);
hipError_t dr_fwd(const DrProblem& p);
hipError_t dr_bwd(const DrProblem& p);

struct DrStep {
  const void *q, *k, *v, *g, *b;
  int64_t qs[2], ks[2], vs[2], gs[2], bs[2];
  float* state;
  const int32_t* slot_ids;
  void* o;
  int64_t B, Hk, H, K, V, slots;
  int64_t bh0;  // first head of a launch
  float scale, eps;
  int dtype, gdtype, normalize;
  hipStream_t stream;
};
hipError_t dr_step(const DrStep& p);

// ------------------------------------------------------------- group norm
struct GnProblem {
  const void *x, *weight, *bias, *gate, *dy;
  void *y, *dx, *dgate, *dweight, *dbias;
  float* ws;
  int64_t M, D, groups;
  float eps;
  int act;
  int dtype, pdtype;
  hipStream_t stream;
};
bool gn_shape_ok(const GnProblem& p);
int64_t gn_bwd_ws_bytes(const GnProblem& p);
hipError_t gn_fwd(const GnProblem& p);
hipError_t gn_bwd(const GnProblem& p);

// ---------------------------------------------------------- residual norm
struct RnProblem {
  const void *x, *branch, *weight, *branch_weight, *gate, *scale, *dy, *dh;
  void *y, *h, *dx, *dbranch, *dgate, *dweight, *dbranch_weight, *dscale;  // h: the backward reads it
  float* ws;
  int64_t M, D;
  float constant, eps;
  int act;
  int dtype, xdtype, pdtype;
  hipStream_t stream;
};
int64_t rn_bwd_ws_bytes(const RnProblem& p);
hipError_t rn_fwd(const RnProblem& p);
hipError_t rn_bwd(const RnProblem& p);

// ------------------------------------------------------- convolution step
struct LrStep {
  const void* x;
  int64_t x_ld;
  const void* z[kMaxGroups];
  const void* U[kMaxGroups];
  const void* static_w[kMaxGroups];  // all null: no static filter
  void* y[kMaxGroups];
  void* state;
  const int32_t* slot_ids;
  int64_t G, N, D, R, W, slots;
  int dtype;
  int residual;
  hipStream_t stream;
};
hipError_t lr_step(const LrStep& p);

}  // namespace dc
