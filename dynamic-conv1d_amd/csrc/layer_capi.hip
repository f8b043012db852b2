// C ABI of include/dynconv_layer.h: argument checks on the host, then one
// launch function per entry point.  Nothing here allocates, synchronises or
// throws.
#include "dynconv_layer.h"
#include "layer_launch.h"

namespace {

constexpr int64_t kI32Max = 2147483647;

bool dtype_ok(int dt) { return dt == DC_DTYPE_BF16 || dt == DC_DTYPE_FP16 || dt == DC_DTYPE_FP32; }
bool aligned_to(const void* p, int a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
int launch_status(hipError_t e) { return e == hipSuccess ? DC_OK : DC_ERR_LAUNCH; }

int device_status() {
  int n = 0;
  static const bool ok = hipGetDeviceCount(&n) == hipSuccess && n > 0;
  return ok ? DC_OK : DC_ERR_DEVICE;
}

// Sizes of linear attention: every head's channels within DC_LA_MAX_DIM, every
// index that the kernels hold in 32 bits within it.
int check_la(int64_t B, int64_t H, int64_t T, int64_t K, int64_t V, int dtype) {
  if (!dtype_ok(dtype)) return DC_ERR_DTYPE;
  if (B <= 0 || H <= 0 || T < 0 || K <= 0 || V <= 0) return DC_ERR_SHAPE;
  if (B > kI32Max || H > kI32Max || T > kI32Max / 2 || B * H > kI32Max / 8) return DC_ERR_SHAPE;
  if (K > DC_LA_MAX_DIM || V > DC_LA_MAX_DIM) return DC_ERR_UNSUPPORTED;
  return DC_OK;
}

bool copy3(int64_t (&to)[3], const int64_t* from) {
  if (!from) return false;
  for (int i = 0; i < 3; ++i) to[i] = from[i];
  return true;
}

}  // namespace

extern "C" {

int64_t dc_linear_attention_ws_bytes(int64_t B, int64_t H, int64_t T, int64_t K, int64_t V, int dtype, int bwd) {
  const int s = check_la(B, H, T, K, V, dtype);
  if (s != DC_OK) return s;
  dc::LaProblem p{};
  p.B = B; p.H = H; p.T = T; p.dtype = dtype;
  p.npass = bwd ? 3 : 1;
  for (int i = 0; i < p.npass; ++i) {
    const bool turned = bwd && i < 2;  // dq and dk: the state is [V, K]
    p.pass[i].K = (int)(turned ? V : K);
    p.pass[i].V = (int)(turned ? K : V);
  }
  return dc::la_ws_bytes(p, bwd == 2);
}

int dc_linear_attention_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                            const void* v, const int64_t* v_strides, const float* log_decay,
                            const float* initial_state, const int32_t* lengths, void* o, const int64_t* o_strides,
                            float* final_state, void* workspace, int64_t ws_bytes, int64_t B, int64_t H, int64_t T,
                            int64_t K, int64_t V, float scale, int dtype, void* stream) {
  const int64_t need = dc_linear_attention_ws_bytes(B, H, T, K, V, dtype, 0);
  if (need < 0) return (int)need;
  if (!log_decay || (T > 0 && (!q || !k || !v || !o))) return DC_ERR_NULL;
  const int es = dc::dtype_size(dtype);
  if (!aligned_to(q, es) || !aligned_to(k, es) || !aligned_to(v, es) || !aligned_to(o, es) ||
      !aligned_to(log_decay, 4) || !aligned_to(initial_state, 4) || !aligned_to(final_state, 4) ||
      !aligned_to(lengths, 4))
    return DC_ERR_ALIGN;
  if (need > 0 && (!workspace || ws_bytes < need || !aligned_to(workspace, 16))) return DC_ERR_WORKSPACE;
  dc::LaProblem p{};
  dc::LaPass& a = p.pass[0];
  if (!copy3(a.qs, q_strides) || !copy3(a.ks, k_strides) || !copy3(a.vs, v_strides) || !copy3(a.os, o_strides))
    return DC_ERR_NULL;
  int s = device_status();
  if (s != DC_OK) return s;
  a.q = q; a.k = k; a.v = v; a.o = o;
  a.s_in = initial_state; a.s_out = final_state; a.s_row = V; a.s_col = 1;
  a.K = (int)K; a.V = (int)V; a.so = scale; a.skv = 1.f;
  p.npass = 1;
  p.log_decay = log_decay; p.lengths = lengths;
  p.B = B; p.H = H; p.T = T; p.dtype = dtype;
  p.ws = workspace; p.stream = (hipStream_t)stream;
  return launch_status(dc::la_run(p));
}

int dc_linear_attention_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                            const void* v, const int64_t* v_strides, const float* log_decay,
                            const float* initial_state, const int32_t* lengths, const void* d_o,
                            const int64_t* do_strides, const float* d_final_state, void* dq,
                            const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                            const int64_t* dv_strides, float* d_initial_state, const void* fwd_workspace,
                            void* workspace, int64_t ws_bytes, int64_t B, int64_t H, int64_t T, int64_t K, int64_t V, float scale, int dtype,
                            void* stream) {
  const int64_t need = dc_linear_attention_ws_bytes(B, H, T, K, V, dtype, fwd_workspace ? 2 : 1);
  if (need < 0) return (int)need;
  if (!log_decay || (T > 0 && (!q || !k || !v || !d_o || !dq || !dk || !dv))) return DC_ERR_NULL;
  const int es = dc::dtype_size(dtype);
  for (const void* t : {q, k, v, d_o, (const void*)dq, (const void*)dk, (const void*)dv})
    if (!aligned_to(t, es)) return DC_ERR_ALIGN;
  for (const void* t : {(const void*)log_decay, (const void*)initial_state, (const void*)d_final_state,
                        (const void*)d_initial_state, (const void*)lengths})
    if (!aligned_to(t, 4)) return DC_ERR_ALIGN;
  if (need > 0 && (!workspace || ws_bytes < need || !aligned_to(workspace, 16))) return DC_ERR_WORKSPACE;
  if (!aligned_to(fwd_workspace, 16)) return DC_ERR_WORKSPACE;
  for (const int64_t* t : {q_strides, k_strides, v_strides, do_strides, dq_strides, dk_strides, dv_strides})
    if (!t) return DC_ERR_NULL;
  int s = device_status();
  if (s != DC_OK) return s;
  dc::LaProblem p{};
  // dq = the operator on (do, v, k), its state the forward's turned over
  dc::LaPass& a = p.pass[0];
  a.q = d_o; a.k = v; a.v = k; a.o = dq;
  copy3(a.qs, do_strides); copy3(a.ks, v_strides); copy3(a.vs, k_strides); copy3(a.os, dq_strides);
  a.s_in = initial_state; a.s_row = 1; a.s_col = V;
  a.K = (int)V; a.V = (int)K; a.so = scale; a.skv = 1.f;
  // dk = the operator on (v, do, q) from the last token on, the state's gradient turned over
  dc::LaPass& b = p.pass[1];
  b.q = v; b.k = d_o; b.v = q; b.o = dk;
  copy3(b.qs, v_strides); copy3(b.ks, do_strides); copy3(b.vs, q_strides); copy3(b.os, dk_strides);
  b.s_in = d_final_state; b.s_row = 1; b.s_col = V;
  b.K = (int)V; b.V = (int)K; b.rev = 1; b.so = 1.f; b.skv = scale;
  // dv = the operator on (k, q, do) from the last token on
  dc::LaPass& c = p.pass[2];
  c.q = k; c.k = q; c.v = d_o; c.o = dv;
  copy3(c.qs, k_strides); copy3(c.ks, q_strides); copy3(c.vs, do_strides); copy3(c.os, dv_strides);
  c.s_in = d_final_state; c.s_out = d_initial_state; c.s_row = V; c.s_col = 1;
  c.K = (int)K; c.V = (int)V; c.rev = 1; c.so = 1.f; c.skv = scale;
  p.npass = 3;
  p.fwd_states = static_cast<const float*>(fwd_workspace);
  p.log_decay = log_decay; p.lengths = lengths;
  p.B = B; p.H = H; p.T = T; p.dtype = dtype;
  p.ws = workspace; p.stream = (hipStream_t)stream;
  return launch_status(dc::la_run(p));
}

int dc_linear_attention_step(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                             const void* v, const int64_t* v_strides, const float* log_decay, float* state,
                             const int32_t* slot_ids, void* o, int64_t B, int64_t H, int64_t K, int64_t V,
                             int64_t slots, float scale, int dtype, void* stream) {
  int s = check_la(B, H, 1, K, V, dtype);
  if (s != DC_OK) return s;
  if (slots <= 0 || slots > kI32Max || (!slot_ids && B > slots)) return DC_ERR_SHAPE;
  if (!q || !k || !v || !o || !log_decay || !state || !q_strides || !k_strides || !v_strides) return DC_ERR_NULL;
  const int es = dc::dtype_size(dtype);
  if (!aligned_to(q, es) || !aligned_to(k, es) || !aligned_to(v, es) || !aligned_to(o, es) ||
      !aligned_to(log_decay, 4) || !aligned_to(state, 4) || !aligned_to(slot_ids, 4))
    return DC_ERR_ALIGN;
  if ((s = device_status()) != DC_OK) return s;
  dc::LaStep p{};
  p.q = q; p.k = k; p.v = v;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = q_strides[i];
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
  }
  p.log_decay = log_decay; p.state = state; p.slot_ids = slot_ids; p.o = o;
  p.B = B; p.H = H; p.K = K; p.V = V; p.slots = slots;
  p.scale = scale; p.dtype = dtype; p.stream = (hipStream_t)stream;
  return launch_status(dc::la_step(p));
}

}  // extern "C"

// Sizes of a group norm.
static int check_gn(int64_t M, int64_t D, int64_t groups, int act, int dtype, int pdtype) {
  if (!dtype_ok(dtype) || (pdtype != dtype && pdtype != DC_DTYPE_FP32)) return DC_ERR_DTYPE;
  if (M <= 0 || D <= 0 || groups <= 0 || M > kI32Max || D > kI32Max || D % groups != 0) return DC_ERR_SHAPE;
  if (act != DC_ACT_NONE && act != DC_ACT_SILU) return DC_ERR_UNSUPPORTED;
  dc::GnProblem p{};
  p.M = M; p.D = D; p.groups = groups; p.dtype = dtype;
  return dc::gn_shape_ok(p) ? DC_OK : DC_ERR_UNSUPPORTED;
}

extern "C" {

int dc_group_norm_fwd(const void* x, const void* weight, const void* bias, const void* gate, void* y, int64_t M,
                      int64_t D, int64_t groups, float eps, int activation, int dtype, int param_dtype, void* stream) {
  int s = check_gn(M, D, groups, activation, dtype, param_dtype);
  if (s != DC_OK) return s;
  if (!x || !y) return DC_ERR_NULL;
  const int es = dc::dtype_size(dtype), ps = dc::dtype_size(param_dtype);
  if (!aligned_to(x, es) || !aligned_to(gate, es) || !aligned_to(y, es) || !aligned_to(weight, ps) ||
      !aligned_to(bias, ps))
    return DC_ERR_ALIGN;
  if ((s = device_status()) != DC_OK) return s;
  dc::GnProblem p{};
  p.x = x; p.weight = weight; p.bias = bias; p.gate = gate; p.y = y;
  p.M = M; p.D = D; p.groups = groups; p.eps = eps; p.act = activation;
  p.dtype = dtype; p.pdtype = param_dtype; p.stream = (hipStream_t)stream;
  return launch_status(dc::gn_fwd(p));
}

int64_t dc_group_norm_bwd_ws_bytes(int64_t M, int64_t D, int64_t groups, int dtype) {
  const int s = check_gn(M, D, groups, DC_ACT_NONE, dtype, dtype);
  if (s != DC_OK) return s;
  dc::GnProblem p{};
  p.M = M; p.D = D; p.groups = groups; p.dtype = dtype;
  return dc::gn_bwd_ws_bytes(p);
}

int dc_group_norm_bwd(const void* x, const void* weight, const void* bias, const void* gate, const void* dy, void* dx,
                      void* dgate, void* dweight, void* dbias, void* workspace, int64_t ws_bytes, int64_t M, int64_t D,
                      int64_t groups, float eps, int activation, int dtype, int param_dtype, void* stream) {
  int s = check_gn(M, D, groups, activation, dtype, param_dtype);
  if (s != DC_OK) return s;
  if (!x || !dy || !dx || (gate == nullptr) != (dgate == nullptr)) return DC_ERR_NULL;
  const int es = dc::dtype_size(dtype), ps = dc::dtype_size(param_dtype);
  if (!aligned_to(x, es) || !aligned_to(gate, es) || !aligned_to(dy, es) || !aligned_to(dx, es) ||
      !aligned_to(dgate, es) || !aligned_to(weight, ps) || !aligned_to(bias, ps) || !aligned_to(dweight, ps) ||
      !aligned_to(dbias, ps))
    return DC_ERR_ALIGN;
  if (dweight || dbias) {
    const int64_t need = dc_group_norm_bwd_ws_bytes(M, D, groups, dtype);
    if (!workspace || ws_bytes < need || !aligned_to(workspace, 16)) return DC_ERR_WORKSPACE;
  }
  if ((s = device_status()) != DC_OK) return s;
  dc::GnProblem p{};
  p.x = x; p.weight = weight; p.bias = bias; p.gate = gate; p.dy = dy;
  p.dx = dx; p.dgate = dgate; p.dweight = dweight; p.dbias = dbias; p.ws = (float*)workspace;
  p.M = M; p.D = D; p.groups = groups; p.eps = eps; p.act = activation;
  p.dtype = dtype; p.pdtype = param_dtype; p.stream = (hipStream_t)stream;
  return launch_status(dc::gn_bwd(p));
}

int dc_lowrank_step_grouped(int64_t G, const void* x, int64_t x_ld, const void* const* z, const void* const* U,
                            const void* const* static_w, void* state, const int32_t* slot_ids, void* const* y,
                            int64_t N, int64_t D, int64_t R, int64_t W, int64_t slots, int dtype, int residual,
                            void* stream) {
  if (!dtype_ok(dtype)) return DC_ERR_DTYPE;
  if (G < 1 || G > DC_MAX_GROUPS || N <= 0 || D <= 0 || R <= 0 || W <= 0 || slots <= 0) return DC_ERR_SHAPE;
  if (N > kI32Max || slots > kI32Max || D > kI32Max / DC_MAX_GROUPS || (!slot_ids && N > slots)) return DC_ERR_SHAPE;
  if (W > DC_MAX_W || R + (static_w ? 1 : 0) > DC_MAX_R) return DC_ERR_UNSUPPORTED;
  if (W * D > kI32Max || x_ld < G * D) return DC_ERR_SHAPE;
  if (!x || !z || !U || !y || (W > 1 && !state)) return DC_ERR_NULL;
  const int es = dc::dtype_size(dtype);
  if (!aligned_to(x, es) || !aligned_to(state, es) || !aligned_to(slot_ids, 4)) return DC_ERR_ALIGN;
  dc::LrStep p{};
  for (int64_t g = 0; g < G; ++g) {
    if (!z[g] || !U[g] || !y[g] || (static_w && !static_w[g])) return DC_ERR_NULL;
    if (!aligned_to(z[g], es) || !aligned_to(U[g], es) || !aligned_to(y[g], es) ||
        (static_w && !aligned_to(static_w[g], es)))
      return DC_ERR_ALIGN;
    p.z[g] = z[g];
    p.U[g] = U[g];
    p.static_w[g] = static_w ? static_w[g] : nullptr;
    p.y[g] = y[g];
  }
  const int s = device_status();
  if (s != DC_OK) return s;
  p.x = x; p.x_ld = x_ld; p.state = state; p.slot_ids = slot_ids;
  p.G = G; p.N = N; p.D = D; p.R = R; p.W = W; p.slots = slots;
  p.dtype = dtype; p.residual = residual ? 1 : 0; p.stream = (hipStream_t)stream;
  return launch_status(dc::lr_step(p));
}

}  // extern "C"
