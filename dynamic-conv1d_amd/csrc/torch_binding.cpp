// Native autograd binding of the C ABI (include/dynconv.h, dynconv_layer.h) for PyTorch: the
// operators' autograd Functions as C++ nodes, called from dynconv/*.py.
//
// A small or medium call is bound by its host path.  Through Python's
// autograd.Function and ctypes a forward takes 11-15 us and a backward 70-100 us
// of host time (the engine's thread has to take the GIL, and every argument
// passes through Python), against 5-20 us of kernels; here the checks, the
// allocations and the launches are native and the backward runs without the GIL.
//
// Each entry point returns None for every call it does not take (another type,
// layout, device or dtype than the plain one, function transforms, forward-mode
// derivatives, tracing, dispatch modes, failed preconditions): the Python
// Functions then take the call, and raise what they raise.  So this file holds
// no second copy of the operators' error behaviour.  What a taken call computes,
// saves and launches is what those Functions do (headwise.py:218-309,
// lowrank.py:214-299); kernel errors surface as the same RuntimeError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <dlfcn.h>

#include <cmath>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "dynconv.h"
#include "dynconv_layer.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// The C ABI, from the library that dynconv._capi loaded.
struct Abi {
  decltype(&dc_status_string) status_string;
  decltype(&dc_headwise_fwd) headwise_fwd;
  decltype(&dc_headwise_bwd_ws_bytes) headwise_bwd_ws_bytes;
  decltype(&dc_headwise_bwd) headwise_bwd;
  decltype(&dc_lowrank_zeff_bytes) lowrank_zeff_bytes;
  decltype(&dc_lowrank_fwd) lowrank_fwd;
  decltype(&dc_lowrank_bwd_ws_bytes) lowrank_bwd_ws_bytes;
  decltype(&dc_lowrank_bwd) lowrank_bwd;
  decltype(&dc_lowrank_fwd_grouped) lowrank_fwd_grouped;
  decltype(&dc_lowrank_bwd_grouped_ws_bytes) lowrank_bwd_grouped_ws_bytes;
  decltype(&dc_lowrank_bwd_grouped) lowrank_bwd_grouped;
  decltype(&dc_proj_in_fwd) proj_in_fwd;
  decltype(&dc_proj_in_bwd_ws_bytes) proj_in_bwd_ws_bytes;
  decltype(&dc_proj_in_bwd) proj_in_bwd;
  decltype(&dc_linear_attention_ws_bytes) linear_attention_ws_bytes;
  decltype(&dc_linear_attention_fwd) linear_attention_fwd;
  decltype(&dc_linear_attention_bwd) linear_attention_bwd;
  decltype(&dc_linear_attention_step) linear_attention_step;
  decltype(&dc_delta_rule_ws_bytes) delta_rule_ws_bytes;
  decltype(&dc_delta_rule_fwd) delta_rule_fwd;
  decltype(&dc_delta_rule_bwd) delta_rule_bwd;
  decltype(&dc_delta_rule_step) delta_rule_step;
  decltype(&dc_residual_norm_fwd) residual_norm_fwd;
  decltype(&dc_residual_norm_bwd_ws_bytes) residual_norm_bwd_ws_bytes;
  decltype(&dc_residual_norm_bwd) residual_norm_bwd;
  decltype(&dc_group_norm_fwd) group_norm_fwd;
  decltype(&dc_group_norm_bwd_ws_bytes) group_norm_bwd_ws_bytes;
  decltype(&dc_group_norm_bwd) group_norm_bwd;
  decltype(&dc_lowrank_step_grouped) lowrank_step_grouped;
};
Abi abi{};
bool ready = false;

void check(int64_t status, const char* what) {
  TORCH_CHECK(status >= 0, "dynconv ", what, " failed: ", abi.status_string((int)status), " (status ", status, ")");
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return DC_DTYPE_BF16;
    case at::kHalf: return DC_DTYPE_FP16;
    case at::kFloat: return DC_DTYPE_FP32;
    default: return -1;
  }
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// n bytes of device memory beside t (n == 0: none).
Tensor bytes_like(const Tensor& t, int64_t n) {
  return n > 0 ? at::empty({n}, t.options().dtype(at::kByte)) : Tensor();
}
// A kernel has written t through its pointer: what autograd has saved of it is stale, as after torch's in-place operations
// (tensors of inference mode have no version, and are not saved).
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// A gradient as the kernels read it: contiguous, in x's dtype.
Tensor grad_in(const Tensor& dy, at::ScalarType dtype) { return dy.contiguous().to(dtype); }

// ---------------------------------------------------------------- headwise
Tensor headwise_forward(const Tensor& x, const Tensor& w, const Tensor& sw, bool residual) {
  Tensor y = at::empty_like(x);
  check(abi.headwise_fwd(ptr(x), ptr(w), ptr(sw), ptr(y), x.size(0), x.size(1), x.size(2), w.size(2), w.size(3),
                         dtype_code(x), residual, stream_of(x)),
        "headwise forward");
  return y;
}

struct HeadwiseFn : public Function<HeadwiseFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& sw,
                        bool residual) {
    const Tensor s = sw.value_or(Tensor());
    Tensor y = headwise_forward(x, w, s, residual);
    ctx->save_for_backward({x, w, s});
    ctx->saved_data["residual"] = residual;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &sw = saved[2];
    const c10::DeviceGuard guard(x.device());
    const Tensor dy = grad_in(grads[0], x.scalar_type());
    Tensor dx = at::empty_like(x), dw = at::empty_like(w), dsw = sw.defined() ? at::empty_like(sw) : Tensor();
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2), H = w.size(2), W = w.size(3);
    const int dt = dtype_code(x);
    const int64_t n = abi.headwise_bwd_ws_bytes(B, T, D, H, W, dt, sw.defined());
    check(n, "headwise backward workspace query");
    const Tensor ws = bytes_like(x, n);
    check(abi.headwise_bwd(ptr(x), ptr(w), ptr(sw), ptr(dy), ptr(dx), ptr(dw), ptr(dsw), ptr(ws), n, B, T, D, H, W, dt,
                           ctx->saved_data["residual"].toBool(), stream_of(x)),
          "headwise backward");
    return {dx, dw, dsw, Tensor()};
  }
};

// ----------------------------------------------------------------- lowrank
struct LowrankFn : public Function<LowrankFn> {
  // zeff: the padded z copy that the forward keeps for the backward (null: none)
  static Tensor run(const Tensor& x, const Tensor& z, const Tensor& U, const Tensor& sw, const Tensor& zeff,
                    int64_t nzeff, bool residual) {
    Tensor y = at::empty_like(x);
    const int64_t D = x.size(2);
    check(abi.lowrank_fwd(ptr(x), ptr(z), ptr(U), ptr(sw), ptr(y), ptr(zeff), nzeff, x.size(0), x.size(1), D, z.size(2),
                          U.size(1) / D, dtype_code(x), residual, stream_of(x)),
          "lowrank forward");
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& z, const Tensor& U,
                        const std::optional<Tensor>& sw, bool residual) {
    const Tensor s = sw.value_or(Tensor());
    const int64_t D = x.size(2);
    const int64_t nz = abi.lowrank_zeff_bytes(x.size(0), x.size(1), D, z.size(2), U.size(1) / D, dtype_code(x), s.defined());
    check(nz, "lowrank z_eff size query");
    const Tensor zeff = bytes_like(x, nz);
    Tensor y = run(x, z, U, s, zeff, nz, residual);
    ctx->save_for_backward({x, z, U, s});
    ctx->saved_data["residual"] = residual;
    if (zeff.defined()) ctx->saved_data["zeff"] = zeff;  // internal buffer, a function of z
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &z = saved[1], &U = saved[2], &sw = saved[3];
    const c10::DeviceGuard guard(x.device());
    const Tensor dy = grad_in(grads[0], x.scalar_type());
    Tensor dx = at::empty_like(x), dz = at::empty_like(z), dU = at::empty_like(U);
    Tensor dsw = sw.defined() ? at::empty_like(sw) : Tensor();
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2), R = z.size(2), W = U.size(1) / D;
    const int dt = dtype_code(x);
    const int64_t n = abi.lowrank_bwd_ws_bytes(B, T, D, R, W, dt, sw.defined());
    check(n, "lowrank backward workspace query");
    const Tensor ws = bytes_like(x, n);
    const auto it = ctx->saved_data.find("zeff");
    const Tensor zeff = it != ctx->saved_data.end() ? it->second.toTensor() : Tensor();
    check(abi.lowrank_bwd(ptr(x), ptr(z), ptr(U), ptr(sw), ptr(zeff), zeff.defined() ? zeff.numel() : 0, ptr(dy),
                          ptr(dx), ptr(dz), ptr(dU), ptr(dsw), ptr(ws), n, B, T, D, R, W, dt,
                          ctx->saved_data["residual"].toBool(), stream_of(x)),
          "lowrank backward");
    return {dx, dz, dU, dsw, Tensor()};
  }
};

// ------------------------------------------------- grouped lowrank, with proj_in
// G device pointers, `stride` bytes apart from base (base null: all null).
struct Ptrs {
  void* p[DC_MAX_GROUPS] = {};
  Ptrs() = default;
  Ptrs(void* base, int64_t stride, int64_t G) {
    for (int64_t g = 0; g < G && base; ++g) p[g] = static_cast<char*>(base) + g * stride;
  }
  const void* const* in() const { return p; }
  void* const* out() const { return p; }
};

constexpr int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// The sizes of a grouped module call: x [B, T, G*D], pre_z [B, T, K], w_in [G*R, K],
// U [G, R, W*D], sw [G, W, D].
struct GroupedShape {
  int64_t G, B, T, D, R, W, K, zbytes, es;
  int dt;
  GroupedShape(const Tensor& x, const Tensor& pre, const Tensor& U)
      : G(U.size(0)), B(x.size(0)), T(x.size(1)), D(x.size(2) / U.size(0)), R(U.size(1)), W(U.size(2) / D),
        K(pre.size(2)), es(x.element_size()), dt(dtype_code(x)) {
    zbytes = round256(B * T * R * es);  // one group's z (or dz), on its own aligned range of one buffer
  }
};

// GroupedLowRankDynamicShortConvolution: z = proj_in(pre_z), then the grouped
// operator, as one node: the parameters' gradients are written as the whole
// tensors they belong to (slicing them per group costs a fill, a copy and an
// add per slice in the backward: 16 launches, 85 us of 864 at B2 T8192 D4096).
struct GroupedModuleFn : public Function<GroupedModuleFn> {
  static variable_list run(const Tensor& x, const Tensor& pre, const Tensor& w_in, const Tensor& U, const Tensor& sw,
                           int64_t hd, const GroupedShape& s, const Tensor& z, const Tensor& zeff, int64_t nzeff) {
    void* st = stream_of(x);
    const Ptrs zs(ptr(z), s.zbytes, s.G);
    check(abi.proj_in_fwd(ptr(pre), ptr(w_in), zs.out(), s.G, s.B * s.T, s.K, s.R, s.dt, st), "proj_in forward");
    variable_list ys;
    Ptrs yp;
    for (int64_t g = 0; g < s.G; ++g) {
      ys.push_back(hd ? at::empty({s.B, s.D / hd, s.T, hd}, x.options()) : at::empty({s.B, s.T, s.D}, x.options()));
      yp.p[g] = ptr(ys.back());
    }
    const Ptrs Us(ptr(U), s.R * s.W * s.D * s.es, s.G), sws(ptr(sw), s.W * s.D * s.es, s.G);
    const Ptrs ze(ptr(zeff), round256(nzeff), s.G);
    check(abi.lowrank_fwd_grouped(s.G, ptr(x), x.stride(1), zs.in(), Us.in(), sws.in(), yp.out(),
                                  zeff.defined() ? ze.out() : nullptr, nzeff, hd, s.B, s.T, s.D, s.R, s.W, s.dt, 1, st),
          "grouped lowrank forward");
    return ys;
  }
  static Tensor z_buffer(const Tensor& x, const GroupedShape& s) {
    return at::empty({s.G * s.zbytes / s.es}, x.options());
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& pre, const Tensor& w_in,
                               const Tensor& U, const Tensor& sw, int64_t hd) {
    const GroupedShape s(x, pre, U);
    const int64_t nz = abi.lowrank_zeff_bytes(s.B, s.T, s.D, s.R, s.W, s.dt, 1);
    check(nz, "lowrank z_eff size query");
    const Tensor z = z_buffer(x, s), zeff = bytes_like(x, s.G * round256(nz));
    variable_list ys = run(x, pre, w_in, U, sw, hd, s, z, zeff, nz);
    ctx->save_for_backward({x, pre, w_in, U, sw, z});
    ctx->saved_data["hd"] = hd;
    if (zeff.defined()) ctx->saved_data["zeff"] = zeff;
    return ys;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &pre = saved[1], &w_in = saved[2], &U = saved[3], &sw = saved[4], &z = saved[5];
    const c10::DeviceGuard guard(x.device());
    const GroupedShape s(x, pre, U);
    const int64_t hd = ctx->saved_data["hd"].toInt(), C = s.G * s.D;
    void* st = stream_of(x);
    variable_list dys;
    Ptrs dyp;
    for (int64_t g = 0; g < s.G; ++g) {
      dys.push_back(grad_in(grads[g], x.scalar_type()));
      dyp.p[g] = ptr(dys.back());
    }
    // pre_z or proj_in.weight wanted (inputs 1, 2): a frozen projection has no backward
    const bool proj = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    Tensor dx = at::empty({s.B, s.T, C}, x.options()), dpre, dw;
    if (proj) {
      dpre = at::empty_like(pre);
      dw = at::empty_like(w_in);
    }
    Tensor dU = at::empty_like(U), dsw = at::empty_like(sw);
    const Tensor dz = z_buffer(x, s);
    const auto it = ctx->saved_data.find("zeff");
    const Tensor zeff = it != ctx->saved_data.end() ? it->second.toTensor() : Tensor();
    const int64_t nz = zeff.defined() ? abi.lowrank_zeff_bytes(s.B, s.T, s.D, s.R, s.W, s.dt, 1) : 0;
    const int64_t n1 = abi.lowrank_bwd_grouped_ws_bytes(s.G, s.B, s.T, s.D, s.R, s.W, s.dt, 1);
    check(n1, "grouped lowrank backward workspace query");
    const int64_t n2 = proj ? abi.proj_in_bwd_ws_bytes(s.G, s.B * s.T, s.K, s.R, s.dt) : 0;
    check(n2, "proj_in backward workspace query");
    // one workspace: proj_in's backward runs after the convolutions' on the same stream
    const Tensor ws = bytes_like(x, std::max<int64_t>(std::max(n1, n2), 1));
    const Ptrs zs(ptr(z), s.zbytes, s.G), dzs(ptr(dz), s.zbytes, s.G), ze(ptr(zeff), round256(nz), s.G);
    const int64_t ub = s.R * s.W * s.D * s.es, sb = s.W * s.D * s.es;
    const Ptrs Us(ptr(U), ub, s.G), sws(ptr(sw), sb, s.G), dUs(ptr(dU), ub, s.G), dsws(ptr(dsw), sb, s.G);
    check(abi.lowrank_bwd_grouped(s.G, ptr(x), x.stride(1), zs.in(), Us.in(), sws.in(),
                                  zeff.defined() ? ze.in() : nullptr, nz, dyp.in(), hd, ptr(dx), C, dzs.out(),
                                  dUs.out(), dsws.out(), ptr(ws), n1, s.B, s.T, s.D, s.R, s.W, s.dt, 1, st),
          "grouped lowrank backward");
    if (proj)
      check(abi.proj_in_bwd(ptr(pre), ptr(w_in), dzs.in(), ptr(dpre), ptr(dw), ptr(ws), n2, s.G, s.B * s.T, s.K, s.R,
                            s.dt, st),
            "proj_in backward");
    return {dx, dpre, dw, dU, dsw, Tensor()};
  }
};

// ------------------------------------------------------- linear attention
struct LinearAttentionFn : public Function<LinearAttentionFn> {
  // o over token-major memory, and the final state if it is wanted
  static variable_list run(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const Tensor& s0,
                           const Tensor& lengths, double scale, bool want_state, Tensor* states = nullptr) {
    const int64_t B = q.size(0), H = q.size(1), T = q.size(2), K = q.size(3), V = v.size(3);
    const int dt = dtype_code(q);
    Tensor o = at::empty({B, T, H, V}, q.options()).transpose(1, 2);
    Tensor st = want_state ? at::empty({B, H, K, V}, lam.options()) : Tensor();
    const int64_t n = abi.linear_attention_ws_bytes(B, H, T, K, V, dt, 0);
    check(n, "linear attention workspace query");
    const Tensor ws = bytes_like(q, n);
    check(abi.linear_attention_fwd(ptr(q), q.strides().data(), ptr(k), k.strides().data(), ptr(v), v.strides().data(),
                                   static_cast<float*>(ptr(lam)), static_cast<float*>(ptr(s0)),
                                   static_cast<int32_t*>(ptr(lengths)), ptr(o), o.strides().data(),
                                   static_cast<float*>(ptr(st)), ptr(ws), n, B, H, T, K, V, (float)scale, dt,
                                   stream_of(q)),
          "linear attention forward");
    if (states) *states = ws;
    variable_list out{o};
    if (want_state) out.push_back(st);
    return out;
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const std::optional<Tensor>& s0, const Tensor& lam, const std::optional<Tensor>& lengths,
                               double scale, bool want_state) {
    const Tensor s = s0.value_or(Tensor()), n = lengths.value_or(Tensor());
    Tensor states;  // before each segment, a function of the inputs: the backward starts from them
    variable_list out = run(q, k, v, lam, s, n, scale, want_state, &states);
    ctx->save_for_backward({q, k, v, s, lam, n, states});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &s0 = saved[3], &lam = saved[4], &lengths = saved[5],
                 &states = saved[6];
    const c10::DeviceGuard guard(q.device());
    const int64_t B = q.size(0), H = q.size(1), T = q.size(2), K = q.size(3), V = v.size(3);
    const int dt = dtype_code(q);
    // an output that did not reach the loss has no gradient
    Tensor d = grads[0].defined() ? grads[0].to(q.scalar_type()) : at::zeros({B, H, T, V}, q.options());
    if (V > 1 && d.stride(3) != 1) d = d.contiguous();
    const Tensor ds = grads.size() > 1 && grads[1].defined() ? grad_in(grads[1], at::kFloat) : Tensor();
    Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
    Tensor ds0 = s0.defined() && ctx->needs_input_grad(3) ? at::empty_like(s0) : Tensor();
    const int64_t n = abi.linear_attention_ws_bytes(B, H, T, K, V, dt, states.defined() ? 2 : 1);
    check(n, "linear attention backward workspace query");
    const Tensor ws = bytes_like(q, n);
    check(abi.linear_attention_bwd(ptr(q), q.strides().data(), ptr(k), k.strides().data(), ptr(v), v.strides().data(),
                                   static_cast<float*>(ptr(lam)), static_cast<float*>(ptr(s0)),
                                   static_cast<int32_t*>(ptr(lengths)), ptr(d), d.strides().data(),
                                   static_cast<float*>(ptr(ds)), ptr(dq), dq.strides().data(), ptr(dk),
                                   dk.strides().data(), ptr(dv), dv.strides().data(), static_cast<float*>(ptr(ds0)),
                                   ptr(states), ptr(ws), n, B, H, T, K, V, (float)ctx->saved_data["scale"].toDouble(), dt,
                                   stream_of(q)),
          "linear attention backward");
    return {dq, dk, dv, ds0, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------- gated delta rule
struct DeltaSizes {
  int64_t B, Hk, H, T, K, V;
  int dt, gdt;
  DeltaSizes(const Tensor& q, const Tensor& v, const Tensor& beta)
      : B(q.size(0)), Hk(q.size(1)), H(v.size(1)), T(q.size(2)), K(q.size(3)), V(v.size(3)), dt(dtype_code(q)),
        gdt(dtype_code(beta)) {}
};

struct GatedDeltaRuleFn : public Function<GatedDeltaRuleFn> {
  // o over token-major memory, and the final state if it is wanted
  static variable_list run(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& b,
                           const Tensor& s0, const Tensor& lengths, double scale, double eps, int64_t flags,
                           bool want_state, Tensor* kept = nullptr) {
    const DeltaSizes z(q, v, b);
    Tensor o = at::empty({z.B, z.T, z.H, z.V}, q.options()).transpose(1, 2);
    Tensor st = want_state ? at::empty({z.B, z.H, z.K, z.V}, q.options().dtype(at::kFloat)) : Tensor();
    const int64_t n = abi.delta_rule_ws_bytes(z.B, z.Hk, z.H, z.T, z.K, z.V, z.dt, (int)flags, 0);
    check(n, "gated delta rule workspace query");
    const Tensor ws = bytes_like(q, n);
    check(abi.delta_rule_fwd(ptr(q), q.strides().data(), ptr(k), k.strides().data(), ptr(v), v.strides().data(), ptr(g),
                             g.strides().data(), ptr(b), b.strides().data(), static_cast<float*>(ptr(s0)),
                             static_cast<int32_t*>(ptr(lengths)), ptr(o), o.strides().data(),
                             static_cast<float*>(ptr(st)), ptr(ws), n, z.B, z.Hk, z.H, z.T, z.K, z.V, (float)scale,
                             (float)eps, z.dt, z.gdt, (int)flags, stream_of(q)),
          "gated delta rule forward");
    if (kept) *kept = ws;
    variable_list out{o};
    if (want_state) out.push_back(st);
    return out;
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                               const Tensor& b, const std::optional<Tensor>& s0, const std::optional<Tensor>& lengths,
                               double scale, double eps, int64_t flags, bool want_state) {
    const Tensor s = s0.value_or(Tensor()), n = lengths.value_or(Tensor());
    Tensor kept;  // each chunk's triangular systems, a function of the inputs, which the backward takes up again
    variable_list out = run(q, k, v, g, b, s, n, scale, eps, flags, want_state, &kept);
    ctx->save_for_backward({q, k, v, g, b, s, n, kept});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["flags"] = flags;
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &g = saved[3], &b = saved[4], &s0 = saved[5],
                 &lengths = saved[6], &kept = saved[7];
    const c10::DeviceGuard guard(q.device());
    const DeltaSizes z(q, v, b);
    const int flags = (int)ctx->saved_data["flags"].toInt();
    // an output that did not reach the loss has no gradient
    Tensor d = grads[0].defined() ? grads[0].to(q.scalar_type()) : at::zeros({z.B, z.H, z.T, z.V}, q.options());
    if (z.V > 1 && d.stride(3) != 1) d = d.contiguous();
    const Tensor ds = grads.size() > 1 && grads[1].defined() ? grad_in(grads[1], at::kFloat) : Tensor();
    Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v), dg = at::empty_like(g), db = at::empty_like(b);
    Tensor ds0 = s0.defined() && ctx->needs_input_grad(5) ? at::empty_like(s0) : Tensor();
    const int64_t n = abi.delta_rule_ws_bytes(z.B, z.Hk, z.H, z.T, z.K, z.V, z.dt, flags, kept.defined() ? 2 : 1);
    check(n, "gated delta rule backward workspace query");
    const Tensor ws = bytes_like(q, n);
    check(abi.delta_rule_bwd(ptr(q), q.strides().data(), ptr(k), k.strides().data(), ptr(v), v.strides().data(), ptr(g),
                             g.strides().data(), ptr(b), b.strides().data(), static_cast<float*>(ptr(s0)),
                             static_cast<int32_t*>(ptr(lengths)), ptr(d), d.strides().data(),
                             static_cast<float*>(ptr(ds)), ptr(dq), dq.strides().data(), ptr(dk), dk.strides().data(),
                             ptr(dv), dv.strides().data(), ptr(dg), dg.strides().data(), ptr(db), db.strides().data(),
                             static_cast<float*>(ptr(ds0)), ptr(kept), ptr(ws), n, z.B, z.Hk, z.H, z.T, z.K, z.V,
                             (float)ctx->saved_data["scale"].toDouble(), (float)ctx->saved_data["eps"].toDouble(), z.dt,
                             z.gdt, flags, stream_of(q)),
          "gated delta rule backward");
    return {dq, dk, dv, dg, db, ds0, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ----------------------------------------------------------- residual norm
struct ResidualNormFn : public Function<ResidualNormFn> {
  static int param_code(const Tensor& branch, const Tensor& w, const Tensor& bw, const Tensor& sc) {
    return dtype_code(w.defined() ? w : bw.defined() ? bw : sc.defined() ? sc : branch);
  }
  static variable_list run(const Tensor& x, const Tensor& branch, const Tensor& w, const Tensor& bw, const Tensor& gate,
                           const Tensor& sc, double constant, int64_t act, double eps) {
    Tensor y = at::empty_like(branch), h = at::empty_like(x);
    const int64_t D = x.size(-1);
    check(abi.residual_norm_fwd(ptr(x), ptr(branch), ptr(w), ptr(bw), ptr(gate), ptr(sc), ptr(y), ptr(h), x.numel() / D, D,
                                (float)constant, (float)eps, (int)act, dtype_code(branch), dtype_code(x),
                                param_code(branch, w, bw, sc), stream_of(x)),
          "residual norm forward");
    return {y, h};
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& branch, const std::optional<Tensor>& w,
                               const std::optional<Tensor>& bw, const std::optional<Tensor>& gate,
                               const std::optional<Tensor>& sc, double constant, int64_t act, double eps) {
    const Tensor wt = w.value_or(Tensor()), bt = bw.value_or(Tensor()), gt = gate.value_or(Tensor()), st = sc.value_or(Tensor());
    variable_list out = run(x, branch, wt, bt, gt, st, constant, act, eps);
    ctx->save_for_backward({out[1], branch, wt, bt, gt, st});
    ctx->saved_data["constant"] = constant;
    ctx->saved_data["act"] = act;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &branch = saved[1], &w = saved[2], &bw = saved[3], &gate = saved[4], &sc = saved[5];
    const c10::DeviceGuard guard(h.device());
    const int64_t D = h.size(-1), M = h.numel() / D;
    // an output that did not reach the loss has no gradient
    const Tensor dy = grads[0].defined() ? grad_in(grads[0], branch.scalar_type()) : Tensor();
    const Tensor dh = grads[1].defined() ? grad_in(grads[1], h.scalar_type()) : Tensor();
    Tensor dx = at::empty_like(h), dbranch = at::empty_like(branch), dgate = gate.defined() ? at::empty_like(gate) : Tensor();
    // an input that is None has no place among the indexes
    size_t at = 2;
    const bool want_w = w.defined() && ctx->needs_input_grad(at++), want_b = bw.defined() && ctx->needs_input_grad(at++);
    at += gate.defined();
    const bool want_s = sc.defined() && ctx->needs_input_grad(at);
    Tensor dw = want_w ? at::empty_like(w) : Tensor(), dbw = want_b ? at::empty_like(bw) : Tensor(),
           ds = want_s ? at::empty_like(sc) : Tensor();
    const int dt = dtype_code(branch);
    const int64_t n = want_w || want_b || want_s ? abi.residual_norm_bwd_ws_bytes(M, D, dt) : 0;
    check(n, "residual norm backward workspace query");
    const Tensor ws = bytes_like(h, n);
    check(abi.residual_norm_bwd(ptr(h), ptr(branch), ptr(w), ptr(bw), ptr(gate), ptr(sc), ptr(dy), ptr(dh), ptr(dx),
                                ptr(dbranch), ptr(dgate), ptr(dw), ptr(dbw), ptr(ds), ptr(ws), n, M, D,
                                (float)ctx->saved_data["constant"].toDouble(), (float)ctx->saved_data["eps"].toDouble(),
                                (int)ctx->saved_data["act"].toInt(), dt, dtype_code(h), param_code(branch, w, bw, sc),
                                stream_of(h)),
          "residual norm backward");
    return {dx, dbranch, dw, dbw, dgate, ds, Tensor(), Tensor(), Tensor()};
  }
};

// -------------------------------------------------------------- group norm
struct GroupNormFn : public Function<GroupNormFn> {
  static int param_code(const Tensor& x, const Tensor& w, const Tensor& b) {
    return dtype_code(w.defined() ? w : b.defined() ? b : x);
  }
  static Tensor run(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& gate, int64_t groups, int64_t act,
                    double eps) {
    Tensor y = at::empty_like(x);
    const int64_t D = x.size(-1);
    check(abi.group_norm_fwd(ptr(x), ptr(w), ptr(b), ptr(gate), ptr(y), x.numel() / D, D, groups, (float)eps, (int)act,
                             dtype_code(x), param_code(x, w, b), stream_of(x)),
          "group norm forward");
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& w,
                        const std::optional<Tensor>& b, const std::optional<Tensor>& gate, int64_t groups, int64_t act,
                        double eps) {
    const Tensor wt = w.value_or(Tensor()), bt = b.value_or(Tensor()), gt = gate.value_or(Tensor());
    Tensor y = run(x, wt, bt, gt, groups, act, eps);
    ctx->save_for_backward({x, wt, bt, gt});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &gate = saved[3];
    const c10::DeviceGuard guard(x.device());
    const int64_t D = x.size(-1), M = x.numel() / D, groups = ctx->saved_data["groups"].toInt();
    const Tensor dy = grad_in(grads[0], x.scalar_type());
    Tensor dx = at::empty_like(x), dgate = gate.defined() ? at::empty_like(gate) : Tensor();
    Tensor dw = w.defined() && ctx->needs_input_grad(1) ? at::empty_like(w) : Tensor();
    // an input that is None has no place among the indexes
    Tensor db = b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1) ? at::empty_like(b) : Tensor();
    const int dt = dtype_code(x);
    const int64_t n = dw.defined() || db.defined() ? abi.group_norm_bwd_ws_bytes(M, D, groups, dt) : 0;
    check(n, "group norm backward workspace query");
    const Tensor ws = bytes_like(x, n);
    check(abi.group_norm_bwd(ptr(x), ptr(w), ptr(b), ptr(gate), ptr(dy), ptr(dx), ptr(dgate), ptr(dw), ptr(db), ptr(ws),
                             n, M, D, groups, (float)ctx->saved_data["eps"].toDouble(),
                             (int)ctx->saved_data["act"].toInt(), dt, param_code(x, w, b), stream_of(x)),
          "group norm backward");
    return {dx, dw, db, dgate, Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------ entry points
// No function transform, dispatch mode or tracer is looking at this call.
bool plain_call() {
  using c10::DispatchKey;
  return ready && !c10::impl::tls_is_dispatch_key_included(DispatchKey::FuncTorchDynamicLayerFrontMode) &&
         !c10::impl::tls_is_dispatch_key_included(DispatchKey::Python) &&
         !c10::impl::TorchDispatchModeTLS::any_modes_set() && !torch::jit::tracer::isTracing();
}

// A torch.Tensor or Parameter (no subclass) in dense device memory, of x's dtype
// and device when given, without a forward-mode tangent.
bool plain_tensor(PyObject* o, Tensor* out, const Tensor* like = nullptr) {
  if (!THPVariable_CheckExact(o)) return false;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.numel() == 0 || !t.has_storage()) return false;
  if (t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                               c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Negative,
                                               c10::DispatchKey::Functionalize})))
    return false;
  if (t._fw_grad(/*level=*/0).defined()) return false;
  if (like && (t.scalar_type() != like->scalar_type() || t.device() != like->device())) return false;
  *out = t;
  return true;
}

bool any_requires_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

#define DC_DECLINE_UNLESS(cond) \
  if (!(cond)) Py_RETURN_NONE

std::optional<Tensor> opt(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// A tuple of tensors.
PyObject* wrap_all(variable_list ts) {
  PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
  if (!out) return nullptr;
  for (size_t i = 0; i < ts.size(); ++i) {
    PyObject* o = THPVariable_Wrap(std::move(ts[i]));
    if (!o) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, (Py_ssize_t)i, o);
  }
  return out;
}

// headwise(x, weight, static_w or None, residual) -> y, or None (not taken)
PyObject* py_headwise(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor x, w, sw;
  DC_DECLINE_UNLESS(nargs == 4 && plain_call() && plain_tensor(args[0], &x) && plain_tensor(args[1], &w, &x));
  DC_DECLINE_UNLESS(args[2] == Py_None || plain_tensor(args[2], &sw, &x));
  DC_DECLINE_UNLESS(dtype_code(x) >= 0 && x.dim() == 3 && w.dim() == 4 && x.is_contiguous() && w.is_contiguous());
  DC_DECLINE_UNLESS(w.size(0) == x.size(0) && w.size(1) == x.size(1) && x.size(2) % w.size(2) == 0);
  DC_DECLINE_UNLESS(!sw.defined() || (sw.dim() == 2 && sw.size(0) == w.size(3) && sw.size(1) == x.size(2) &&
                                      sw.is_contiguous()));
  const int residual = PyObject_IsTrue(args[3]);
  if (residual < 0) return nullptr;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(x.device());
    y = any_requires_grad({&x, &w, &sw}) ? HeadwiseFn::apply(x, w, opt(sw), residual != 0)
                                         : headwise_forward(x, w, sw, residual != 0);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// lowrank(x, z, U, static_w or None, residual) -> y, or None (not taken)
PyObject* py_lowrank(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor x, z, U, sw;
  DC_DECLINE_UNLESS(nargs == 5 && plain_call() && plain_tensor(args[0], &x) && plain_tensor(args[1], &z, &x) &&
                    plain_tensor(args[2], &U, &x));
  DC_DECLINE_UNLESS(args[3] == Py_None || plain_tensor(args[3], &sw, &x));
  DC_DECLINE_UNLESS(dtype_code(x) >= 0 && x.dim() == 3 && z.dim() == 3 && U.dim() == 2);
  DC_DECLINE_UNLESS(x.is_contiguous() && z.is_contiguous() && U.is_contiguous());
  const int64_t D = x.size(2), R = z.size(2), rank = R + (sw.defined() ? 1 : 0);
  DC_DECLINE_UNLESS((rank & (rank - 1)) == 0 && z.size(0) == x.size(0) && z.size(1) == x.size(1));
  DC_DECLINE_UNLESS(U.size(0) == R && U.size(1) % D == 0);
  DC_DECLINE_UNLESS(!sw.defined() || (sw.dim() == 2 && sw.size(0) == U.size(1) / D && sw.size(1) == D &&
                                      sw.is_contiguous()));
  const int residual = PyObject_IsTrue(args[4]);
  if (residual < 0) return nullptr;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(x.device());
    y = any_requires_grad({&x, &z, &U, &sw}) ? LowrankFn::apply(x, z, U, opt(sw), residual != 0)
                                             : LowrankFn::run(x, z, U, sw, Tensor(), 0, residual != 0);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// grouped_module(x, pre_z, w_in, proj_out, proj_out_bias, head_dim) -> tuple of G outputs, or None (not taken)
PyObject* py_grouped_module(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor x, pre, w_in, U, sw;
  DC_DECLINE_UNLESS(nargs == 6 && plain_call() && plain_tensor(args[0], &x) && plain_tensor(args[1], &pre, &x) &&
                    plain_tensor(args[2], &w_in, &x) && plain_tensor(args[3], &U, &x) && plain_tensor(args[4], &sw, &x));
  DC_DECLINE_UNLESS(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf);
  DC_DECLINE_UNLESS(x.dim() == 3 && pre.dim() == 3 && w_in.dim() == 2 && U.dim() == 3 && sw.dim() == 3);
  const int64_t G = U.size(0), B = x.size(0), T = x.size(1), R = U.size(1), K = pre.size(2);
  DC_DECLINE_UNLESS(G >= 1 && G <= DC_MAX_GROUPS && x.size(2) % G == 0);
  const int64_t D = x.size(2) / G;
  DC_DECLINE_UNLESS(((R + 1) & R) == 0 && U.size(2) % D == 0 && sw.size(0) == G && sw.size(1) == U.size(2) / D &&
                    sw.size(2) == D);
  DC_DECLINE_UNLESS(pre.size(0) == B && pre.size(1) == T && w_in.size(0) == G * R && w_in.size(1) == K);
  DC_DECLINE_UNLESS(x.stride(2) == 1 && x.stride(0) == T * x.stride(1));
  DC_DECLINE_UNLESS(pre.is_contiguous() && w_in.is_contiguous() && U.is_contiguous() && sw.is_contiguous());
  // proj_in on the library's kernels (modules._proj_in_native)
  DC_DECLINE_UNLESS(G * R <= 128 && K % 8 == 0 && aligned16(pre) && aligned16(w_in));
  int64_t hd = 0;
  if (args[5] != Py_None) {
    hd = PyLong_AsLongLong(args[5]);
    if (hd == -1 && PyErr_Occurred()) return nullptr;
    DC_DECLINE_UNLESS(hd > 0 && hd <= D && D % hd == 0);
  }
  variable_list ys;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(x.device());
    if (any_requires_grad({&x, &pre, &w_in, &U, &sw})) {
      ys = GroupedModuleFn::apply(x, pre, w_in, U, sw, hd);
    } else {
      const GroupedShape s(x, pre, U);
      ys = GroupedModuleFn::run(x, pre, w_in, U, sw, hd, s, GroupedModuleFn::z_buffer(x, s), Tensor(), 0);
    }
  }
  return wrap_all(std::move(ys));
  END_HANDLE_TH_ERRORS
}

// None (t stays undefined), or a plain tensor on like's device.
bool optional_tensor(PyObject* o, Tensor* t, const Tensor& like) {
  return o == Py_None || (plain_tensor(o, t) && t->device() == like.device());
}

bool rows_whole(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

// log_decay [H] and the scale of linear attention's calls; false: not taken (err: an exception is set)
bool decay_and_scale(PyObject* decay, PyObject* scale, const Tensor& q, Tensor* lam, double* s, bool* err) {
  if (!plain_tensor(decay, lam) || lam->device() != q.device() || lam->scalar_type() != at::kFloat || lam->dim() != 1 ||
      lam->size(0) != q.size(1) || !lam->is_contiguous() || any_requires_grad({lam}))
    return false;
  if (scale == Py_None) {
    *s = 1.0 / std::sqrt((double)q.size(-1));
  } else {
    *s = PyFloat_AsDouble(scale);
    *err = *s == -1.0 && PyErr_Occurred();
  }
  return !*err;
}

bool int_vector(const Tensor& t, int64_t n) {
  return !t.defined() || (t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous());
}

// linear_attention(q, k, v, log_decay, scale, initial_state, lengths, return_state) -> o or (o, state), or None (not taken)
PyObject* py_linear_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, lam, s0, lengths;
  DC_DECLINE_UNLESS(nargs == 8 && plain_call() && plain_tensor(args[0], &q) && plain_tensor(args[1], &k, &q) &&
                    plain_tensor(args[2], &v, &q));
  DC_DECLINE_UNLESS(dtype_code(q) >= 0 && q.dim() == 4 && v.dim() == 4 && k.sizes() == q.sizes());
  const int64_t B = q.size(0), H = q.size(1), K = q.size(3), V = v.size(3);
  DC_DECLINE_UNLESS(v.size(0) == B && v.size(1) == H && v.size(2) == q.size(2) && K <= DC_LA_MAX_DIM && V <= DC_LA_MAX_DIM);
  DC_DECLINE_UNLESS(rows_whole(q) && rows_whole(k) && rows_whole(v));
  DC_DECLINE_UNLESS(optional_tensor(args[5], &s0, q) && optional_tensor(args[6], &lengths, q) && int_vector(lengths, B));
  DC_DECLINE_UNLESS(!s0.defined() || (s0.scalar_type() == at::kFloat && s0.is_contiguous() && s0.dim() == 4 &&
                                      s0.size(0) == B && s0.size(1) == H && s0.size(2) == K && s0.size(3) == V));
  double scale = 0;
  bool err = false;
  if (!decay_and_scale(args[3], args[4], q, &lam, &scale, &err)) {
    if (err) return nullptr;
    Py_RETURN_NONE;
  }
  const int want = PyObject_IsTrue(args[7]);
  if (want < 0) return nullptr;
  variable_list out;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(q.device());
    out = any_requires_grad({&q, &k, &v, &s0}) ? LinearAttentionFn::apply(q, k, v, opt(s0), lam, opt(lengths), scale, want != 0)
                                               : LinearAttentionFn::run(q, k, v, lam, s0, lengths, scale, want != 0);
  }
  return want ? wrap_all(std::move(out)) : THPVariable_Wrap(std::move(out[0]));
  END_HANDLE_TH_ERRORS
}

// linear_attention_step(q, k, v, log_decay, state, scale, slots) -> o, or None (not taken)
PyObject* py_linear_attention_step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, lam, state, slots;
  DC_DECLINE_UNLESS(nargs == 7 && plain_call() && plain_tensor(args[0], &q) && plain_tensor(args[1], &k, &q) &&
                    plain_tensor(args[2], &v, &q) && plain_tensor(args[4], &state) && state.device() == q.device());
  DC_DECLINE_UNLESS(dtype_code(q) >= 0 && q.dim() == 3 && v.dim() == 3 && k.sizes() == q.sizes());
  const int64_t B = q.size(0), H = q.size(1), K = q.size(2), V = v.size(2);
  DC_DECLINE_UNLESS(v.size(0) == B && v.size(1) == H && K <= DC_LA_MAX_DIM && V <= DC_LA_MAX_DIM);
  DC_DECLINE_UNLESS(rows_whole(q) && rows_whole(k) && rows_whole(v) && !any_requires_grad({&q, &k, &v, &state}));
  DC_DECLINE_UNLESS(state.scalar_type() == at::kFloat && state.is_contiguous() && state.dim() == 4 && state.size(1) == H &&
                    state.size(2) == K && state.size(3) == V);
  DC_DECLINE_UNLESS(optional_tensor(args[6], &slots, q) && int_vector(slots, B) &&
                    (slots.defined() || B <= state.size(0)));
  double scale = 0;
  bool err = false;
  if (!decay_and_scale(args[3], args[5], q, &lam, &scale, &err)) {
    if (err) return nullptr;
    Py_RETURN_NONE;
  }
  Tensor o;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(q.device());
    o = at::empty({B, H, V}, q.options());
    check(abi.linear_attention_step(ptr(q), q.strides().data(), ptr(k), k.strides().data(), ptr(v), v.strides().data(),
                                    static_cast<float*>(ptr(lam)), static_cast<float*>(ptr(state)),
                                    static_cast<int32_t*>(ptr(slots)), ptr(o), B, H, K, V, state.size(0), (float)scale,
                                    dtype_code(q), stream_of(q)),
          "linear attention step");
    written(state);
  }
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

// Whether q, k [B, Hk, ..., K], v [B, H, ..., V] and the gates (v's shape without its channels) are of the plain kind, with
// `rows` axes between heads and channels.
bool delta_inputs(PyObject* const* args, int rows, Tensor* q, Tensor* k, Tensor* v, Tensor* g, Tensor* b) {
  if (!plain_tensor(args[0], q) || !plain_tensor(args[1], k, q) || !plain_tensor(args[2], v, q) ||
      !plain_tensor(args[3], g) || !plain_tensor(args[4], b, g))
    return false;
  const int64_t n = 3 + rows;
  if (dtype_code(*q) < 0 || q->dim() != n || v->dim() != n || k->sizes() != q->sizes() || g->device() != q->device() ||
      (g->scalar_type() != q->scalar_type() && g->scalar_type() != at::kFloat))
    return false;
  if (v->size(0) != q->size(0) || v->size(1) % q->size(1) != 0 || (rows && v->size(2) != q->size(2)) ||
      q->size(-1) > DC_LA_MAX_DIM || v->size(-1) > DC_LA_MAX_DIM)
    return false;
  return g->sizes() == v->sizes().slice(0, n - 1) && b->sizes() == g->sizes() && rows_whole(*q) && rows_whole(*k) &&
         rows_whole(*v);
}

// scale (None: 1 / sqrt(K)) and eps; false: an exception is set
bool scale_and_eps(PyObject* scale, PyObject* eps, const Tensor& q, double* s, double* e) {
  *s = scale == Py_None ? 1.0 / std::sqrt((double)q.size(-1)) : PyFloat_AsDouble(scale);
  *e = PyFloat_AsDouble(eps);
  return !PyErr_Occurred();
}

// gated_delta_rule(q, k, v, log_decay, beta, scale, initial_state, lengths, return_state, normalize, eps) -> o or (o, state),
// or None (not taken)
PyObject* py_gated_delta_rule(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, g, b, s0, lengths;
  DC_DECLINE_UNLESS(nargs == 11 && plain_call() && delta_inputs(args, 1, &q, &k, &v, &g, &b));
  DC_DECLINE_UNLESS(optional_tensor(args[6], &s0, q) && optional_tensor(args[7], &lengths, q) && int_vector(lengths, q.size(0)));
  DC_DECLINE_UNLESS(!s0.defined() || (s0.scalar_type() == at::kFloat && s0.is_contiguous() && s0.dim() == 4 &&
                                      s0.size(0) == q.size(0) && s0.size(1) == v.size(1) && s0.size(2) == q.size(3) &&
                                      s0.size(3) == v.size(3)));
  double scale = 0, eps = 0;
  if (!scale_and_eps(args[5], args[10], q, &scale, &eps)) return nullptr;
  const int want = PyObject_IsTrue(args[8]), unit = PyObject_IsTrue(args[9]);
  if (want < 0 || unit < 0) return nullptr;
  // delta._wide_results: whether a result of a call in 16 bits is float32
  const bool gates = g.scalar_type() == at::kFloat && any_requires_grad({&g, &b});
  const bool wide = q.scalar_type() != at::kFloat && (want || gates || any_requires_grad({&s0}));
  const bool grads = any_requires_grad({&q, &k, &v, &g, &b, &s0});
  const int64_t flags = (unit ? DC_DELTA_NORMALIZE : 0) | (wide ? DC_DELTA_PRECISE : 0) | (grads ? DC_DELTA_KEEP : 0);
  variable_list out;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(q.device());
    out = grads
              ? GatedDeltaRuleFn::apply(q, k, v, g, b, opt(s0), opt(lengths), scale, eps, flags, want != 0)
              : GatedDeltaRuleFn::run(q, k, v, g, b, s0, lengths, scale, eps, flags, want != 0);
  }
  return want ? wrap_all(std::move(out)) : THPVariable_Wrap(std::move(out[0]));
  END_HANDLE_TH_ERRORS
}

// gated_delta_rule_step(q, k, v, log_decay, beta, state, scale, slots, normalize, eps) -> o, or None (not taken)
PyObject* py_gated_delta_rule_step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, g, b, state, slots;
  DC_DECLINE_UNLESS(nargs == 10 && plain_call() && delta_inputs(args, 0, &q, &k, &v, &g, &b) &&
                    plain_tensor(args[5], &state) && state.device() == q.device());
  const int64_t B = q.size(0), Hk = q.size(1), K = q.size(2), H = v.size(1), V = v.size(2);
  DC_DECLINE_UNLESS(!any_requires_grad({&q, &k, &v, &g, &b, &state}));
  DC_DECLINE_UNLESS(state.scalar_type() == at::kFloat && state.is_contiguous() && state.dim() == 4 && state.size(1) == H &&
                    state.size(2) == K && state.size(3) == V);
  DC_DECLINE_UNLESS(optional_tensor(args[7], &slots, q) && int_vector(slots, B) &&
                    (slots.defined() || B <= state.size(0)));
  double scale = 0, eps = 0;
  if (!scale_and_eps(args[6], args[9], q, &scale, &eps)) return nullptr;
  const int unit = PyObject_IsTrue(args[8]);
  if (unit < 0) return nullptr;
  Tensor o;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(q.device());
    o = at::empty({B, H, V}, q.options());
    check(abi.delta_rule_step(ptr(q), q.strides().data(), ptr(k), k.strides().data(), ptr(v), v.strides().data(), ptr(g),
                              g.strides().data(), ptr(b), b.strides().data(), static_cast<float*>(ptr(state)),
                              static_cast<int32_t*>(ptr(slots)), ptr(o), B, Hk, H, K, V, state.size(0), (float)scale,
                              (float)eps, dtype_code(q), dtype_code(b), unit ? DC_DELTA_NORMALIZE : 0, stream_of(q)),
          "gated delta rule step");
    written(state);
  }
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

// residual_norm(x, branch, weight, branch_weight, gate, activation code, scale, constant, eps) -> (y, h), or None (not taken)
PyObject* py_residual_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor x, branch, w, bw, gate, sc;
  DC_DECLINE_UNLESS(nargs == 9 && plain_call() && plain_tensor(args[0], &x) && plain_tensor(args[1], &branch) &&
                    branch.device() == x.device() && dtype_code(branch) >= 0 && x.dim() >= 1);
  DC_DECLINE_UNLESS(x.scalar_type() == branch.scalar_type() || x.scalar_type() == at::kFloat);
  DC_DECLINE_UNLESS(x.sizes() == branch.sizes() && x.is_contiguous() && branch.is_contiguous() && PyLong_CheckExact(args[5]));
  DC_DECLINE_UNLESS(optional_tensor(args[2], &w, x) && optional_tensor(args[3], &bw, x) && optional_tensor(args[6], &sc, x));
  DC_DECLINE_UNLESS(args[4] == Py_None || (plain_tensor(args[4], &gate, &branch) && gate.is_contiguous() &&
                                           gate.sizes() == x.sizes()));
  const int64_t D = x.size(-1), act = PyLong_AsLongLong(args[5]);
  const double constant = PyFloat_AsDouble(args[7]), eps = PyFloat_AsDouble(args[8]);
  if (PyErr_Occurred()) return nullptr;
  DC_DECLINE_UNLESS(D <= DC_RN_MAX_DIM && (gate.defined() || act == 0));
  const Tensor* one = nullptr;
  for (const Tensor* p : {&w, &bw, &sc}) {
    if (!p->defined()) continue;
    DC_DECLINE_UNLESS(p->dim() == 1 && p->size(0) == D && p->is_contiguous() &&
                      (p->scalar_type() == at::kFloat || p->scalar_type() == branch.scalar_type()) &&
                      (!one || one->scalar_type() == p->scalar_type()));
    one = p;
  }
  variable_list out;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(x.device());
    out = any_requires_grad({&x, &branch, &w, &bw, &gate, &sc})
              ? ResidualNormFn::apply(x, branch, opt(w), opt(bw), opt(gate), opt(sc), constant, act, eps)
              : ResidualNormFn::run(x, branch, w, bw, gate, sc, constant, act, eps);
  }
  return wrap_all(std::move(out));
  END_HANDLE_TH_ERRORS
}

// group_norm(x, groups, weight, bias, gate, activation code, eps) -> y, or None (not taken)
PyObject* py_group_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor x, w, b, gate;
  DC_DECLINE_UNLESS(nargs == 7 && plain_call() && plain_tensor(args[0], &x) && dtype_code(x) >= 0 && x.dim() >= 1 &&
                    x.is_contiguous());
  DC_DECLINE_UNLESS(PyLong_CheckExact(args[1]) && PyLong_CheckExact(args[5]));
  DC_DECLINE_UNLESS(optional_tensor(args[2], &w, x) && optional_tensor(args[3], &b, x));
  DC_DECLINE_UNLESS(args[4] == Py_None || (plain_tensor(args[4], &gate, &x) && gate.is_contiguous() && gate.sizes() == x.sizes()));
  const int64_t D = x.size(-1), groups = PyLong_AsLongLong(args[1]), act = PyLong_AsLongLong(args[5]);
  const double eps = PyFloat_AsDouble(args[6]);
  if (PyErr_Occurred()) return nullptr;
  DC_DECLINE_UNLESS(groups > 0 && D % groups == 0 && D / groups <= 4096);
  for (const Tensor* p : {&w, &b})
    DC_DECLINE_UNLESS(!p->defined() || (p->dim() == 1 && p->size(0) == D && p->is_contiguous() &&
                                        (p->scalar_type() == at::kFloat || p->scalar_type() == x.scalar_type())));
  DC_DECLINE_UNLESS(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type());
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(x.device());
    y = any_requires_grad({&x, &w, &b, &gate}) ? GroupNormFn::apply(x, opt(w), opt(b), opt(gate), groups, act, eps)
                                               : GroupNormFn::run(x, w, b, gate, groups, act, eps);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// lowrank_step(x, z list, U list, state, static_w list or None, residual, slots) -> tuple of G tensors, or None (not taken)
PyObject* py_lowrank_step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor x, state, slots, z[DC_MAX_GROUPS], U[DC_MAX_GROUPS], sw[DC_MAX_GROUPS];
  DC_DECLINE_UNLESS(nargs == 7 && plain_call() && plain_tensor(args[0], &x) && plain_tensor(args[3], &state, &x) &&
                    dtype_code(x) >= 0 && x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= x.size(1));
  const bool has_static = args[4] != Py_None;
  DC_DECLINE_UNLESS(PyList_CheckExact(args[1]) && PyList_CheckExact(args[2]) && (!has_static || PyList_CheckExact(args[4])));
  const int64_t G = PyList_GET_SIZE(args[1]);
  DC_DECLINE_UNLESS(G >= 1 && G <= DC_MAX_GROUPS && PyList_GET_SIZE(args[2]) == G &&
                    (!has_static || PyList_GET_SIZE(args[4]) == G) && x.size(1) % G == 0);
  const int64_t N = x.size(0), D = x.size(1) / G;
  int64_t R = 0, W = 0;
  for (int64_t g = 0; g < G; ++g) {
    DC_DECLINE_UNLESS(plain_tensor(PyList_GET_ITEM(args[1], g), &z[g], &x) && plain_tensor(PyList_GET_ITEM(args[2], g), &U[g], &x) &&
                      (!has_static || plain_tensor(PyList_GET_ITEM(args[4], g), &sw[g], &x)));
    if (g == 0) {
      DC_DECLINE_UNLESS(z[0].dim() == 2 && U[0].dim() == 2);
      R = z[0].size(1);
      W = U[0].size(1) / D;
    }
    DC_DECLINE_UNLESS(z[g].dim() == 2 && z[g].size(0) == N && z[g].size(1) == R && z[g].is_contiguous());
    DC_DECLINE_UNLESS(U[g].dim() == 2 && U[g].size(0) == R && U[g].size(1) == W * D && U[g].is_contiguous());
    DC_DECLINE_UNLESS(!has_static || (sw[g].dim() == 2 && sw[g].size(0) == W && sw[g].size(1) == D && sw[g].is_contiguous()));
    DC_DECLINE_UNLESS(!any_requires_grad({&z[g], &U[g], &sw[g]}));
  }
  const int64_t rank = R + (has_static ? 1 : 0);
  DC_DECLINE_UNLESS(W > 1 && (rank & (rank - 1)) == 0 && !any_requires_grad({&x, &state}));
  DC_DECLINE_UNLESS(state.is_contiguous() && state.dim() == 3 && state.size(1) == W - 1 && state.size(2) == G * D);
  DC_DECLINE_UNLESS(optional_tensor(args[6], &slots, x) && int_vector(slots, N) && (slots.defined() || N <= state.size(0)));
  const int residual = PyObject_IsTrue(args[5]);
  if (residual < 0) return nullptr;
  variable_list ys;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(x.device());
    const void *zp[DC_MAX_GROUPS], *Up[DC_MAX_GROUPS], *sp[DC_MAX_GROUPS];
    void* yp[DC_MAX_GROUPS];
    const Tensor y = at::empty({G, N, D}, x.options());
    for (int64_t g = 0; g < G; ++g) {
      zp[g] = ptr(z[g]);
      Up[g] = ptr(U[g]);
      sp[g] = ptr(sw[g]);
      ys.push_back(y.select(0, g));
      yp[g] = ptr(ys.back());
    }
    check(abi.lowrank_step_grouped(G, ptr(x), x.stride(0), zp, Up, has_static ? sp : nullptr, ptr(state),
                                   static_cast<int32_t*>(ptr(slots)), yp, N, D, R, W, state.size(0), dtype_code(x),
                                   residual != 0, stream_of(x)),
          "lowrank step");
    written(state);
  }
  return wrap_all(std::move(ys));
  END_HANDLE_TH_ERRORS
}

// init(path): take the C ABI from the library at path (loaded already by dynconv._capi).
PyObject* py_init(PyObject*, PyObject* path) {
  HANDLE_TH_ERRORS
  const char* p = PyUnicode_AsUTF8(path);
  if (!p) return nullptr;
  void* lib = dlopen(p, RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(lib != nullptr, "cannot load ", p, ": ", dlerror());
  auto sym = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(lib, name));
    TORCH_CHECK(f != nullptr, p, " has no symbol ", name);
  };
  sym(abi.status_string, "dc_status_string");
  sym(abi.headwise_fwd, "dc_headwise_fwd");
  sym(abi.headwise_bwd_ws_bytes, "dc_headwise_bwd_ws_bytes");
  sym(abi.headwise_bwd, "dc_headwise_bwd");
  sym(abi.lowrank_zeff_bytes, "dc_lowrank_zeff_bytes");
  sym(abi.lowrank_fwd, "dc_lowrank_fwd");
  sym(abi.lowrank_bwd_ws_bytes, "dc_lowrank_bwd_ws_bytes");
  sym(abi.lowrank_bwd, "dc_lowrank_bwd");
  sym(abi.lowrank_fwd_grouped, "dc_lowrank_fwd_grouped");
  sym(abi.lowrank_bwd_grouped_ws_bytes, "dc_lowrank_bwd_grouped_ws_bytes");
  sym(abi.lowrank_bwd_grouped, "dc_lowrank_bwd_grouped");
  sym(abi.proj_in_fwd, "dc_proj_in_fwd");
  sym(abi.proj_in_bwd_ws_bytes, "dc_proj_in_bwd_ws_bytes");
  sym(abi.proj_in_bwd, "dc_proj_in_bwd");
  sym(abi.linear_attention_ws_bytes, "dc_linear_attention_ws_bytes");
  sym(abi.linear_attention_fwd, "dc_linear_attention_fwd");
  sym(abi.linear_attention_bwd, "dc_linear_attention_bwd");
  sym(abi.linear_attention_step, "dc_linear_attention_step");
  sym(abi.delta_rule_ws_bytes, "dc_delta_rule_ws_bytes");
  sym(abi.delta_rule_fwd, "dc_delta_rule_fwd");
  sym(abi.delta_rule_bwd, "dc_delta_rule_bwd");
  sym(abi.delta_rule_step, "dc_delta_rule_step");
  sym(abi.residual_norm_fwd, "dc_residual_norm_fwd");
  sym(abi.residual_norm_bwd_ws_bytes, "dc_residual_norm_bwd_ws_bytes");
  sym(abi.residual_norm_bwd, "dc_residual_norm_bwd");
  sym(abi.group_norm_fwd, "dc_group_norm_fwd");
  sym(abi.group_norm_bwd_ws_bytes, "dc_group_norm_bwd_ws_bytes");
  sym(abi.group_norm_bwd, "dc_group_norm_bwd");
  sym(abi.lowrank_step_grouped, "dc_lowrank_step_grouped");
  ready = true;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"init", py_init, METH_O, "Take the C ABI from the library at a path."},
    {"headwise", (PyCFunction)(void*)py_headwise, METH_FASTCALL, "headwise(x, weight, static_w, residual)"},
    {"lowrank", (PyCFunction)(void*)py_lowrank, METH_FASTCALL, "lowrank(x, z, U, static_w, residual)"},
    {"grouped_module", (PyCFunction)(void*)py_grouped_module, METH_FASTCALL,
     "grouped_module(x, pre_z, w_in, proj_out, proj_out_bias, head_dim)"},
    {"linear_attention", (PyCFunction)(void*)py_linear_attention, METH_FASTCALL,
     "linear_attention(q, k, v, log_decay, scale, initial_state, lengths, return_state)"},
    {"linear_attention_step", (PyCFunction)(void*)py_linear_attention_step, METH_FASTCALL,
     "linear_attention_step(q, k, v, log_decay, state, scale, slots)"},
    {"gated_delta_rule", (PyCFunction)(void*)py_gated_delta_rule, METH_FASTCALL,
     "gated_delta_rule(q, k, v, log_decay, beta, scale, initial_state, lengths, return_state, normalize, eps)"},
    {"gated_delta_rule_step", (PyCFunction)(void*)py_gated_delta_rule_step, METH_FASTCALL,
     "gated_delta_rule_step(q, k, v, log_decay, beta, state, scale, slots, normalize, eps)"},
    {"residual_norm", (PyCFunction)(void*)py_residual_norm, METH_FASTCALL,
     "residual_norm(x, branch, weight, branch_weight, gate, activation, scale, constant, eps)"},
    {"group_norm", (PyCFunction)(void*)py_group_norm, METH_FASTCALL,
     "group_norm(x, groups, weight, bias, gate, activation, eps)"},
    {"lowrank_step", (PyCFunction)(void*)py_lowrank_step, METH_FASTCALL,
     "lowrank_step(x, z, U, state, static_w, residual, slots)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION_BUILT) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
