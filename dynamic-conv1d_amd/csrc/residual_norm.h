// The norms around a block, its gate, its residual scale and the residual sum (include/dynconv_layer.h), and their
// gradients:
//
//   n = branch rb bw,   h = x + n f,   y = h rh w,     f = constant scale act(gate),  r. = 1/sqrt(mean(.^2) + eps)
//   dx = dh + rh (dy w - h rh^2 mean(dy w h)),   dbranch = rb (dx f bw - branch rb^2 mean(dx f bw branch))
//   dw = sum dy h rh,   dbw = sum dx f branch rb,   dscale = constant sum dx n act,   dgate = constant dx n scale act'
//
// Streams, bound by HBM: forward x, branch, gate in and h, y out; backward h, branch, gate, dy, dh in and dx, dbranch,
// dgate out, each once.  A row's channels stay in the registers of a wavefront (up to 16 to a lane) or of a workgroup's 256
// lanes, which walk rows with the parameters, and backward the sums of their gradients, in registers; each workgroup writes
// those sums once, and reduce_partials adds them in a fixed order.  The backward forms the norms' factors again.
// 16384 x 4096, gate, scale, bf16: forward 124 us (0.67 GB, 5.4 TB/s), backward 193 (1.07 GB, 5.6 TB/s) and 7 of sums;
// 8 x 2048 forward 4.2 us, the launch.
#pragma once

#include "group_norm.h"

namespace dc {
namespace rn {

using gn::kWaves;
using gn::Lane;
using gn::Row;

struct Args {
  gn::GnArgs g;  // the row as one group: D, size, lanes
  const void *x, *branch, *weight, *branch_weight, *gate, *scale, *dy, *dh;
  void *y, *h, *dx, *dbranch, *dgate;
  float *pw, *pb, *ps;  // partial sums of the parameters' gradients, [row blocks][D] each (null: not wanted)
  float constant;
};

// N sums over a row at once; WIDE: over the workgroup (`slot` alternates, so one barrier serves).
template <bool WIDE, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[kWaves][4], int& slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = gn::lane_sum(v[i], 64);
  if constexpr (WIDE) {
    if (threadIdx.x % 64 == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) red[slot][threadIdx.x / 64][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (red[slot][0][i] + red[slot][1][i]) + (red[slot][2][i] + red[slot][3][i]);
    slot ^= 1;
  }
}

// A row's pieces through buffers of the row's range: channels past it, rows past the last (there: false) and tensors that
// are not given read as zeros and are not written, without a branch.  Under branches every load was waited for at once, and
// the next row never was on its way (16384 x 4096 gated bf16 backward 350 -> 210 us).
template <typename T, int VEC, int NV>
__device__ __forceinline__ void fetch(Row<T, VEC, NV>& r, const Lane<VEC, NV>& L, const void* p, int64_t row, int64_t D, bool there) {
  const rsrc_t rs = make_rsrc_wave((const T*)p + row * D, p && there ? D * (int64_t)sizeof(T) : 0);
#pragma unroll
  for (int i = 0; i < NV; ++i) bload_raw(r.v[i], rs, ((int)L.ch + i * L.step) * (int)sizeof(T));
}
template <typename T, int VEC, int NV>
__device__ __forceinline__ void leave(const Lane<VEC, NV>& L, void* p, int64_t row, int64_t D, const float (&v)[NV][VEC]) {
  const rsrc_t rs = make_rsrc_wave((T*)p + row * D, D * (int64_t)sizeof(T));
#pragma unroll
  for (int i = 0; i < NV; ++i) bstore_vals<T, VEC, VEC * sizeof(T) % 16 == 0>(rs, ((int)L.ch + i * L.step) * (int)sizeof(T), v[i]);
}
// What was asked for before this row's stores is waited for behind them, where the compiler can count them; at the top of the
// loop it would wait for the stores too.
template <typename T, int VEC, int NV>
__device__ __forceinline__ void arrived(Row<T, VEC, NV>& r) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < Raw<T, VEC>::NU; ++j) asm volatile("" : "+v"(r.v[i].u[j]));
}

// act(a) and its derivative
__device__ __forceinline__ void activate(int act, float a, float& f, float& d) {
  const float sg = gn::sigmoid(a);
  f = act == 1 ? a * sg : act == 2 ? sg : a;
  d = act == 1 ? sg * (1.f + a * (1.f - sg)) : act == 2 ? sg * (1.f - sg) : 1.f;
}

template <typename T, int VEC, int NV>
__device__ __forceinline__ void params(const Lane<VEC, NV>& L, const Args& A, const void* p, float (&v)[NV][VEC]) {
  if (A.g.wide_params) gn::load_param<float, VEC, NV>(L, p, A.g.param_pieces, 1.f, v);
  else gn::load_param<T, VEC, NV>(L, p, A.g.param_pieces, 1.f, v);
}

template <typename T, typename XT, int VEC, int NV, bool WIDE, bool GATE>
__global__ __launch_bounds__(64 * kWaves) void rn_fwd_kernel(Args A) {
  __shared__ float red[2][kWaves][4];
  int slot = 0;
  const Lane<VEC, NV> L(A.g);
  const int64_t step = (int64_t)gridDim.y * (WIDE ? 1 : kWaves), D = A.g.D;
  int64_t m = WIDE ? (int64_t)blockIdx.y : (int64_t)blockIdx.y * kWaves + wave_id();
  if (m >= A.g.M) return;
  Row<XT, VEC, NV> xr;
  Row<T, VEC, NV> br, ar;
  auto next = [&](int64_t row) {
    fetch(br, L, A.branch, row, D, row < A.g.M);
    fetch(xr, L, A.x, row, D, row < A.g.M);
    if (GATE) fetch(ar, L, A.gate, row, D, row < A.g.M);
  };
  next(m);
  float w[NV][VEC], bw[NV][VEC], sc[NV][VEC];
  params<T, VEC, NV>(L, A, A.weight, w);
  params<T, VEC, NV>(L, A, A.branch_weight, bw);
  params<T, VEC, NV>(L, A, A.scale, sc);
  const float inv = 1.f / A.g.size;
  for (; m < A.g.M; m += step) {
    float x[NV][VEC], b[NV][VEC], a[NV][VEC];
    xr.get(x);
    br.get(b);
    if (GATE) ar.get(a);
    next(m + step);
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] += b[i][j] * b[i][j];
    row_sum<WIDE>(s, red, slot);
    const float rb = gn::rsqrt_of(s[0] * inv + A.g.eps);
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float f = 1.f, d;
        if (GATE) activate(A.g.act, a[i][j], f, d);
        x[i][j] = (float)(XT)(x[i][j] + b[i][j] * rb * bw[i][j] * (f * sc[i][j] * A.constant));  // h as it is returned
        s[0] += x[i][j] * x[i][j];
      }
    }
    leave<XT, VEC, NV>(L, A.h, m, D, x);
    row_sum<WIDE>(s, red, slot);
    const float rh = gn::rsqrt_of(s[0] * inv + A.g.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i][j] *= rh * w[i][j];
    leave<T, VEC, NV>(L, A.y, m, D, x);
    arrived(br);
    arrived(xr);
    if (GATE) arrived(ar);
  }
}

template <typename T, typename XT, int VEC, int NV, bool WIDE, bool GATE>
__global__ __launch_bounds__(64 * kWaves) void rn_bwd_kernel(Args A) {
  constexpr bool kAhead = VEC * NV <= 16;  // the next row on its way while registers last
  __shared__ float red[2][kWaves][4], sum[WIDE ? 1 : kWaves][WIDE ? 1 : 64 * VEC];
  int slot = 0;
  const Lane<VEC, NV> L(A.g);
  const int64_t step = (int64_t)gridDim.y * (WIDE ? 1 : kWaves), D = A.g.D;
  int64_t m = WIDE ? (int64_t)blockIdx.y : (int64_t)blockIdx.y * kWaves + wave_id();
  Row<XT, VEC, NV> hr, er;
  Row<T, VEC, NV> br, ar, dr;
  auto next = [&](int64_t row) {
    fetch(hr, L, A.h, row, D, row < A.g.M);
    fetch(br, L, A.branch, row, D, row < A.g.M);
    fetch(dr, L, A.dy, row, D, row < A.g.M);
    fetch(er, L, A.dh, row, D, row < A.g.M);
    if (GATE) fetch(ar, L, A.gate, row, D, row < A.g.M);
  };
  if (kAhead) next(m);
  float w[NV][VEC], bw[NV][VEC], sc[NV][VEC], gw[NV][VEC], gb[NV][VEC], gs[NV][VEC];
  params<T, VEC, NV>(L, A, A.weight, w);
  params<T, VEC, NV>(L, A, A.branch_weight, bw);
  params<T, VEC, NV>(L, A, A.scale, sc);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    zero_vals<VEC>(gw[i]);
    zero_vals<VEC>(gb[i]);
    zero_vals<VEC>(gs[i]);
  }
  const float inv = 1.f / A.g.size;
  for (; m < A.g.M; m += step) {
    float h[NV][VEC], b[NV][VEC], a[NV][VEC], d[NV][VEC], e[NV][VEC];
    if (!kAhead) next(m);
    hr.get(h);
    br.get(b);
    dr.get(d);
    er.get(e);
    if (GATE) ar.get(a);
    if (kAhead) next(m + step);
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        s[0] += h[i][j] * h[i][j];
        s[1] += b[i][j] * b[i][j];
        s[2] += d[i][j] * w[i][j] * h[i][j];
      }
    row_sum<WIDE>(s, red, slot);
    const float rh = gn::rsqrt_of(s[0] * inv + A.g.eps), rb = gn::rsqrt_of(s[1] * inv + A.g.eps);
    const float c = s[2] * inv * rh * rh;
    float t[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        gw[i][j] += d[i][j] * (h[i][j] * rh);
        const float dx = e[i][j] + rh * (d[i][j] * w[i][j] - h[i][j] * c), bh = b[i][j] * rb;
        e[i][j] = dx;
        float f = 1.f, df = 0.f;
        if (GATE) activate(A.g.act, a[i][j], f, df);
        const float n = bh * bw[i][j], dn = dx * (A.constant * sc[i][j]) * f;
        gs[i][j] += A.constant * dx * n * f;
        gb[i][j] += dn * bh;
        a[i][j] = dx * n * (A.constant * sc[i][j]) * df;
        b[i][j] = bh;
        d[i][j] = dn * bw[i][j];
        t[0] += d[i][j] * bh;
      }
    leave<XT, VEC, NV>(L, A.dx, m, D, e);
    if (GATE) leave<T, VEC, NV>(L, A.dgate, m, D, a);
    row_sum<WIDE>(t, red, slot);
    const float c2 = t[0] * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) d[i][j] = rb * (d[i][j] - b[i][j] * c2);
    leave<T, VEC, NV>(L, A.dbranch, m, D, d);
    if (kAhead) {
      arrived(hr);
      arrived(br);
      arrived(dr);
      arrived(er);
      if (GATE) arrived(ar);
    }
  }
  auto write = [&](float* out, float (&v)[NV][VEC]) {
    if (!out) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float* to = out + (int64_t)blockIdx.y * D + L.ch + i * L.step;
      if constexpr (WIDE) {  // a channel has one lane of the workgroup
        if (L.live[i])
#pragma unroll
          for (int j = 0; j < VEC; ++j) to[j] = v[i][j];
      } else {  // the wavefronts' sums meet in LDS
        const int lane = threadIdx.x % 64, wv = threadIdx.x / 64;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[wv][j * 64 + lane] = v[i][j];
        __syncthreads();
        if (wv == 0 && L.live[i])
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int c = j * 64 + lane;
            to[j] = (sum[0][c] + sum[1][c]) + (sum[2][c] + sum[3][c]);
          }
      }
    }
  };
  write(A.pw, gw);
  write(A.pb, gb);
  write(A.ps, gs);
}

// Pieces of VEC channels; rows in a wavefront or (wide) in a workgroup, nv pieces to a lane.
struct Plan {
  int vec, nv;
  bool wide;
  int64_t gy;
};

template <typename T, typename XT, int VEC, int NV, bool WIDE>
hipError_t launch(bool bwd, const Args& a, const Plan& pl, hipStream_t st) {
  const dim3 grid(1, (unsigned)pl.gy);
  auto run = [&](auto kernel) { kernel<<<grid, 64 * kWaves, 0, st>>>(a); };
  if (bwd) run(a.gate ? rn_bwd_kernel<T, XT, VEC, NV, WIDE, true> : rn_bwd_kernel<T, XT, VEC, NV, WIDE, false>);
  else run(a.gate ? rn_fwd_kernel<T, XT, VEC, NV, WIDE, true> : rn_fwd_kernel<T, XT, VEC, NV, WIDE, false>);
  return hipGetLastError();
}

template <typename T, typename XT, int VEC>
hipError_t launch_nv(bool bwd, const Args& a, const Plan& pl, hipStream_t st) {
  if (!pl.wide) {
    if (pl.nv * VEC > 16) return hipErrorInvalidValue;
    if constexpr (VEC == 1) return launch<T, XT, VEC, 16, false>(bwd, a, pl, st);
    else if (pl.nv == 1) return launch<T, XT, VEC, 1, false>(bwd, a, pl, st);
    else return launch<T, XT, VEC, 16 / VEC, false>(bwd, a, pl, st);
  }
  const int n = pl.nv * VEC;  // channels of a lane
  if constexpr (VEC == 8)
    if (n <= 8) return launch<T, XT, VEC, 1, true>(bwd, a, pl, st);
  if (n <= 16) return launch<T, XT, VEC, 16 / VEC, true>(bwd, a, pl, st);
  return launch<T, XT, VEC, 32 / VEC, true>(bwd, a, pl, st);
}

// Every piece size of one type: 16 bytes of the branch's type, 8 bytes, one channel (instantiated in
// residual_norm_<type>.hip).
template <typename T>
hipError_t launch_vec(bool bwd, const Args& a, const Plan& pl, bool wide_x, hipStream_t st) {
  constexpr int V16 = 16 / (int)sizeof(T);
  auto go = [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    if constexpr (!__is_same(T, float))
      if (wide_x) return launch_nv<T, float, VEC>(bwd, a, pl, st);
    return launch_nv<T, T, VEC>(bwd, a, pl, st);
  };
  if (pl.vec == V16) return go(std::integral_constant<int, V16>());
  if (pl.vec == V16 / 2) return go(std::integral_constant<int, V16 / 2>());
  return go(std::integral_constant<int, 1>());
}
extern template hipError_t launch_vec<bf16>(bool, const Args&, const Plan&, bool, hipStream_t);
extern template hipError_t launch_vec<fp16>(bool, const Args&, const Plan&, bool, hipStream_t);
extern template hipError_t launch_vec<float>(bool, const Args&, const Plan&, bool, hipStream_t);

}  // namespace rn
}  // namespace dc
