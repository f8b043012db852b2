// Group norm over the channels of each row, with an activation or a gate
// (include/dynconv_layer.h), and its gradients:
//
//   xh = (x - mean) rstd,   u = xh w + b,   y = u act(gate)  or  act(u)
//   du = dy act(gate)  or  dy act'(u),      dgate = dy u act'(gate)
//   dw = sum_rows du xh,   db = sum_rows du
//   dx = rstd (du w - mean(du w) - xh mean(du w xh))
//
// Streams, bound by HBM: forward x, gate in and y out; backward x, gate, dy in
// and dx, dgate out, each once.  A group's channels stay in the registers of L
// neighbouring lanes (NV pieces of VEC channels each; L a power of two up to 64,
// so that 64 / L groups share a wavefront): mean, then the sum of squares of the
// differences, both in float32 from the registers, so large means cost no digits.  A
// wavefront keeps its channels and walks rows: weight and bias stay in registers, and
// in the backward dw and db too.  Each workgroup writes them once, as partial sums
// that reduce_partials adds in a fixed order.  The backward forms mean and rstd again
// from x instead of reading them: no statistics go through memory.
#pragma once

#include "dc_common.h"
#include "layer_launch.h"

namespace dc {
namespace gn {

constexpr int kWaves = 4;

struct GnArgs {
  const void *x, *weight, *bias, *gate, *dy;
  void *y, *dx, *dgate;
  float *pw, *pb;  // partial sums of dw and db, [row blocks][D] each (null: not wanted)
  int64_t M, D;
  int size, lanes;  // channels of a group, lanes it takes (a power of two)
  int pdtype;
  float eps;
  int act;
};

__device__ __forceinline__ float param(const void* p, int64_t i, int dtype, float none) {
  if (!p) return none;
  return dtype == kBF16 ? (float)((const bf16*)p)[i] : dtype == kFP16 ? (float)((const fp16*)p)[i] : ((const float*)p)[i];
}

// Sum over the group's lanes: every lane gets it.
__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int m = 1; m < lanes; m *= 2) v += __shfl_xor(v, m);
  return v;
}

__device__ __forceinline__ float sigmoid(float a) { return 1.f / (1.f + __expf(-a)); }

// What a lane holds: its group, its channels, and which of its pieces exist.
template <int VEC, int NV>
struct Lane {
  int64_t ch;       // first channel
  bool live[NV];    // piece i: channels ch + i * lanes * VEC ..
  int step;         // channels from a piece to the next
  __device__ __forceinline__ Lane(const GnArgs& A) {
    const int lane = threadIdx.x % 64, gl = lane & (A.lanes - 1);
    const int64_t group = (int64_t)blockIdx.x * (64 / A.lanes) + lane / A.lanes;
    step = A.lanes * VEC;
    ch = group * A.size + gl * VEC;
#pragma unroll
    for (int i = 0; i < NV; ++i) live[i] = group * A.size < A.D && gl * VEC + i * step < A.size;
  }
};

template <typename T, int VEC, int NV>
__device__ __forceinline__ void load_row(const Lane<VEC, NV>& L, const void* p, int64_t row, float (&v)[NV][VEC]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (L.live[i]) load_vals<T, VEC>((const T*)p + row + L.ch + i * L.step, v[i]);
    else zero_vals<VEC>(v[i]);
  }
}
template <typename T, int VEC, int NV>
__device__ __forceinline__ void store_row(const Lane<VEC, NV>& L, void* p, int64_t row, const float (&v)[NV][VEC]) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (L.live[i]) store_vals<T, VEC>((T*)p + row + L.ch + i * L.step, v[i]);
}

// x -> xh in place; returns rstd.
template <int VEC, int NV>
__device__ __forceinline__ float normalise(const Lane<VEC, NV>& L, const GnArgs& A, float (&x)[NV][VEC]) {
  const float inv = 1.f / A.size;
  float s = 0.f, s2 = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += x[i][j];
  const float mean = group_sum(s, A.lanes) * inv;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      x[i][j] = L.live[i] ? x[i][j] - mean : 0.f;
      s2 += x[i][j] * x[i][j];
    }
  const float rstd = 1.f / sqrtf(group_sum(s2, A.lanes) * inv + A.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[i][j] *= rstd;
  return rstd;
}

template <int VEC, int NV>
__device__ __forceinline__ void load_params(const Lane<VEC, NV>& L, const GnArgs& A, float (&w)[NV][VEC],
                                            float (&b)[NV][VEC]) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      w[i][j] = L.live[i] ? param(A.weight, L.ch + i * L.step + j, A.pdtype, 1.f) : 0.f;
      b[i][j] = L.live[i] ? param(A.bias, L.ch + i * L.step + j, A.pdtype, 0.f) : 0.f;
    }
}

template <typename T, int VEC, int NV>
__global__ __launch_bounds__(64 * kWaves) void gn_fwd_kernel(GnArgs A) {
  const Lane<VEC, NV> L(A);
  float w[NV][VEC], b[NV][VEC];
  load_params<VEC, NV>(L, A, w, b);
  for (int64_t m = (int64_t)blockIdx.y * kWaves + wave_id(); m < A.M; m += (int64_t)gridDim.y * kWaves) {
    float x[NV][VEC], a[NV][VEC];
    load_row<T, VEC, NV>(L, A.x, m * A.D, x);
    if (A.gate) load_row<T, VEC, NV>(L, A.gate, m * A.D, a);
    normalise<VEC, NV>(L, A, x);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float u = x[i][j] * w[i][j] + b[i][j];
        const float sg = A.act ? sigmoid(A.gate ? a[i][j] : u) : 1.f;
        x[i][j] = A.gate ? u * (a[i][j] * sg) : u * sg;
      }
    store_row<T, VEC, NV>(L, A.y, m * A.D, x);
  }
}

template <typename T, int VEC, int NV>
__global__ __launch_bounds__(64 * kWaves) void gn_bwd_kernel(GnArgs A) {
  __shared__ float red[kWaves][64 * VEC];
  const Lane<VEC, NV> L(A);
  float w[NV][VEC], b[NV][VEC], dw[NV][VEC], db[NV][VEC];
  load_params<VEC, NV>(L, A, w, b);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    zero_vals<VEC>(dw[i]);
    zero_vals<VEC>(db[i]);
  }
  const float inv = 1.f / A.size;
  for (int64_t m = (int64_t)blockIdx.y * kWaves + wave_id(); m < A.M; m += (int64_t)gridDim.y * kWaves) {
    float x[NV][VEC], du[NV][VEC], a[NV][VEC];
    load_row<T, VEC, NV>(L, A.x, m * A.D, x);
    load_row<T, VEC, NV>(L, A.dy, m * A.D, du);
    if (A.gate) load_row<T, VEC, NV>(L, A.gate, m * A.D, a);
    const float rstd = normalise<VEC, NV>(L, A, x);
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float u = x[i][j] * w[i][j] + b[i][j];
        const float in = A.gate ? a[i][j] : u, sg = A.act ? sigmoid(in) : 1.f;
        const float d1 = A.act ? sg * (1.f + in * (1.f - sg)) : 1.f;  // act'(in)
        if (A.gate) {
          a[i][j] = du[i][j] * u * d1;
          du[i][j] *= in * sg;
        } else {
          du[i][j] *= d1;
        }
        dw[i][j] += du[i][j] * x[i][j];
        db[i][j] += du[i][j];
        du[i][j] *= w[i][j];
        c1 += du[i][j];
        c2 += du[i][j] * x[i][j];
      }
    c1 = group_sum(c1, A.lanes) * inv;
    c2 = group_sum(c2, A.lanes) * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) du[i][j] = rstd * (du[i][j] - c1 - x[i][j] * c2);
    store_row<T, VEC, NV>(L, A.dx, m * A.D, du);
    if (A.gate) store_row<T, VEC, NV>(L, A.dgate, m * A.D, a);
  }
  // the wavefronts' sums, piece by piece through LDS
  if (!A.pw && !A.pb) return;
  const int lane = threadIdx.x % 64, wv = threadIdx.x / 64;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float* out = t ? A.pb : A.pw;
      if (!out) continue;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < VEC; ++j) red[wv][j * 64 + lane] = t ? db[i][j] : dw[i][j];
      __syncthreads();
      if (wv == 0 && L.live[i])
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int c = j * 64 + lane;
          out[(int64_t)blockIdx.y * A.D + L.ch + i * L.step + j] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
        }
    }
}

// Pieces of VEC channels, lanes of a group and pieces of a lane.
struct Plan {
  int vec, lanes, nv;
  unsigned gx;
  int64_t gy;
};

template <typename T, int VEC, int NV>
void launch(bool bwd, const GnArgs& a, const Plan& pl, hipStream_t st) {
  const dim3 grid(pl.gx, (unsigned)pl.gy);
  if (bwd) gn_bwd_kernel<T, VEC, NV><<<grid, 64 * kWaves, 0, st>>>(a);
  else gn_fwd_kernel<T, VEC, NV><<<grid, 64 * kWaves, 0, st>>>(a);
}

// Lanes hold at most 64 channels (a group of 4096 over 64 lanes).
template <typename T, int VEC>
hipError_t launch_nv(bool bwd, const GnArgs& a, const Plan& pl, hipStream_t st) {
  switch (pl.nv) {
    case 1: launch<T, VEC, 1>(bwd, a, pl, st); break;
    case 2:
      if constexpr (VEC > 1) launch<T, VEC, 2>(bwd, a, pl, st);
      break;
    case 4:
      if constexpr (VEC > 1) launch<T, VEC, 4>(bwd, a, pl, st);
      break;
    case 8: launch<T, VEC, 8>(bwd, a, pl, st); break;
    case 16:
      if constexpr (VEC == 2 || VEC == 4) launch<T, VEC, 16>(bwd, a, pl, st);
      break;
    case 32:
      if constexpr (VEC == 2) launch<T, VEC, 32>(bwd, a, pl, st);
      break;
    default:
      if constexpr (VEC == 1) launch<T, VEC, 64>(bwd, a, pl, st);
      break;
  }
  return hipGetLastError();
}

// Every piece size of one type: 16 bytes, 8 bytes, one channel (instantiated in group_norm_<type>.hip).
template <typename T>
hipError_t launch_vec(bool bwd, const GnArgs& a, const Plan& pl, hipStream_t st) {
  constexpr int V16 = 16 / (int)sizeof(T);
  if (pl.vec == V16) return launch_nv<T, V16>(bwd, a, pl, st);
  if (pl.vec == V16 / 2) return launch_nv<T, V16 / 2>(bwd, a, pl, st);
  return launch_nv<T, 1>(bwd, a, pl, st);
}
extern template hipError_t launch_vec<bf16>(bool, const GnArgs&, const Plan&, hipStream_t);
extern template hipError_t launch_vec<fp16>(bool, const GnArgs&, const Plan&, hipStream_t);
extern template hipError_t launch_vec<float>(bool, const GnArgs&, const Plan&, hipStream_t);

}  // namespace gn
}  // namespace dc
