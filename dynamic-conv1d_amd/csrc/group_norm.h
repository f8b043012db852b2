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
// differences, both in float32 from the registers, so large means cost no digits (a group of more than 128 pieces
// takes the workgroup's 256 lanes).  A
// wavefront keeps its channels and walks rows: weight and bias stay in registers, and
// in the backward dw and db too.  Each workgroup writes them once, as partial sums
// that reduce_partials adds in a fixed order.  The backward forms mean and rstd again
// from x instead of reading them: no statistics go through memory.
//
// Measured: 16384 rows of 4096 channels in 32 groups, gated, bf16: forward 72 us (5.6 TB/s), backward 126 (5.3 TB/s) and
// 5 for the partial sums; 4611 rows of 1000 channels in 10 groups, fp16, no gate: 10.7, 16.3 and 4.9, in 63 with the
// autograd engine (groups of 100 channels go in 8-byte pieces, 25 of 32 lanes live: vector instructions fill 93% of the
// forward's cycles and 85% of the backward's); 8 rows of 2048 forward 3.7, one round trip.
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
  int64_t gx0;      // first block of groups of a launch
  bool wide_params;   // weight and bias are float32 (else of x's type)
  bool param_pieces;  // and 16-byte aligned
  float eps;
  int act;
};

// Sum over the group's lanes: every lane gets it.  Up to 16 lanes by data moves within the registers' rows (each step's
// partner holds the other half's sum), beyond through the exchange network.
__device__ __forceinline__ float lane_sum(float v, int lanes) {
  if (lanes > 1) v += dpp_f<0xB1>(v);   // pairs
  if (lanes > 2) v += dpp_f<0x4E>(v);   // quads
  if (lanes > 4) v += dpp_f<0x141>(v);  // the mirrored lane of 8
  if (lanes > 8) v += dpp_f<0x140>(v);  // of 16
  if (lanes > 16) v += __shfl_xor(v, 16);
  if (lanes > 32) v += __shfl_xor(v, 32);
  return v;
}

// N sums over a group at once.  WIDE: over the workgroup, the wavefronts' sums meeting in LDS (`slot` alternates, so one
// barrier serves).
template <bool WIDE, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], int lanes, float (*red)[kWaves][2], int& slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane_sum(v[i], WIDE ? 64 : lanes);
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

// With the reciprocal instruction (one last place of float32): the division's steps were a quarter of the forward's vector
// instructions, which filled 87% of the SIMDs' cycles (forward 88 -> 73 us).
__device__ __forceinline__ float sigmoid(float a) { return __builtin_amdgcn_rcpf(1.f + __expf(-a)); }

// v^-1/2 by its instruction (one last place), which wants a normal v.
__device__ __forceinline__ float rsqrt_of(float v) {
  const bool tiny = v < 0x1p-100f;
  return __builtin_amdgcn_rsqf(tiny ? v * 0x1p64f : v) * (tiny ? 0x1p32f : 1.f);
}

// What a lane holds: its group, its channels, and which of its pieces exist.
template <int VEC, int NV>
struct Lane {
  int64_t ch;       // first channel
  bool live[NV];    // piece i: channels ch + i * lanes * VEC ..
  int step;         // channels from a piece to the next
  __device__ __forceinline__ Lane(const GnArgs& A) {
    // a group of more lanes than a wavefront's has the workgroup
    const int lane = A.lanes > 64 ? threadIdx.x : threadIdx.x % 64, gl = lane & (A.lanes - 1);
    const int64_t group = (A.gx0 + blockIdx.x) * (A.lanes > 64 ? 1 : 64 / A.lanes) + lane / A.lanes;
    step = A.lanes * VEC;
    ch = group * A.size + gl * VEC;
#pragma unroll
    for (int i = 0; i < NV; ++i) live[i] = group * A.size < A.D && gl * VEC + i * step < A.size;
  }
};

// A row's pieces as they come from memory: on their way while the row before is computed.
template <typename T, int VEC, int NV>
struct Row {
  Raw<T, VEC> v[NV];
  __device__ __forceinline__ void load(const Lane<VEC, NV>& L, const void* p, int64_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (L.live[i]) v[i].load((const T*)p + row + L.ch + i * L.step);
      else v[i].zero();
    }
  }
  __device__ __forceinline__ void get(float (&f)[NV][VEC]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i].to_float(f[i]);
  }
};
template <typename T, int VEC, int NV>
__device__ __forceinline__ void store_row(const Lane<VEC, NV>& L, void* p, int64_t row, const float (&v)[NV][VEC]) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (L.live[i]) store_vals<T, VEC, VEC * sizeof(T) == 16>((T*)p + row + L.ch + i * L.step, v[i]);
}

// x -> xh in place; returns rstd.
template <bool WIDE, int VEC, int NV>
__device__ __forceinline__ float normalise(const Lane<VEC, NV>& L, const GnArgs& A, float (*red)[kWaves][2], int& slot,
                                           float (&x)[NV][VEC]) {
  const float inv = 1.f / A.size;
  float s[1] = {0.f}, s2[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[0] += x[i][j];
  group_sum<WIDE>(s, A.lanes, red, slot);
  const float mean = s[0] * inv;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      x[i][j] = L.live[i] ? x[i][j] - mean : 0.f;
      s2[0] += x[i][j] * x[i][j];
    }
  group_sum<WIDE>(s2, A.lanes, red, slot);
  const float rstd = rsqrt_of(s2[0] * inv + A.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[i][j] *= rstd;
  return rstd;
}

// weight and bias of the lane's channels, of type P (T or float)
template <typename P, int VEC, int NV>
__device__ __forceinline__ void load_param(const Lane<VEC, NV>& L, const void* p, bool pieces, float none,
                                           float (&v)[NV][VEC]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i][j] = L.live[i] ? none : 0.f;
    if (p && L.live[i]) {
      const P* q = (const P*)p + L.ch + i * L.step;
      if (pieces) {
        load_vals<P, VEC>(q, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = (float)q[j];
      }
    }
  }
}
template <typename T, int VEC, int NV>
__device__ __forceinline__ void load_params(const Lane<VEC, NV>& L, const GnArgs& A, float (&w)[NV][VEC],
                                            float (&b)[NV][VEC]) {
  if (A.wide_params) {
    load_param<float, VEC, NV>(L, A.weight, A.param_pieces, 1.f, w);
    load_param<float, VEC, NV>(L, A.bias, A.param_pieces, 0.f, b);
  } else {
    load_param<T, VEC, NV>(L, A.weight, A.param_pieces, 1.f, w);
    load_param<T, VEC, NV>(L, A.bias, A.param_pieces, 0.f, b);
  }
}

template <typename T, int VEC, int NV, bool WIDE>
__global__ __launch_bounds__(64 * kWaves) void gn_fwd_kernel(GnArgs A) {
  __shared__ float red[2][kWaves][2];
  int slot = 0;
  const Lane<VEC, NV> L(A);
  const int64_t step = (int64_t)gridDim.y * (WIDE ? 1 : kWaves);
  int64_t m = WIDE ? (int64_t)blockIdx.y : (int64_t)blockIdx.y * kWaves + wave_id();
  if (m >= A.M) return;
  Row<T, VEC, NV> xr, ar;
  xr.load(L, A.x, m * A.D);
  if (A.gate) ar.load(L, A.gate, m * A.D);
  float w[NV][VEC], b[NV][VEC];
  load_params<T, VEC, NV>(L, A, w, b);
  for (; m < A.M; m += step) {
    float x[NV][VEC], a[NV][VEC];
    xr.get(x);
    if (A.gate) ar.get(a);
    if (m + step < A.M) {
      xr.load(L, A.x, (m + step) * A.D);
      if (A.gate) ar.load(L, A.gate, (m + step) * A.D);
    }
    normalise<WIDE, VEC, NV>(L, A, red, slot, x);
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

template <typename T, int VEC, int NV, bool WIDE>
__global__ __launch_bounds__(64 * kWaves) void gn_bwd_kernel(GnArgs A) {
  __shared__ float red[2][kWaves][2], sum[WIDE ? 1 : kWaves][WIDE ? 1 : 64 * VEC];
  int slot = 0;
  const Lane<VEC, NV> L(A);
  const int64_t step = (int64_t)gridDim.y * (WIDE ? 1 : kWaves);
  int64_t m = WIDE ? (int64_t)blockIdx.y : (int64_t)blockIdx.y * kWaves + wave_id();
  Row<T, VEC, NV> xr, dr, ar;
  auto fetch = [&](int64_t row) {
    if (row >= A.M) return;
    xr.load(L, A.x, row * A.D);
    dr.load(L, A.dy, row * A.D);
    if (A.gate) ar.load(L, A.gate, row * A.D);
  };
  fetch(m);
  float w[NV][VEC], b[NV][VEC], dw[NV][VEC], db[NV][VEC];
  load_params<T, VEC, NV>(L, A, w, b);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    zero_vals<VEC>(dw[i]);
    zero_vals<VEC>(db[i]);
  }
  const float inv = 1.f / A.size;
  for (; m < A.M; m += step) {
    float x[NV][VEC], du[NV][VEC], a[NV][VEC];
    xr.get(x);
    dr.get(du);
    if (A.gate) ar.get(a);
    fetch(m + step);
    const float rstd = normalise<WIDE, VEC, NV>(L, A, red, slot, x);
    float c[2] = {0.f, 0.f};
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
        c[0] += du[i][j];
        c[1] += du[i][j] * x[i][j];
      }
    group_sum<WIDE>(c, A.lanes, red, slot);
    const float c1 = c[0] * inv, c2 = c[1] * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) du[i][j] = rstd * (du[i][j] - c1 - x[i][j] * c2);
    store_row<T, VEC, NV>(L, A.dx, m * A.D, du);
    if (A.gate) store_row<T, VEC, NV>(L, A.dgate, m * A.D, a);
  }
  if (!A.pw && !A.pb) return;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float* out = t ? A.pb : A.pw;
      if (!out) continue;
      out += (int64_t)blockIdx.y * A.D + L.ch + i * L.step;
      if constexpr (WIDE) {  // a channel has one lane of the workgroup
        if (L.live[i])
#pragma unroll
          for (int j = 0; j < VEC; ++j) out[j] = t ? db[i][j] : dw[i][j];
      } else {  // the wavefronts' sums meet in LDS
        const int lane = threadIdx.x % 64, wv = threadIdx.x / 64;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[wv][j * 64 + lane] = t ? db[i][j] : dw[i][j];
        __syncthreads();
        if (wv == 0 && L.live[i])
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int c = j * 64 + lane;
            out[j] = (sum[0][c] + sum[1][c]) + (sum[2][c] + sum[3][c]);
          }
      }
    }
}

// Pieces of VEC channels, lanes of a group and pieces of a lane.
struct Plan {
  int vec, lanes, nv;
  unsigned gx;
  int64_t gy;
};

template <typename T, int VEC, int NV, bool WIDE>
void launch(bool bwd, const GnArgs& args, const Plan& pl, hipStream_t st) {
  constexpr int64_t most = most_workgroups(64 * kWaves);
  GnArgs a = args;
  for (a.gx0 = 0; a.gx0 < pl.gx; a.gx0 += most) {
    const dim3 grid((unsigned)(pl.gx - a.gx0 < most ? pl.gx - a.gx0 : most), (unsigned)pl.gy);
    if (bwd) gn_bwd_kernel<T, VEC, NV, WIDE><<<grid, 64 * kWaves, 0, st>>>(a);
    else gn_fwd_kernel<T, VEC, NV, WIDE><<<grid, 64 * kWaves, 0, st>>>(a);
  }
}

// A group of up to 128 pieces lies in one wavefront, a larger one (up to 4096 channels) in the workgroup.
template <typename T, int VEC>
hipError_t launch_nv(bool bwd, const GnArgs& a, const Plan& pl, hipStream_t st) {
  if (pl.lanes <= 64) {
    if (pl.nv == 1) launch<T, VEC, 1, false>(bwd, a, pl, st);
    else launch<T, VEC, 2, false>(bwd, a, pl, st);
    return hipGetLastError();
  }
  switch (pl.nv) {
    case 1: launch<T, VEC, 1, true>(bwd, a, pl, st); break;
    case 2: launch<T, VEC, 2, true>(bwd, a, pl, st); break;
    case 4:
      if constexpr (VEC <= 4) launch<T, VEC, 4, true>(bwd, a, pl, st);
      break;
    case 8:
      if constexpr (VEC <= 2) launch<T, VEC, 8, true>(bwd, a, pl, st);
      break;
    default:
      if constexpr (VEC == 1) launch<T, VEC, 16, true>(bwd, a, pl, st);
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
