// The gated delta rule, one token of each of B sequences (dc_delta_rule_step):
//
//   u = b (v - a k S),   o = scale (a q S + (q.k) u),   S <- a S + k^T u        (in place, float32)
//
// Bound by the state, K x V floats read and written for each sequence and head.  A workgroup takes 8 lanes of VEC columns
// times 32 rows of one head's state, as linear attention's step does; k S and q S come from the same pass over it, so the
// rows' parts of both meet once (lane exchanges, then LDS), and the state, kept in registers, is written with its
// correction.  256 sequences of 32 heads of 128 x 128: 242 us for 1.08 GB, 4.5 TB/s (16 lanes 258,
// 32 280, 4 328); 8 of 16 heads 6.5 us, the launch.
#include "dc_common.h"
#include "layer_launch.h"

namespace dc {
namespace {

constexpr int kLanes = 8, kRows = 32;  // lanes of VEC columns, rows in flight

__device__ __forceinline__ float gate_of(const void* t, int gdtype, int64_t i) {
  return gdtype == kBF16 ? (float)((const bf16*)t)[i] : gdtype == kFP16 ? (float)((const fp16*)t)[i] : ((const float*)t)[i];
}

template <typename T, int VEC, int KR>
__global__ __launch_bounds__(256) void dr_step_kernel(DrStep p) {
  typedef float vec __attribute__((ext_vector_type(VEC)));
  __shared__ vec red[2][4][kLanes];
  __shared__ float dots[4][3];
  const int nv = (int)((p.V + kLanes * VEC - 1) / (kLanes * VEC));
  const int64_t bh = p.bh0 + blockIdx.x / nv;
  const int64_t b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
  const int lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const int64_t col = ((int64_t)(blockIdx.x % nv) * kLanes + lane) * VEC;
  const bool live = col < p.V;
  T* o = (T*)p.o + bh * p.V + col;
  const int64_t slot = p.slot_ids ? p.slot_ids[b] : b;
  if (slot < 0 || slot >= p.slots) {
    if (row == 0 && live)
#pragma unroll
      for (int j = 0; j < VEC; ++j) o[j] = (T)0.f;
    return;
  }
  float* S = p.state + (slot * p.H + h) * p.K * p.V + col;
  const T* q = (const T*)p.q + b * p.qs[0] + hk * p.qs[1];
  const T* k = (const T*)p.k + b * p.ks[0] + hk * p.ks[1];
  const T* v = (const T*)p.v + b * p.vs[0] + h * p.vs[1] + col;
  vec s[KR], vv = 0.f, ks = 0.f, qs = 0.f;
  float kk[KR], qq[KR], d[3] = {0.f, 0.f, 0.f};  // k.k, q.q, q.k
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int a = row + i * kRows;
    const bool in = a < p.K;
    s[i] = live && in ? *reinterpret_cast<const vec*>(S + a * p.V) : (vec)0.f;
    kk[i] = in ? (float)k[a] : 0.f;
    qq[i] = in ? (float)q[a] : 0.f;
  }
  if (live)
#pragma unroll
    for (int j = 0; j < VEC; ++j) vv[j] = (float)v[j];
  const float a = expf(gate_of(p.g, p.gdtype, b * p.gs[0] + h * p.gs[1]));
  const float be = gate_of(p.b, p.gdtype, b * p.bs[0] + h * p.bs[1]);
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    ks += kk[i] * s[i];
    qs += qq[i] * s[i];
    d[0] += kk[i] * kk[i];
    d[1] += qq[i] * qq[i];
    d[2] += qq[i] * kk[i];
  }
  // the wavefront's 8 rows, then the four wavefronts
#pragma unroll
  for (int m = kLanes; m < 64; m *= 2) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      ks[j] += __shfl_xor(ks[j], m);
      qs[j] += __shfl_xor(qs[j], m);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) d[j] += __shfl_xor(d[j], m);
  }
  const int wv = threadIdx.x / 64;
  if (threadIdx.x % 64 < kLanes) {
    red[0][wv][lane] = ks;
    red[1][wv][lane] = qs;
  }
  if (threadIdx.x % 64 == 0)
#pragma unroll
    for (int j = 0; j < 3; ++j) dots[wv][j] = d[j];
  __syncthreads();
  if (!live) return;
  ks = (red[0][0][lane] + red[0][1][lane]) + (red[0][2][lane] + red[0][3][lane]);
  qs = (red[1][0][lane] + red[1][1][lane]) + (red[1][2][lane] + red[1][3][lane]);
#pragma unroll
  for (int j = 0; j < 3; ++j) d[j] = (dots[0][j] + dots[1][j]) + (dots[2][j] + dots[3][j]);
  const float rk = p.normalize ? 1.f / sqrtf(d[0] + p.eps) : 1.f, rq = p.normalize ? 1.f / sqrtf(d[1] + p.eps) : 1.f;
  const vec u = be * (vv - (a * rk) * ks);
  if (row == 0) {
    const vec out = (p.scale * rq) * (a * qs + (d[2] * rk) * u);
#pragma unroll
    for (int j = 0; j < VEC; ++j) o[j] = (T)out[j];
  }
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int r = row + i * kRows;
    if (r < p.K) *reinterpret_cast<vec*>(S + r * p.V) = a * s[i] + (kk[i] * rk) * u;
  }
}

template <typename T, int VEC>
hipError_t launch(const DrStep& p) {
  const int64_t nv = (p.V + kLanes * VEC - 1) / (kLanes * VEC), heads = p.B * p.H, per = most_workgroups(256) / nv;
  DrStep q = p;
  for (q.bh0 = 0; q.bh0 < heads; q.bh0 += per) {
    const dim3 grid((unsigned)((heads - q.bh0 < per ? heads - q.bh0 : per) * nv));
    if (p.K <= 32) dr_step_kernel<T, VEC, 1><<<grid, 256, 0, p.stream>>>(q);
    else if (p.K <= 64) dr_step_kernel<T, VEC, 2><<<grid, 256, 0, p.stream>>>(q);
    else if (p.K <= 128) dr_step_kernel<T, VEC, 4><<<grid, 256, 0, p.stream>>>(q);
    else dr_step_kernel<T, VEC, 8><<<grid, 256, 0, p.stream>>>(q);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launch_vec(const DrStep& p) {
  // four columns to a lane where rows of the state are whole 16-byte pieces
  const bool v4 = p.V % 4 == 0 && reinterpret_cast<uintptr_t>(p.state) % 16 == 0;
  return v4 ? launch<T, 4>(p) : launch<T, 1>(p);
}

}  // namespace

hipError_t dr_step(const DrStep& p) {
  switch (p.dtype) {
    case kBF16: return launch_vec<bf16>(p);
    case kFP16: return launch_vec<fp16>(p);
    default: return launch_vec<float>(p);
  }
}

}  // namespace dc
