// Linear attention, one token of each of B sequences (dc_linear_attention_step):
//
//   S <- g S + k^T v (in place, float32),   o = scale * q S
//
// Bound by the state: K x V floats read and written for each sequence and head
// (128 KB at 128 x 128), against 2 K + 2 V activations.  A workgroup takes 32
// columns of one head's state (whole 128-byte lines of its rows): 8 lanes of
// four columns times 32 rows, so that at K 128 a thread has its four pieces of
// the state in flight at once and four workgroups share a head, which keeps a
// batch of 8 x 16 heads on every CU.  The 32 rows' parts of o meet through
// lane exchanges and one pass over LDS.  Measured at 128 x 128, bf16: 256 sequences x 32 heads 226 us (1.08 GB, 4.8
// TB/s, the rate of a large copy less 7%), 8 x 16 heads 5.0 us (17 MB, left in the last-level cache by the step before).
#include "dc_common.h"
#include "layer_launch.h"

namespace dc {
namespace {

constexpr int kLanes = 8, kRows = 32;  // lanes of VEC columns, rows in flight

template <typename T, int VEC, int KR>
__global__ __launch_bounds__(256) void la_step_kernel(LaStep p) {
  typedef float vec __attribute__((ext_vector_type(VEC)));
  __shared__ vec red[4][kLanes];
  const int nv = (int)((p.V + kLanes * VEC - 1) / (kLanes * VEC));
  const int64_t bh = p.bh0 + blockIdx.x / nv;
  const int64_t b = bh / p.H, h = bh % p.H;
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
  const float g = expf(p.log_decay[h]);
  float* S = p.state + (slot * p.H + h) * p.K * p.V + col;
  const T* q = (const T*)p.q + b * p.qs[0] + h * p.qs[1];
  const T* k = (const T*)p.k + b * p.ks[0] + h * p.ks[1];
  const T* v = (const T*)p.v + b * p.vs[0] + h * p.vs[1] + col;
  vec s[KR], vv = 0.f, acc = 0.f;
  float kk[KR], qq[KR];
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int a = row + i * kRows;
    const bool in = live && a < p.K;
    s[i] = in ? *reinterpret_cast<const vec*>(S + a * p.V) : (vec)0.f;
    kk[i] = in ? (float)k[a] : 0.f;
    qq[i] = in ? (float)q[a] : 0.f;
  }
  if (live)
#pragma unroll
    for (int j = 0; j < VEC; ++j) vv[j] = (float)v[j];
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int a = row + i * kRows;
    s[i] = g * s[i] + kk[i] * vv;
    acc += qq[i] * s[i];
    if (live && a < p.K) *reinterpret_cast<vec*>(S + a * p.V) = s[i];
  }
  // the wavefront's 8 rows, then the four wavefronts
#pragma unroll
  for (int m = kLanes; m < 64; m *= 2)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += __shfl_xor(acc[j], m);
  if (threadIdx.x % 64 < kLanes) red[threadIdx.x / 64][lane] = acc;
  __syncthreads();
  if (row == 0 && live) {
    const vec t = ((red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane])) * p.scale;
#pragma unroll
    for (int j = 0; j < VEC; ++j) o[j] = (T)t[j];
  }
}

template <typename T, int VEC>
hipError_t launch(const LaStep& p) {
  const int64_t nv = (p.V + kLanes * VEC - 1) / (kLanes * VEC), heads = p.B * p.H, per = most_workgroups(256) / nv;
  LaStep q = p;
  for (q.bh0 = 0; q.bh0 < heads; q.bh0 += per) {
    const dim3 grid((unsigned)((heads - q.bh0 < per ? heads - q.bh0 : per) * nv));
    if (p.K <= 32) la_step_kernel<T, VEC, 1><<<grid, 256, 0, p.stream>>>(q);
    else if (p.K <= 64) la_step_kernel<T, VEC, 2><<<grid, 256, 0, p.stream>>>(q);
    else if (p.K <= 128) la_step_kernel<T, VEC, 4><<<grid, 256, 0, p.stream>>>(q);
    else la_step_kernel<T, VEC, 8><<<grid, 256, 0, p.stream>>>(q);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launch_vec(const LaStep& p) {
  // four columns to a lane where rows of the state are whole 16-byte pieces
  const bool v4 = p.V % 4 == 0 && reinterpret_cast<uintptr_t>(p.state) % 16 == 0;
  return v4 ? launch<T, 4>(p) : launch<T, 1>(p);
}

}  // namespace

hipError_t la_step(const LaStep& p) {
  switch (p.dtype) {
    case kBF16: return launch_vec<bf16>(p);
    case kFP16: return launch_vec<fp16>(p);
    default: return launch_vec<float>(p);
  }
}

}  // namespace dc
