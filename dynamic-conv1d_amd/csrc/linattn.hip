// Linear attention with a decay for each head (include/dynconv_layer.h).
//
//   S_t = g S_{t-1} + skv k_t^T v_t,    o_t = so q_t S_t,    g = exp(log_decay[h])
//
// The forward is one pass of this recurrence; the backward is three more, each
// the same recurrence on other tensors:
//   dq_t = s (S_t do_t)             forward in time on (do, v, k): state S^T
//   dk_t = (dS_t v_t)               backward in time on (v, do, q): state dS^T
//   dv_t = (k_t dS_t)               backward in time on (k, q, do): state dS
// with dS_t = g dS_{t+1} + s q_t^T do_t.  The gradient of the final state enters
// dS at the last token without a factor, and g dS_0 is the initial state's.
//
// This kernel walks the tokens one by one: a workgroup holds 64 columns of one
// head's state in registers, four threads to a column.
#include "dc_common.h"
#include "layer_launch.h"

namespace dc {
namespace {

constexpr int kCols = 64, kRowGroups = 4, kTile = 16;

template <typename T, int KR>
__global__ __launch_bounds__(256) void la_recurrent(LaProblem P) {
  constexpr int KP = KR * kRowGroups;
  __shared__ float sq[kTile][KP], sk[kTile][KP], sv[kTile][kCols], part[kTile][kRowGroups][kCols];
  const LaPass& p = P.pass[blockIdx.z];
  const int64_t b = blockIdx.x / P.H, h = blockIdx.x % P.H;
  const int n = threadIdx.x % kCols, rg = threadIdx.x / kCols;
  const int col0 = blockIdx.y * kCols, col = col0 + n;
  if (col0 >= p.V) return;
  const float g = expf(P.log_decay[h]);
  const int nt_all = (int)P.T;
  const int len = P.lengths ? min(max(P.lengths[b], 0), nt_all) : nt_all;
  const int64_t sbase = (int64_t)blockIdx.x * p.K * p.V;

  float S[KR];
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int a = rg * KR + i;
    S[i] = p.s_in && a < p.K && col < p.V ? p.s_in[sbase + a * p.s_row + col * p.s_col] : 0.f;
  }
  const T* q = (const T*)p.q + b * p.qs[0] + h * p.qs[1];
  const T* k = (const T*)p.k + b * p.ks[0] + h * p.ks[1];
  const T* v = (const T*)p.v + b * p.vs[0] + h * p.vs[1];
  T* o = (T*)p.o + b * p.os[0] + h * p.os[1];

  for (int t0 = 0; t0 < len; t0 += kTile) {
    const int nt = min(kTile, len - t0);
    for (int i = threadIdx.x; i < nt * KP; i += 256) {
      const int r = i / KP, a = i % KP;
      const int64_t t = p.rev ? len - 1 - t0 - r : t0 + r;
      sq[r][a] = a < p.K ? (float)q[t * p.qs[2] + a] : 0.f;
      sk[r][a] = a < p.K ? (float)k[t * p.ks[2] + a] : 0.f;
    }
    for (int i = threadIdx.x; i < nt * kCols; i += 256) {
      const int r = i / kCols, c = i % kCols;
      const int64_t t = p.rev ? len - 1 - t0 - r : t0 + r;
      sv[r][c] = col0 + c < p.V ? (float)v[t * p.vs[2] + col0 + c] * p.skv : 0.f;
    }
    __syncthreads();
    for (int r = 0; r < nt; ++r) {
      const float d = p.rev && t0 + r == 0 ? 1.f : g, vn = sv[r][n];
      float acc = 0.f;
#pragma unroll
      for (int i = 0; i < KR; ++i) {
        S[i] = d * S[i] + sk[r][rg * KR + i] * vn;
        acc += sq[r][rg * KR + i] * S[i];
      }
      part[r][rg][n] = acc;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nt * kCols; i += 256) {
      const int r = i / kCols, c = i % kCols;
      const int64_t t = p.rev ? len - 1 - t0 - r : t0 + r;
      if (col0 + c < p.V)
        o[t * p.os[2] + col0 + c] = (T)(p.so * ((part[r][0][c] + part[r][1][c]) + (part[r][2][c] + part[r][3][c])));
    }
  }
  for (int64_t i = threadIdx.x; i < (int64_t)(nt_all - len) * kCols; i += 256) {
    const int64_t t = len + i / kCols;
    const int c = i % kCols;
    if (col0 + c < p.V) o[t * p.os[2] + col0 + c] = (T)0.f;
  }
  if (p.s_out) {
    const float d = p.rev && len > 0 ? g : 1.f;
#pragma unroll
    for (int i = 0; i < KR; ++i) {
      const int a = rg * KR + i;
      if (a < p.K && col < p.V) p.s_out[sbase + a * p.s_row + col * p.s_col] = d * S[i];
    }
  }
}

template <typename T>
hipError_t launch_recurrent(const LaProblem& p) {
  int K = 0, V = 0;
  for (int i = 0; i < p.npass; ++i) {
    K = max(K, p.pass[i].K);
    V = max(V, p.pass[i].V);
  }
  const dim3 grid((unsigned)(p.B * p.H), (unsigned)((V + kCols - 1) / kCols), (unsigned)p.npass);
  if (K <= 32) la_recurrent<T, 8><<<grid, 256, 0, p.stream>>>(p);
  else if (K <= 64) la_recurrent<T, 16><<<grid, 256, 0, p.stream>>>(p);
  else if (K <= 128) la_recurrent<T, 32><<<grid, 256, 0, p.stream>>>(p);
  else la_recurrent<T, 64><<<grid, 256, 0, p.stream>>>(p);
  return hipGetLastError();
}

}  // namespace

int64_t la_ws_bytes(const LaProblem&) { return 0; }

hipError_t la_run(const LaProblem& p) {
  switch (p.dtype) {
    case kBF16: return launch_recurrent<bf16>(p);
    case kFP16: return launch_recurrent<fp16>(p);
    default: return launch_recurrent<float>(p);
  }
}

}  // namespace dc
