// The gated delta rule over whole sequences (include/dynconv_layer.h).
//
//   S' = a S,   u = b (v - k S'),   S <- S' + k^T u,   o = scale q S
//
// in chunks of C tokens.  With the state S before a chunk, c_i the sum of its logarithms of decays up to token i,
// G_i = e^{c_i}, E_ij = e^{c_i - c_j}, D_i = e^{c_C - c_i}, and q, k normed and q scaled:
//
//   A_ij = b_i E_ij k_i.k_j (j < i),   P_ij = E_ij q_i.k_j (j <= i),   Tb = (1 + A)^-1 diag(b)
//   X = V - G k S,   U = Tb X,   O = G q S + P U,   S <- G_C S + k^T D U
//
// and backward, dS the gradient of the state after the chunk:
//
//   dU = P^T dO + D k dS,   dX = Tb^T dU = dV,   dS <- G_C dS + q^T G dO - k^T G dX
//   dP = dO U^T (j <= i),   N = -dX U^T (j < i)
//   dq = G dO S^T + (dP E) k
//   W  = (dP E)^T q + D U dS^T + (N E)^T k,   R = -G dX S^T + (N E) k,   dk = W + R
//   db_i = (dX_i . U_i) / b_i^2
//   dc_i = q_i.dq_i + k_i.(R_i - W_i),   dc_C += <S after the chunk, dS>;   dlog_decay_i = sum_{l >= i} dc_l
//
// Four launches: what each chunk needs of its own keys (Tb, P and the decays), the states from chunk to chunk with the
// outputs, the same against time for the states' gradients, and the gradients chunk by chunk.  A b of zero counts as
// 2^-60, so that db has its quotient.
#include "dc_common.h"
#include "layer_launch.h"

namespace dc {
namespace {

constexpr int C = 64;
// floats of a token that the chunks keep: c (two parts), G, D, b, 1/|k|, 1/|q|
constexpr int kVecs = 7;
constexpr float kTiny = 0x1p-60f;

struct Ws {
  float *vec, *tb, *p;       // of the forward
  float *u, *s, *ds;         // of the backward: U and dX, states before each chunk and their gradients after it
  int64_t n;                 // chunks of a head
};

int64_t fwd_floats(const DrProblem& p) {
  const int64_t n = (p.T + C - 1) / C;
  return p.B * p.H * n * (kVecs * C + 2 * C * C);
}

Ws ws_of(const DrProblem& p, bool bwd) {
  Ws w{};
  w.n = (p.T + C - 1) / C;
  const int64_t heads = p.B * p.H * w.n;
  float* f = static_cast<float*>(bwd && p.fwd_ws ? const_cast<void*>(p.fwd_ws) : p.ws);
  w.vec = f;
  w.tb = w.vec + heads * kVecs * C;
  w.p = w.tb + heads * C * C;
  if (bwd) {
    w.u = static_cast<float*>(p.ws) + (p.fwd_ws ? 0 : fwd_floats(p));
    w.s = w.u + heads * 2 * C * p.V;
    w.ds = w.s + heads * p.K * p.V;
  }
  return w;
}

struct Args {
  DrProblem p;
  Ws w;
  int64_t blk0;
};

__device__ __forceinline__ int length_of(const DrProblem& p, int64_t b) {
  const int T = (int)p.T;
  return p.lengths ? min(max(p.lengths[b], 0), T) : T;
}
__device__ __forceinline__ float gate_at(const void* t, int gdtype, int64_t i) {
  return gdtype == kBF16 ? (float)((const bf16*)t)[i] : gdtype == kFP16 ? (float)((const fp16*)t)[i] : ((const float*)t)[i];
}
__device__ __forceinline__ void put_gate(void* t, int gdtype, int64_t i, float v) {
  if (gdtype == kBF16) ((bf16*)t)[i] = (bf16)v;
  else if (gdtype == kFP16) ((fp16*)t)[i] = (fp16)v;
  else ((float*)t)[i] = v;
}

template <typename T>
__global__ __launch_bounds__(256) void dr_prep(Args a) {
  const DrProblem& p = a.p;
  __shared__ float A[C][C + 1], X[C][C + 1], rk[C], rq[C], bb[C];
  __shared__ double c[C];
  const int64_t blk = a.blk0 + blockIdx.x, n = blk % a.w.n, bh = blk / a.w.n, b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
  const int t0 = (int)n * C, len = length_of(p, b), t = threadIdx.x;
  if (t0 >= len) return;
  const T* q = (const T*)p.q + b * p.qs[0] + hk * p.qs[1];
  const T* k = (const T*)p.k + b * p.ks[0] + hk * p.ks[1];
  const int cnt = min(C, len - t0), K = (int)p.K;
  if (t < C) {
    const bool live = t < cnt;
    const float g = live ? gate_at(p.g, p.gdtype, b * p.gs[0] + h * p.gs[1] + (t0 + t) * p.gs[2]) : 0.f;
    c[t] = g < -128.f ? -128.f : g;
    const float be = live ? gate_at(p.b, p.gdtype, b * p.bs[0] + h * p.bs[1] + (t0 + t) * p.bs[2]) : 0.f;
    bb[t] = fabsf(be) < kTiny ? kTiny : be;
    float nk = 0.f, nq = 0.f;
    if (live && p.normalize)
      for (int i = 0; i < K; ++i) {
        const float x = (float)k[(t0 + t) * p.ks[2] + i], y = (float)q[(t0 + t) * p.qs[2] + i];
        nk += x * x;
        nq += y * y;
      }
    rk[t] = p.normalize ? 1.f / sqrtf(nk + p.eps) : 1.f;
    rq[t] = p.normalize ? 1.f / sqrtf(nq + p.eps) : 1.f;
  }
  __syncthreads();
  if (t == 0)
    for (int i = 1; i < C; ++i) c[i] += c[i - 1];
  __syncthreads();
  float* vec = a.w.vec + blk * kVecs * C;
  if (t < C) {
    const float hi = (float)c[t];
    vec[t] = hi;
    vec[C + t] = (float)(c[t] - hi);
    vec[2 * C + t] = expf((float)c[t]);
    vec[3 * C + t] = expf((float)(c[C - 1] - c[t]));
    vec[4 * C + t] = bb[t];
    vec[5 * C + t] = rk[t];
    vec[6 * C + t] = rq[t];
  }
  for (int e = t; e < C * C; e += 256) {
    const int i = e / C, j = e % C;
    float kk = 0.f, qk = 0.f;
    if (j <= i && i < cnt)
      for (int d = 0; d < K; ++d) {
        const float x = (float)k[(t0 + j) * p.ks[2] + d];
        kk += (float)k[(t0 + i) * p.ks[2] + d] * x;
        qk += (float)q[(t0 + i) * p.qs[2] + d] * x;
      }
    const float E = j <= i ? expf((float)(c[i] - c[j])) : 0.f;
    A[i][j] = j < i ? bb[i] * E * kk * rk[i] * rk[j] : 0.f;
    a.w.p[blk * C * C + e] = j <= i ? p.scale * E * qk * rq[i] * rk[j] : 0.f;
  }
  __syncthreads();
  if (t < C) {
    for (int i = 0; i < C; ++i) {
      float s = i == t ? 1.f : 0.f;
      for (int l = t; l < i; ++l) s -= A[i][l] * X[l][t];
      X[i][t] = s;
    }
    for (int i = 0; i < C; ++i) a.w.tb[blk * C * C + i * C + t] = X[i][t] * bb[t];
  }
}

// The states from chunk to chunk.  KEEP: U and the state before each chunk for the backward, instead of o.
template <typename T, bool KEEP>
__global__ __launch_bounds__(256) void dr_chain(Args a) {
  const DrProblem& p = a.p;
  __shared__ float S[256][17], X[C][17], U[C][17];
  const int nvb = (int)(p.V + 15) / 16;
  const int64_t blk = a.blk0 + blockIdx.x, bh = blk / nvb, b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
  const int col = threadIdx.x % 16, row = threadIdx.x / 16, nn = (int)(blk % nvb) * 16 + col, K = (int)p.K;
  const bool live = nn < p.V;
  const int len = length_of(p, b);
  const T* q = (const T*)p.q + b * p.qs[0] + hk * p.qs[1];
  const T* k = (const T*)p.k + b * p.ks[0] + hk * p.ks[1];
  const T* v = (const T*)p.v + b * p.vs[0] + h * p.vs[1] + nn;
  T* o = (T*)p.o + b * p.os[0] + h * p.os[1] + nn;
  const int64_t sb = bh * p.K * p.V + nn;
  for (int i = row; i < K; i += 16) S[i][col] = live && p.s_in ? p.s_in[sb + i * p.V] : 0.f;
  __syncthreads();
  for (int t0 = 0; t0 < len; t0 += C) {
    const int cnt = min(C, len - t0);
    const int64_t ch = bh * a.w.n + t0 / C;
    const float* vec = a.w.vec + ch * kVecs * C;
    const float *tb = a.w.tb + ch * C * C, *P = a.w.p + ch * C * C;
    if (KEEP && live)
      for (int i = row; i < K; i += 16) a.w.s[ch * p.K * p.V + i * p.V + nn] = S[i][col];
    for (int i = row; i < C; i += 16) {
      float s = 0.f;
      if (i < cnt && live) {
        for (int d = 0; d < K; ++d) s += (float)k[(t0 + i) * p.ks[2] + d] * S[d][col];
        s = (float)v[(t0 + i) * p.vs[2]] - vec[2 * C + i] * vec[5 * C + i] * s;
      }
      X[i][col] = s;
    }
    __syncthreads();
    for (int i = row; i < C; i += 16) {
      float s = 0.f;
      for (int j = 0; j <= i; ++j) s += tb[i * C + j] * X[j][col];
      U[i][col] = s;
      if (KEEP && live) a.w.u[ch * 2 * C * p.V + i * p.V + nn] = s;
    }
    __syncthreads();
    if (!KEEP)
      for (int i = row; i < cnt; i += 16) {
        float s = 0.f, w = 0.f;
        for (int d = 0; d < K; ++d) s += (float)q[(t0 + i) * p.qs[2] + d] * S[d][col];
        for (int j = 0; j <= i; ++j) w += P[i * C + j] * U[j][col];
        if (live) o[(t0 + i) * p.os[2]] = (T)(p.scale * vec[2 * C + i] * vec[6 * C + i] * s + w);
      }
    __syncthreads();
    for (int d = row; d < K; d += 16) {
      float s = vec[2 * C + C - 1] * S[d][col];
      for (int j = 0; j < cnt; ++j) s += (float)k[(t0 + j) * p.ks[2] + d] * vec[5 * C + j] * vec[3 * C + j] * U[j][col];
      S[d][col] = s;
    }
    __syncthreads();
  }
  if (!live || KEEP) return;
  if (p.s_out)
    for (int i = row; i < K; i += 16) p.s_out[sb + i * p.V] = S[i][col];
  for (int64_t t = len + row; t < p.T; t += 16) o[t * p.os[2]] = (T)0.f;
}

// The states' gradients from the last chunk on, and dv.
template <typename T>
__global__ __launch_bounds__(256) void dr_chain_bwd(Args a) {
  const DrProblem& p = a.p;
  __shared__ float S[256][17], X[C][17], U[C][17];
  const int nvb = (int)(p.V + 15) / 16;
  const int64_t blk = a.blk0 + blockIdx.x, bh = blk / nvb, b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
  const int col = threadIdx.x % 16, row = threadIdx.x / 16, nn = (int)(blk % nvb) * 16 + col, K = (int)p.K;
  const bool live = nn < p.V;
  const int len = length_of(p, b);
  const T* q = (const T*)p.q + b * p.qs[0] + hk * p.qs[1];
  const T* k = (const T*)p.k + b * p.ks[0] + hk * p.ks[1];
  const T* d_o = (const T*)p.d_o + b * p.dos[0] + h * p.dos[1] + nn;
  T* dv = (T*)p.dv + b * p.dvs[0] + h * p.dvs[1] + nn;
  const int64_t sb = bh * p.K * p.V + nn;
  for (int i = row; i < K; i += 16) S[i][col] = live && p.ds_in ? p.ds_in[sb + i * p.V] : 0.f;
  __syncthreads();
  for (int t0 = (len + C - 1) / C * C - C; t0 >= 0; t0 -= C) {
    const int cnt = min(C, len - t0);
    const int64_t ch = bh * a.w.n + t0 / C;
    const float* vec = a.w.vec + ch * kVecs * C;
    const float *tb = a.w.tb + ch * C * C, *P = a.w.p + ch * C * C;
    if (live)
      for (int i = row; i < K; i += 16) a.w.ds[ch * p.K * p.V + i * p.V + nn] = S[i][col];
    for (int j = row; j < C; j += 16) {
      float s = 0.f, w = 0.f;
      if (j < cnt && live) {
        for (int d = 0; d < K; ++d) s += (float)k[(t0 + j) * p.ks[2] + d] * S[d][col];
        for (int i = j; i < cnt; ++i) w += P[i * C + j] * (float)d_o[(t0 + i) * p.dos[2]];
      }
      U[j][col] = vec[3 * C + j] * vec[5 * C + j] * s + w;
    }
    __syncthreads();
    for (int j = row; j < C; j += 16) {
      float s = 0.f;
      for (int i = j; i < C; ++i) s += tb[i * C + j] * U[i][col];
      X[j][col] = s;
      if (live && j < cnt) dv[(t0 + j) * p.dvs[2]] = (T)s;
    }
    __syncthreads();
    if (live)
      for (int j = row; j < C; j += 16) a.w.u[ch * 2 * C * p.V + (C + j) * p.V + nn] = X[j][col];
    for (int d = row; d < K; d += 16) {
      float s = vec[2 * C + C - 1] * S[d][col];
      if (live)
        for (int i = 0; i < cnt; ++i)
          s += vec[2 * C + i] * ((float)q[(t0 + i) * p.qs[2] + d] * vec[6 * C + i] * p.scale * (float)d_o[(t0 + i) * p.dos[2]] -
                                 (float)k[(t0 + i) * p.ks[2] + d] * vec[5 * C + i] * X[i][col]);
      S[d][col] = s;
    }
    __syncthreads();
  }
  if (!live) return;
  if (p.ds_out)
    for (int i = row; i < K; i += 16) p.ds_out[sb + i * p.V] = S[i][col];
  for (int64_t t = len + row; t < p.T; t += 16) dv[t * p.dvs[2]] = (T)0.f;
}

// Gradients of q, k and the gates, chunk by chunk: the value heads of one key head to a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void dr_grads(Args a) {
  const DrProblem& p = a.p;
  __shared__ float PE[C][C + 1], NE[C][C + 1], dc[C][4], diag[C], red[256];
  const int64_t blk = a.blk0 + blockIdx.x, n = blk % a.w.n, bhk = blk / a.w.n, b = bhk / p.Hk, hk = bhk % p.Hk;
  const int t0 = (int)n * C, len = length_of(p, b), cnt = min(C, max(len - t0, 0)), t = threadIdx.x, i = t / 4, part = t % 4;
  const int K = (int)p.K, V = (int)p.V, group = (int)(p.H / p.Hk);
  const int64_t ti = t0 + i;
  const T* q = (const T*)p.q + b * p.qs[0] + hk * p.qs[1];
  const T* k = (const T*)p.k + b * p.ks[0] + hk * p.ks[1];
  float dq[64], dk[64];
#pragma unroll
  for (int m = 0; m < 64; ++m) dq[m] = dk[m] = 0.f;
  const float* vec = nullptr;
  for (int g = 0; g < group; ++g) {
    const int64_t h = hk * group + g, bh = b * p.H + h, ch = bh * a.w.n + n;
    vec = a.w.vec + ch * kVecs * C;
    const float *U = a.w.u + ch * 2 * C * V, *X = U + C * V, *S = a.w.s + ch * K * V, *dS = a.w.ds + ch * K * V;
    const T* d_o = (const T*)p.d_o + b * p.dos[0] + h * p.dos[1];
    __syncthreads();
    for (int e = t; e < C * C; e += 256) {
      const int r = e / C, j = e % C;
      float dp = 0.f, nn = 0.f;
      if (j <= r && r < cnt)
        for (int m = 0; m < V; ++m) {
          dp += (float)d_o[(t0 + r) * p.dos[2] + m] * U[j * V + m];
          nn -= X[r * V + m] * U[j * V + m];
        }
      const float E = j <= r && r < cnt ? expf((vec[r] - vec[j]) + (vec[C + r] - vec[C + j])) : 0.f;
      PE[r][j] = dp * E;
      NE[r][j] = j < r ? nn * E : 0.f;
      if (j == r) diag[r] = -nn;
    }
    __syncthreads();
    float kept = 0.f, sum = 0.f;
    if (i < cnt) {
      const float G = vec[2 * C + i], D = vec[3 * C + i], rki = vec[5 * C + i], rqi = vec[6 * C + i] * p.scale;
#pragma unroll
      for (int m = 0; m < 64; ++m) {
        const int d = part + 4 * m;
        if (d < K) {
          float doS = 0.f, xS = 0.f, uS = 0.f;
          for (int x = 0; x < V; ++x) {
            const float s = S[d * V + x];
            doS += (float)d_o[ti * p.dos[2] + x] * s;
            xS += X[i * V + x] * s;
            uS += U[i * V + x] * dS[d * V + x];
          }
          float a1 = G * doS, R = -G * xS, W = D * uS;
          for (int j = 0; j < cnt; ++j) {
            const float kj = (float)k[(t0 + j) * p.ks[2] + d] * vec[5 * C + j];
            const float qj = (float)q[(t0 + j) * p.qs[2] + d] * vec[6 * C + j] * p.scale;
            if (j <= i) {
              a1 += PE[i][j] * kj;
              R += NE[i][j] * kj;
            }
            if (j >= i) W += PE[j][i] * qj + NE[j][i] * kj;
          }
          const float ki = (float)k[ti * p.ks[2] + d] * rki, qi = (float)q[ti * p.qs[2] + d] * rqi;
          sum += qi * a1 + ki * (R - W);
          kept += D * ki * uS;
          dq[m] += a1;
          dk[m] += R + W;
        }
      }
    }
    float ss = 0.f;
    if (cnt > 0)
      for (int e = t; e < K * V; e += 256) ss += S[e] * dS[e];
    dc[i][part] = sum;
    red[t] = cnt > 0 ? kept + vec[2 * C + C - 1] * ss : 0.f;
    __syncthreads();
    if (t < C && t0 + t < p.T) {
      float s = 0.f;
      for (int m = 0; m < 256; ++m) s += red[m];
      for (int m = cnt - 1; m >= t; --m) s += (dc[m][0] + dc[m][1]) + (dc[m][2] + dc[m][3]);
      put_gate(p.dg, p.gdtype, b * p.dgs[0] + h * p.dgs[1] + (t0 + t) * p.dgs[2], t < cnt ? s : 0.f);
      const float be = cnt > 0 ? vec[4 * C + t] : 1.f;
      put_gate(p.db, p.gdtype, b * p.dbs[0] + h * p.dbs[1] + (t0 + t) * p.dbs[2], t < cnt ? diag[t] / be / be : 0.f);
    }
  }
  float nk = 0.f, nq = 0.f;
  const float rki = cnt > 0 ? vec[5 * C + i] : 0.f, rqi = cnt > 0 ? vec[6 * C + i] : 0.f;
  if (i < cnt && p.normalize)
#pragma unroll
    for (int m = 0; m < 64; ++m)
      if (part + 4 * m < K) {
        nk += dk[m] * (float)k[ti * p.ks[2] + part + 4 * m] * rki;
        nq += dq[m] * (float)q[ti * p.qs[2] + part + 4 * m] * rqi;
      }
  nk += __shfl_xor(nk, 1); nk += __shfl_xor(nk, 2);
  nq += __shfl_xor(nq, 1); nq += __shfl_xor(nq, 2);
  if (ti >= p.T) return;
  T* oq = (T*)p.dq + b * p.dqs[0] + hk * p.dqs[1] + ti * p.dqs[2];
  T* ok = (T*)p.dk + b * p.dks[0] + hk * p.dks[1] + ti * p.dks[2];
#pragma unroll
  for (int m = 0; m < 64; ++m) {
    const int d = part + 4 * m;
    if (d >= K) break;
    const float ki = i < cnt ? (float)k[ti * p.ks[2] + d] * rki : 0.f, qi = i < cnt ? (float)q[ti * p.qs[2] + d] * rqi : 0.f;
    ok[d] = (T)(i < cnt ? rki * (dk[m] - ki * nk) : 0.f);
    oq[d] = (T)(i < cnt ? p.scale * rqi * (dq[m] - qi * nq) : 0.f);
  }
}

// Workgroups in as many launches as it takes.
template <typename F>
hipError_t launch(F kernel, Args a, int64_t blocks) {
  constexpr int64_t most = most_workgroups(256);
  for (a.blk0 = 0; a.blk0 < blocks; a.blk0 += most) {
    kernel<<<(unsigned)(blocks - a.blk0 < most ? blocks - a.blk0 : most), 256, 0, a.p.stream>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T>
hipError_t fwd(const DrProblem& p) {
  Args a{p, ws_of(p, false), 0};
  const int64_t heads = p.B * p.H;
  const hipError_t e = launch(dr_prep<T>, a, heads * a.w.n);
  return e != hipSuccess ? e : launch(dr_chain<T, false>, a, heads * ((p.V + 15) / 16));
}

template <typename T>
hipError_t bwd(const DrProblem& p) {
  Args a{p, ws_of(p, true), 0};
  const int64_t heads = p.B * p.H, cols = heads * ((p.V + 15) / 16);
  hipError_t e = p.fwd_ws ? hipSuccess : launch(dr_prep<T>, a, heads * a.w.n);
  if (e == hipSuccess) e = launch(dr_chain<T, true>, a, cols);
  if (e == hipSuccess) e = launch(dr_chain_bwd<T>, a, cols);
  return e != hipSuccess ? e : launch(dr_grads<T>, a, p.B * p.Hk * a.w.n);
}

}  // namespace

int64_t dr_ws_bytes(const DrProblem& p, int bwd) {
  const int64_t n = p.B * p.H * ((p.T + C - 1) / C);
  return 4 * ((bwd == 2 ? 0 : fwd_floats(p)) + (bwd ? n * (2 * C * p.V + 2 * p.K * p.V) : 0));
}

hipError_t dr_fwd(const DrProblem& p) {
  return p.dtype == kBF16 ? fwd<bf16>(p) : p.dtype == kFP16 ? fwd<fp16>(p) : fwd<float>(p);
}
hipError_t dr_bwd(const DrProblem& p) {
  return p.dtype == kBF16 ? bwd<bf16>(p) : p.dtype == kFP16 ? bwd<fp16>(p) : bwd<float>(p);
}

}  // namespace dc
