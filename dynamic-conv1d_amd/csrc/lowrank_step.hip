// The lowrank convolution of one token of each of N sequences, for G groups
// (dc_lowrank_step_grouped):
//
//   y[n, d] = sum_w (sum_r z[n, r] U[r, w*D + d] + static_w[w, d]) x_w[n, d]  (+ x_0)
//
// with x_0 the new input and x_w, w >= 1, row W-1-w of the sequence's state; the
// state then drops row 0 and takes x_0 behind the others.
//
// A workgroup takes kN sequences and 64 * VEC channels of one group; its four
// wavefronts take the taps in turn (wavefront i: taps i, i + 4, ..), so the four
// chains of U loads run side by side, and add their sums of y in LDS in a fixed
// order.  z is staged in LDS as float, U is read once for the kN sequences.
#include "dc_common.h"
#include "layer_launch.h"

namespace dc {
namespace {

constexpr int kN = 8;      // sequences of a workgroup
constexpr int kWaves = 4;  // wavefronts, which share the taps

template <typename T, int VEC>
__global__ __launch_bounds__(64 * kWaves) void lr_step_kernel(LrStep p) {
  extern __shared__ float sz[];  // [kN][R], then the sums of y [kWaves][kN][64 * VEC]
  const int R = (int)p.R, W = (int)p.W;
  const int64_t D = p.D, C = p.G * D;
  float* sy = sz + kN * R;
  const int g = blockIdx.z;
  const int64_t n0 = (int64_t)blockIdx.y * kN;
  const int nn = (int)min((int64_t)kN, p.N - n0);
  const int wv = wave_id(), lane = threadIdx.x % 64;
  const int64_t d = ((int64_t)blockIdx.x * 64 + lane) * VEC;
  const bool live = d < D;
  const T* z = (const T*)p.z[g];
  const T* U = (const T*)p.U[g] + d;
  const T* sw = p.static_w[g] ? (const T*)p.static_w[g] + d : nullptr;
  const T* x = (const T*)p.x + n0 * p.x_ld + g * D + d;
  T* st = (T*)p.state + g * D + d;

  for (int i = threadIdx.x; i < kN * R; i += 64 * kWaves) {
    const int n = i / R, r = i % R;
    sz[i] = n < nn ? (float)z[(n0 + n) * R + r] : 0.f;
  }
  __syncthreads();

  int64_t slot[kN];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const int64_t s = n >= nn ? -1 : p.slot_ids ? (int64_t)p.slot_ids[n0 + n] : n0 + n;
    slot[n] = s < p.slots ? s : -1;
  }
  float y[kN][VEC];
#pragma unroll
  for (int n = 0; n < kN; ++n) zero_vals<VEC>(y[n]);
  for (int w = wv; w < W; w += kWaves) {
    float k[kN][VEC];
#pragma unroll
    for (int n = 0; n < kN; ++n) zero_vals<VEC>(k[n]);
    if (live) {
      if (sw) {
        float s[VEC];
        load_vals<T, VEC>(sw + w * D, s);
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < VEC; ++j) k[n][j] = s[j];
      }
#pragma unroll 8
      for (int r = 0; r < R; ++r) {
        float u[VEC];
        load_vals<T, VEC>(U + (int64_t)r * W * D + w * D, u);
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < VEC; ++j) k[n][j] += sz[n * R + r] * u[j];
      }
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        if (slot[n] < 0) continue;
        float xv[VEC];
        load_vals<T, VEC>(w == 0 ? x + n * p.x_ld : st + (slot[n] * (W - 1) + W - 1 - w) * C, xv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[n][j] += (k[n][j] + (w == 0 && p.residual ? 1.f : 0.f)) * xv[j];
      }
    }
  }
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int j = 0; j < VEC; ++j) sy[((wv * kN + n) * VEC + j) * 64 + lane] = y[n][j];
  __syncthreads();  // every tap has been read: the state may move
  if (!live) return;
  T* out = (T*)p.y[g] + n0 * D + d;
  for (int n = wv; n < nn; n += kWaves) {
    float t[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float* s = sy + (n * VEC + j) * 64 + lane;
      constexpr int step = kN * VEC * 64;
      t[j] = (s[0] + s[step]) + (s[2 * step] + s[3 * step]);
    }
    store_vals<T, VEC>(out + n * D, t);
    const int64_t s = p.slot_ids ? (int64_t)p.slot_ids[n0 + n] : n0 + n;
    if (s < 0 || s >= p.slots) continue;
    T* row = st + s * (W - 1) * C;
    Raw<T, VEC> v;
    for (int w = 0; w < W - 1; ++w) {
      v.load(w == W - 2 ? x + n * p.x_ld : row + (w + 1) * C);
#pragma unroll
      for (int i = 0; i < Raw<T, VEC>::NU; ++i) reinterpret_cast<typename Raw<T, VEC>::U*>(row + w * C)[i] = v.u[i];
    }
  }
}

template <typename T, int VEC>
hipError_t launch(const LrStep& p) {
  const int64_t nx = (p.D + 64 * VEC - 1) / (64 * VEC);
  const int64_t lds = 4 * (kN * p.R + kWaves * kN * VEC * 64);
  const int64_t ny = (p.N + kN - 1) / kN;
  // the grid's second axis holds 65535 blocks: larger batches go in parts
  for (int64_t y0 = 0; y0 < ny; y0 += 65535) {
    LrStep q = p;
    const int64_t n0 = y0 * kN, part = ny - y0 < 65535 ? ny - y0 : 65535;
    q.N = p.N - n0 < part * kN ? p.N - n0 : part * kN;
    q.x = (const T*)p.x + n0 * p.x_ld;
    if (p.slot_ids) q.slot_ids = p.slot_ids + n0;
    else if (p.state) q.state = (T*)p.state + n0 * (p.W - 1) * p.G * p.D;
    for (int64_t g = 0; g < p.G; ++g) {
      q.z[g] = (const T*)p.z[g] + n0 * p.R;
      q.y[g] = (T*)p.y[g] + n0 * p.D;
    }
    lr_step_kernel<T, VEC><<<dim3((unsigned)nx, (unsigned)part, (unsigned)p.G), 64 * kWaves, lds, p.stream>>>(q);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launch_vec(const LrStep& p) {
  // two channels to a lane where every row starts on a pair
  bool v2 = p.D % 2 == 0 && p.x_ld % 2 == 0;
  const uintptr_t a = 2 * sizeof(T);
  for (const void* t : {p.x, (const void*)p.state}) v2 = v2 && reinterpret_cast<uintptr_t>(t) % a == 0;
  for (int64_t g = 0; g < p.G; ++g)
    for (const void* t : {p.U[g], p.static_w[g], (const void*)p.y[g]})
      v2 = v2 && reinterpret_cast<uintptr_t>(t) % a == 0;
  return v2 ? launch<T, 2>(p) : launch<T, 1>(p);
}

}  // namespace

hipError_t lr_step(const LrStep& p) {
  switch (p.dtype) {
    case kBF16: return launch_vec<bf16>(p);
    case kFP16: return launch_vec<fp16>(p);
    default: return launch_vec<float>(p);
  }
}

}  // namespace dc
