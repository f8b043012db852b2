// The lowrank convolution of one token of each of N sequences, for G groups
// (dc_lowrank_step_grouped):
//
//   y[n, d] = sum_w (sum_r z[n, r] U[r, w*D + d] + static_w[w, d]) x_w[n, d]  (+ x_0)
//
// with x_0 the new input and x_w, w >= 1, row W-1-w of the sequence's state; the
// state then drops row 0 and takes x_0 behind the others.
//
// Matrix cores (lr_step_mma), where rows are whole 16-byte pieces: a workgroup
// takes 32 sequences and 128 channels of one group, a wavefront 32 channels; the
// taps' weights of a tap w are U_w^T z^T (v_mfma_f32_32x32x16: channels by
// sequences, the static filter as one more rank with z = 1), in float32, and meet
// x_w in the registers.  Bound by the state's and x's rows (W read, W - 1 written)
// and U, and at few sequences by the latency of one round of loads: TAPS taps' pieces
// of U and x are in flight at once.  A thread's pieces of the state move on as it
// holds them: taps go from the oldest on, so the row that x_w is written to has
// been read by the same thread.
//
// Measured, q|k|v in one launch, W 4, static filter: 256 sequences, D 4096, rank 31, bf16 13.6 us (53 MB, 3.9 TB/s; 47.7
// with lr_step_any), 8 sequences, D 2048, rank 15 (lr_step_taps) 4.4 us behind one another, one round trip of loads and
// the launch (lr_step_mma 5.1).
//
// Few workgroups of those take lr_step_taps; rows off the 16-byte pieces take lr_step_any, a thread to a channel on the
// vector units, which loads elements and forms every weight for 8 sequences only (256 sequences as above, D 4097: 81 us).
#include "linattn_mfma.h"

namespace dc {
namespace {

constexpr int kN = 8;      // sequences of a workgroup (lr_step_any)
constexpr int kWaves = 4;  // wavefronts, which there share the taps
constexpr int kSeqs = 32, kChans = 128;

template <typename T, int RP, int TAPS>
__global__ __launch_bounds__(256) void lr_step_mma(LrStep p) {
  typedef la::Ops<T> O;
  constexpr int VE = 16 / (int)sizeof(T), PR = kChans / VE, UP = RP * PR / 256, XP = kSeqs * PR / 256;
  constexpr int RU = la::row_elems<T, kChans, false>(), RX = kChans + VE, RZ = RP + VE;
  __shared__ __align__(16) T su[RP * RU];
  __shared__ __align__(16) T sx[kSeqs * RX];
  __shared__ __align__(16) T sz[kSeqs * RZ];
  const int R = (int)p.R, W = (int)p.W, g = blockIdx.z, tid = threadIdx.x;
  const int64_t D = p.D, C = p.G * D, d0 = (int64_t)blockIdx.x * kChans, n0 = (int64_t)blockIdx.y * kSeqs;
  const int lane = tid % 64, half = lane / 32, col = lane % 32, wv = wave_id();
  const T* z = (const T*)p.z[g];
  const T* U = (const T*)p.U[g] + d0;
  const T* sw = p.static_w[g] ? (const T*)p.static_w[g] + d0 : nullptr;

  // this thread's pieces of x and the state: their sequences' rows, if they take part
  const int c = tid % PR * VE;
  const bool in = d0 + c < D;
  const T* xr[XP];
  T* sr[XP];
#pragma unroll
  for (int i = 0; i < XP; ++i) {
    const int64_t n = n0 + tid / PR + i * (256 / PR);
    const int64_t slot = n >= p.N ? -1 : p.slot_ids ? (int64_t)p.slot_ids[n] : n;
    const bool live = in && slot >= 0 && slot < p.slots;
    xr[i] = live ? (const T*)p.x + n * p.x_ld + g * D + d0 + c : nullptr;
    sr[i] = (T*)p.state + slot * (W - 1) * C + g * D + d0 + c;
  }
  for (int i = tid; i < kSeqs * RP; i += 256) {
    const int n = i / RP, r = i % RP;
    const int64_t slot = n0 + n >= p.N ? -1 : p.slot_ids ? (int64_t)p.slot_ids[n0 + n] : n0 + n;
    const bool live = slot >= 0 && slot < p.slots;  // whatever the others' z holds, their y is zero
    sz[n * RZ + r] = !live ? (T)0.f : r < R ? z[(n0 + n) * R + r] : r == R && sw ? (T)1.f : (T)0.f;
  }

  float y[16];
  zero_vals<16>(y);
  for (int w1 = W; w1 > 0; w1 -= TAPS) {  // taps w1 - 1 .. w1 - TAPS, the oldest first
    u32x4 u[TAPS][UP], x[TAPS][XP];
#pragma unroll
    for (int k = 0; k < TAPS; ++k) {
      const int w = w1 - 1 - k;
#pragma unroll
      for (int i = 0; i < XP; ++i) {
        x[k][i] = u32x4{0, 0, 0, 0};
        if (w >= 0 && xr[i]) x[k][i] = *reinterpret_cast<const u32x4*>(w == 0 ? xr[i] : sr[i] + (W - 1 - w) * C);
      }
#pragma unroll
      for (int i = 0; i < UP; ++i) {
        const int r = tid / PR + i * (256 / PR);
        u[k][i] = u32x4{0, 0, 0, 0};
        if (w >= 0 && in && r < R) u[k][i] = *reinterpret_cast<const u32x4*>(U + ((int64_t)r * W + w) * D + c);
        else if (w >= 0 && in && r == R && sw) u[k][i] = *reinterpret_cast<const u32x4*>(sw + w * D + c);
      }
    }
#pragma unroll
    for (int k = 0; k < TAPS; ++k) {
      const int w = w1 - 1 - k;
      if (w < 0) break;
      __syncthreads();  // the tap before has been read
#pragma unroll
      for (int i = 0; i < XP; ++i) {
        *reinterpret_cast<u32x4*>(sx + (tid / PR + i * (256 / PR)) * RX + c) = x[k][i];
        if (xr[i] && w < W - 1) *reinterpret_cast<u32x4*>(sr[i] + (W - 2 - w) * C) = x[k][i];
      }
#pragma unroll
      for (int i = 0; i < UP; ++i) *reinterpret_cast<u32x4*>(su + (tid / PR + i * (256 / PR)) * RU + c) = u[k][i];
      __syncthreads();
      la::f32x16 acc = {};
#pragma unroll
      for (int s = 0; s < RP / 16; ++s) {
        // both in the order of columns read (row 4 half + e%4 + 8 (e/4) of the step's 16)
        const T* zr = sz + col * RZ + s * 16 + 4 * half;
        float t[8];
        load_vals<T, 4>(zr, t);
        load_vals<T, 4>(zr + 8, t + 4);
        acc = O::mma(O::template cols<false>(su + s * 16 * RU + wv * 32, RU, lane), O::pack(t), acc);
      }
      const float one = w == 0 && p.residual ? 1.f : 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float xv[4];
        load_vals<T, 4>(sx + col * RX + wv * 32 + 8 * q + 4 * half, xv);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[4 * q + j] += (acc[4 * q + j] + one) * xv[j];
      }
    }
  }
  // y through LDS, so that its rows go out in 16-byte pieces
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; ++q) store_vals<T, 4>(sx + col * RX + wv * 32 + 8 * q + 4 * half, y + 4 * q);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < XP; ++i) {
    const int n = tid / PR + i * (256 / PR);
    // zeros where a sequence takes no part: of its zeros, infinities and NaN in the filters make NaN
    if (in && n0 + n < p.N)
      *reinterpret_cast<u32x4*>((T*)p.y[g] + (n0 + n) * D + d0 + c) =
          xr[i] ? *reinterpret_cast<const u32x4*>(sx + n * RX + c) : u32x4{0, 0, 0, 0};
  }
}

// lr_step_mma for few workgroups: 32 channels to one, and the taps go round its wavefronts, so four times the workgroups
// and a quarter of the chain.  A thread has TAPS taps of U and x in flight; four of them at a time lie in LDS.  The
// wavefronts' sums of y meet in a fixed order.
template <typename T, int RP, int TAPS>
__global__ __launch_bounds__(256) void lr_step_taps(LrStep p) {
  typedef la::Ops<T> O;
  constexpr int CH = 32, VE = 16 / (int)sizeof(T), PR = CH / VE, ROWS = 256 / PR, UP = RP > ROWS ? RP / ROWS : 1;
  constexpr int RU = la::row_elems<T, CH, false>(), RX = CH + VE, RZ = RP + VE, RY = CH + 1;
  constexpr int UB = kWaves * RP * RU * (int)sizeof(T), YB = kWaves * kSeqs * RY * (int)sizeof(float);
  __shared__ __align__(16) unsigned char buf[UB > YB ? UB : YB];  // U's taps, then the sums of y
  __shared__ __align__(16) T sx[kWaves * kSeqs * RX];
  __shared__ __align__(16) T sz[kSeqs * RZ];
  T* const su = reinterpret_cast<T*>(buf);
  float* const sy = reinterpret_cast<float*>(buf);
  const int R = (int)p.R, W = (int)p.W, g = blockIdx.z, tid = threadIdx.x;
  const int64_t D = p.D, C = p.G * D, d0 = (int64_t)blockIdx.x * CH, n0 = (int64_t)blockIdx.y * kSeqs;
  const int lane = tid % 64, half = lane / 32, col = lane % 32, wv = wave_id();
  const T* z = (const T*)p.z[g];
  const T* U = (const T*)p.U[g] + d0;
  const T* sw = p.static_w[g] ? (const T*)p.static_w[g] + d0 : nullptr;

  const int c = tid % PR * VE, row = tid / PR;
  const bool in = d0 + c < D;
  const int64_t n = n0 + row;
  const int64_t slot = row >= kSeqs || n >= p.N ? -1 : p.slot_ids ? (int64_t)p.slot_ids[n] : n;
  const bool live = in && slot >= 0 && slot < p.slots;
  const T* xr = live ? (const T*)p.x + n * p.x_ld + g * D + d0 + c : nullptr;
  T* sr = (T*)p.state + slot * (W - 1) * C + g * D + d0 + c;

  float y[16];
  zero_vals<16>(y);
  for (int w1 = W; w1 > 0; w1 -= TAPS) {  // taps w1 - 1 .. w1 - TAPS, the oldest first
    u32x4 u[TAPS][UP], x[TAPS];
#pragma unroll
    for (int k = 0; k < TAPS; ++k) {
      const int w = w1 - 1 - k;
      x[k] = u32x4{0, 0, 0, 0};
      if (w >= 0 && xr) x[k] = *reinterpret_cast<const u32x4*>(w == 0 ? xr : sr + (W - 1 - w) * C);
#pragma unroll
      for (int i = 0; i < UP; ++i) {
        const int r = row + i * ROWS;
        u[k][i] = u32x4{0, 0, 0, 0};
        if (w >= 0 && in && r < R) u[k][i] = *reinterpret_cast<const u32x4*>(U + ((int64_t)r * W + w) * D + c);
        else if (w >= 0 && in && r == R && sw) u[k][i] = *reinterpret_cast<const u32x4*>(sw + w * D + c);
      }
    }
    if (w1 == W)  // behind the loads
      for (int i = tid; i < kSeqs * RP; i += 256) {
        const int m = i / RP, r = i % RP;
        const int64_t of = n0 + m >= p.N ? -1 : p.slot_ids ? (int64_t)p.slot_ids[n0 + m] : n0 + m;
        const bool part = of >= 0 && of < p.slots;  // whatever the others' z holds, their y is zero
        sz[m * RZ + r] = !part ? (T)0.f : r < R ? z[(n0 + m) * R + r] : r == R && sw ? (T)1.f : (T)0.f;
      }
#pragma unroll
    for (int k0 = 0; k0 < TAPS; k0 += kWaves) {
      if (w1 - 1 - k0 < 0) break;
      __syncthreads();  // the taps before have been read
#pragma unroll
      for (int k = k0; k < k0 + kWaves; ++k) {
        const int w = w1 - 1 - k;
        if (w < 0) break;
        if (row < kSeqs) *reinterpret_cast<u32x4*>(sx + ((k - k0) * kSeqs + row) * RX + c) = x[k];
        if (xr && w < W - 1) *reinterpret_cast<u32x4*>(sr + (W - 2 - w) * C) = x[k];
#pragma unroll
        for (int i = 0; i < UP; ++i)
          if (row + i * ROWS < RP) *reinterpret_cast<u32x4*>(su + ((k - k0) * RP + row + i * ROWS) * RU + c) = u[k][i];
      }
      __syncthreads();
      const int w = w1 - 1 - k0 - wv;
      if (w < 0) continue;
      la::f32x16 acc = {};
#pragma unroll
      for (int s = 0; s < RP / 16; ++s) {
        const T* zr = sz + col * RZ + s * 16 + 4 * half;
        float t[8];
        load_vals<T, 4>(zr, t);
        load_vals<T, 4>(zr + 8, t + 4);
        acc = O::mma(O::template cols<false>(su + (wv * RP + s * 16) * RU, RU, lane), O::pack(t), acc);
      }
      const float one = w == 0 && p.residual ? 1.f : 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float xv[4];
        load_vals<T, 4>(sx + (wv * kSeqs + col) * RX + 8 * q + 4 * half, xv);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[4 * q + j] += (acc[4 * q + j] + one) * xv[j];
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 16; ++q) sy[(wv * kSeqs + col) * RY + 8 * (q / 4) + 4 * half + q % 4] = y[q];
  __syncthreads();
  if (row < kSeqs && in && n < p.N) {
    float v[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const float* t = sy + row * RY + c + j;
      constexpr int next = kSeqs * RY;
      v[j] = xr ? (t[0] + t[next]) + (t[2 * next] + t[3 * next]) : 0.f;  // as in lr_step_mma
    }
    store_vals<T, VE>((T*)p.y[g] + n * D + d0 + c, v);
  }
}

// A wavefront takes 64 channels, kN sequences and every fourth tap; the wavefronts' sums of y meet in LDS in a fixed order.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void lr_step_any(LrStep p) {
  extern __shared__ float sz[];  // [kN][R], then the sums of y [kWaves][kN][64]
  const int R = (int)p.R, W = (int)p.W;
  const int64_t D = p.D, C = p.G * D;
  float* sy = sz + kN * R;
  const int g = blockIdx.z;
  const int64_t n0 = (int64_t)blockIdx.y * kN;
  const int nn = (int)min((int64_t)kN, p.N - n0);
  const int wv = wave_id(), lane = threadIdx.x % 64;
  const int64_t d = (int64_t)blockIdx.x * 64 + lane;
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
  float y[kN];
  zero_vals<kN>(y);
  for (int w = wv; w < W && live; w += kWaves) {
    float k[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) k[n] = sw ? (float)sw[w * D] : 0.f;
#pragma unroll 8
    for (int r = 0; r < R; ++r) {
      const float u = (float)U[((int64_t)r * W + w) * D];
#pragma unroll
      for (int n = 0; n < kN; ++n) k[n] += sz[n * R + r] * u;
    }
#pragma unroll
    for (int n = 0; n < kN; ++n)
      if (slot[n] >= 0)
        y[n] += (k[n] + (w == 0 && p.residual ? 1.f : 0.f)) *
                (float)(w == 0 ? x[n * p.x_ld] : st[(slot[n] * (W - 1) + W - 1 - w) * C]);
  }
#pragma unroll
  for (int n = 0; n < kN; ++n) sy[(wv * kN + n) * 64 + lane] = y[n];
  __syncthreads();  // every tap has been read: the state may move
  if (!live) return;
  T* out = (T*)p.y[g] + n0 * D + d;
  for (int n = wv; n < nn; n += kWaves) {
    const float* s = sy + n * 64 + lane;
    constexpr int step = kN * 64;
    out[n * D] = (T)((s[0] + s[step]) + (s[2 * step] + s[3 * step]));
    const int64_t sl = p.slot_ids ? (int64_t)p.slot_ids[n0 + n] : n0 + n;
    if (sl < 0 || sl >= p.slots) continue;
    T* row = st + sl * (W - 1) * C;
    for (int w = 0; w < W - 1; ++w) row[w * C] = w == W - 2 ? x[n * p.x_ld] : row[(w + 1) * C];
  }
}

bool whole(const void* t) { return reinterpret_cast<uintptr_t>(t) % 16 == 0; }

// Whether lr_step_mma takes a problem: rows of whole 16-byte pieces throughout.
bool mma_ok(const LrStep& p) {
  const int64_t ve = 16 / dtype_size(p.dtype);
  // float32 above 128 ranks: a tap of U would pass the LDS
  bool ok = p.dtype != kFP32 || p.R + (p.static_w[0] ? 1 : 0) <= 128;
  ok = ok && p.D % ve == 0 && p.x_ld % ve == 0 && whole(p.x) && whole(p.state);
  for (int64_t g = 0; g < p.G; ++g) ok = ok && whole(p.U[g]) && whole(p.static_w[g]) && whole(p.y[g]);
  return ok;
}

// Whether lr_step_taps takes a problem: its workgroups, four for each of lr_step_mma's, then have a CU each in 16 bits
// (float32's, of half the channels to a piece, gain to three rounds).  Measured, lr_step_taps against lr_step_mma, us, 32
// sequences, W 4 rank 16 / W 8 rank 32 / W 16 rank 64, bf16: D 2048 4.3 / 6.6 / 11.3 against 5.3 / 8.7 / 19.6, D 8192 (64
// workgroups) 5.0 / 7.9 / 18.6 against 5.6 / 9.2 / 20.3, D 12288 5.6 / 9.3 / 21.9 against 5.7 / 9.6 / 30.2 but W 16 rank 32
// 17.9 against 15.3, D 16384 6.0 against 5.9; float32, 64 sequences, D 12288 (192) 7.3 / 15.3 / 52 against 9.0 / 21.5 / 65,
// D 32768 19.2 against 16.3.
bool few(const LrStep& p) {
  return (p.D + kChans - 1) / kChans * ((p.N + kSeqs - 1) / kSeqs) * p.G <= (p.dtype == kFP32 ? 192 : 64);
}

// Sequences in parts of what the grid's second axis holds.
template <typename T, typename F>
hipError_t in_parts(const LrStep& p, int per, F launch) {
  for (int64_t n0 = 0; n0 < p.N; n0 += (int64_t)per * 65535) {
    LrStep q = p;
    q.N = p.N - n0 < (int64_t)per * 65535 ? p.N - n0 : (int64_t)per * 65535;
    q.x = (const T*)p.x + n0 * p.x_ld;
    if (p.slot_ids) q.slot_ids = p.slot_ids + n0;
    else if (p.state) q.state = (T*)p.state + n0 * (p.W - 1) * p.G * p.D;
    for (int64_t g = 0; g < p.G; ++g) {
      q.z[g] = (const T*)p.z[g] + n0 * p.R;
      q.y[g] = (T*)p.y[g] + n0 * p.D;
    }
    launch(q, (unsigned)((q.N + per - 1) / per));
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launch(const LrStep& p) {
  const unsigned G = (unsigned)p.G;
  if (!mma_ok(p))
    return in_parts<T>(p, kN, [&](const LrStep& q, unsigned ny) {
      const size_t lds = 4 * (kN * p.R + kWaves * kN * 64);
      lr_step_any<T><<<dim3((unsigned)((p.D + 63) / 64), ny, G), 64 * kWaves, lds, p.stream>>>(q);
    });
  const int64_t rank = p.R + (p.static_w[0] ? 1 : 0);
  if (few(p))
    return in_parts<T>(p, kSeqs, [&](const LrStep& q, unsigned ny) {
      const dim3 grid((unsigned)((p.D + 31) / 32), ny, G);
      // taps in flight: eight, or as many as there are or registers hold
      const bool four = p.W <= 4;
      auto run = [&](auto kernel) { kernel<<<grid, 256, 0, p.stream>>>(q); };
      if (rank <= 16) run(four ? lr_step_taps<T, 16, 4> : lr_step_taps<T, 16, 8>);
      else if (rank <= 32) run(four ? lr_step_taps<T, 32, 4> : lr_step_taps<T, 32, 8>);
      else if (rank <= 64) run(four ? lr_step_taps<T, 64, 4> : lr_step_taps<T, 64, 8>);
      else if (rank <= 128) run(lr_step_taps<T, 128, 4>);
      else if constexpr (sizeof(T) == 2) run(lr_step_taps<T, 256, 4>);
    });
  return in_parts<T>(p, kSeqs, [&](const LrStep& q, unsigned ny) {
    const dim3 grid((unsigned)((p.D + kChans - 1) / kChans), ny, G);
    // taps in flight: what 64 registers hold of U
    if (rank <= 16) lr_step_mma<T, 16, 4><<<grid, 256, 0, p.stream>>>(q);
    else if (rank <= 32) lr_step_mma<T, 32, 4><<<grid, 256, 0, p.stream>>>(q);
    else if (rank <= 64) lr_step_mma<T, 64, sizeof(T) == 2 ? 4 : 2><<<grid, 256, 0, p.stream>>>(q);
    else if (rank <= 128) lr_step_mma<T, 128, sizeof(T) == 2 ? 2 : 1><<<grid, 256, 0, p.stream>>>(q);
    else if constexpr (sizeof(T) == 2) lr_step_mma<T, 256, 1><<<grid, 256, 0, p.stream>>>(q);
  });
}

}  // namespace

hipError_t lr_step(const LrStep& p) {
  switch (p.dtype) {
    case kBF16: return launch<bf16>(p);
    case kFP16: return launch<fp16>(p);
    default: return launch<float>(p);
  }
}

}  // namespace dc
