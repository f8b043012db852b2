// The gated delta rule in chunks of tokens on matrix cores (formulas: delta.hip).
//
// Operands and results.  v_mfma_f32_16x16x32 leaves element (row, col) of its result in lane col + 16 (row/4), register
// row%4; an operand wants 8 values of the summed index in a lane.  Products sum in the order that two results of 16 rows
// come in (step s: 32 s + 16 (e/4) + 4 (lane/16) + e%4 for element e), so that the chain from the state to the next one,
// k S, T X, k^T Z, goes from results to operands without leaving the lane: a wavefront keeps 16 columns of S.  Rows of
// tiles lie in LDS so that a lane's 8 values of that order are neighbours (spot()); columns are read through transposing
// reads.
//
// Precision.  Operands are bf16 parts: q, k, v and dO one part (bf16), two (fp16: all of its bits) or three (float32); what is
// computed NP parts: three where a result is float32 (24 bits), else two (16 bits; results have 8 or 11).  In bf16 what goes
// through memory for the gradients takes 16 bits a value all the same: S, dS and Z are halves of 11 bits over a power of two
// of each lane's own (Half), and dX is dv, whose own rounding it is.  That leaves o, dq and dv at one rounding of their norm
// (1.7e-3 of it), dk and dlog_decay at 1.1 and dbeta (by k.W: dX.Z would have dX's rounding whole, 1.4) at 1.2.  With one bf16
// part of each (8 bits) they were 1.5, 1.7, 1.5, 1.9, 2.4 and 2.1 roundings off, in 0.8 of the time (B4 T4096 H16 hd128 training
// 663 us, 814).  A product of parts keeps those down to the last part's size.
// Sums, S and dS, decays and norms are float32; sums of logarithms of decays are float64.
#pragma once

#include <type_traits>

#include "layer_launch.h"
#include "lowrank_mfma.h"

namespace dc {
namespace dr {

constexpr float kTiny = 0x1p-60f;  // stands for a b of zero
// What a token's chunk keeps of it, floats: c in two parts, b, 1/|k|, 1/|q|, G/|k|, D b/|k|, scale G/|q| (the last five zero
// behind the last token).
constexpr int kC = 0, kB = 2, kRk = 3, kRq = 4, kGk = 5, kDk = 6, kGq = 7, kVecs = 8;

template <typename T> constexpr int parts_of() { return sizeof(T) == 4 ? 3 : __is_same(T, fp16) ? 2 : 1; }
// What goes through memory for the gradients is halves, and dX dv itself (B4 T4096 H16 hd128: 67 MB less to write).
template <typename T, int NP> constexpr bool kHalves = __is_same(T, bf16) && NP == 2;
constexpr int planes(bool halves, int np) { return halves ? 1 : np; }  // 16-bit words of a value there
// Tokens of a chunk: 64, or 32 where tiles of 64 would pass the LDS (three parts) or it and the registers (256 channels: B2 T4096
// H8 training in bf16 2509 us with 64, 1416 with 32).  np: parts of what is computed.
__host__ __device__ constexpr int chunk_of(int np, int kp) { return np == 3 || kp == 256 ? 32 : 64; }
__host__ __device__ constexpr int cover(int n) { return n <= 64 ? 64 : n <= 128 ? 128 : 256; }

struct Args {
  DrProblem p;
  float* vec;          // [chunks][kVecs][C]
  bf16 *tt, *pp;       // T and P, [chunks][NP][C][C], spot() order
  // Z and dX (not if kHalves) [chunks][planes][C][VP], states before and their gradients after [chunks][planes][KP][VP]; and if
  // kHalves the lanes' exponents of Z, states and gradients, [chunks][4][VP]
  bf16 *z, *x, *s, *ds;
  uint8_t *ez, *es, *eds;
  // tokens cut into nseg segments of seg (whole chunks): the states before each but the first [heads][nseg][K][V], the
  // gradients after each but the last, and what a segment makes of the state before it, [heads][nseg][KP][KP]
  float *start, *dstart, *trans;
  int seg, nseg, nw;  // nw: wavefronts of a chain's workgroup, 16 columns each
  int64_t n;           // chunks of a head
  int vp;              // V in whole 32 columns
  int64_t blk0, blocks;  // of this launch the first workgroup, of all its launches their number
  int nblk;
  bool kept;  // the forward keeps Z and the states
};

// Where column c of a row lies: of each 32 the quads of both halves side by side.
__host__ __device__ constexpr int spot(int c) { return (c & ~31) | ((c & 12) << 1) | ((c & 16) >> 2) | (c & 3); }

constexpr int kOut = 0x7FFFFFF0;  // a byte offset past every buffer's range

template <int N> struct Frag { u32x4 p[N]; };

template <int NA, int NB>
__device__ __forceinline__ f32x4 mma(const Frag<NA>& a, const Frag<NB>& b, f32x4 c) {
  constexpr int N = NA > NB ? NA : NB;
#pragma unroll
  for (int t = N - 1; t >= 0; --t)  // the smallest first
#pragma unroll
    for (int i = t; i >= 0; --i)
      if (i < NA && t - i < NB) c = Mma32<bf16>::run(a.p[i], b.p[t - i], c);
  return c;
}

// Two floats in N parts, a word of two for each.
template <int N>
__device__ __forceinline__ void split(float a, float b, uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = pack2<bf16>(a, b);
    if (i + 1 < N) {
      a -= __uint_as_float(w[i] << 16);
      b -= __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
}
// The operand of two results of 16 rows each.
template <int N>
__device__ __forceinline__ Frag<N> pack(f32x4 a, f32x4 b) {
  Frag<N> f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t w[N];
    if (e < 2) split<N>(a[2 * e], a[2 * e + 1], w);
    else split<N>(b[2 * e - 4], b[2 * e - 3], w);
#pragma unroll
    for (int i = 0; i < N; ++i) f.p[i][e] = w[i];
  }
  return f;
}

// Tiles that loads write themselves have no padding: of a row's 16-byte pieces, piece i lies at i ^ turn<W>(row), so that
// neither 16 rows of one piece nor 4 rows of 4 pieces meet in a bank.
template <int W>
__device__ __forceinline__ int turn(int row) {
  return W == 32 ? row >> 2 & 3 : W == 64 ? (row << 1 & 4) | (row >> 2 & 3) : (row << 2 & 12) | (row >> 2 & 3);
}

// Float32 values of a lane in halves over a power of two of the lane's own, which takes the largest of them to 2^14 .. 2^15:
// 11 bits of each that is not below 2^-28 of it.  A byte holds the power as a float's exponent bits.
struct Half {
  uint32_t byte;
  float by;
  template <int N>
  __device__ __forceinline__ explicit Half(const f32x4 (&v)[N]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(v[i][r]));
    byte = max((int)(__float_as_uint(m) >> 23) - 14, 1);
    by = __uint_as_float((254 - byte) << 23);
  }
  // as pack()
  __device__ __forceinline__ Frag<1> operator()(f32x4 a, f32x4 b) const {
    Frag<1> f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f.p[0][e] = e < 2 ? pack2<fp16>(a[2 * e] * by, a[2 * e + 1] * by) : pack2<fp16>(b[2 * e - 4] * by, b[2 * e - 3] * by);
    return f;
  }
};
// Eight such halves over the powers `by`, in two bf16 parts (8 and 3 bits, exact); `v`: their values.
__device__ __forceinline__ Frag<2> halves(u32x4 w, const f32x4 (&by)[2], float (&v)[8]) {
  Frag<2> f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t lo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = 2 * e + i;
      v[j] = Mma16<fp16>::to_f(i ? w[e] >> 16 : w[e] & 0xFFFFu) * by[j / 4][j % 4];
      lo[i] = __float_as_uint(v[j] - __uint_as_float(__float_as_uint(v[j]) & 0xFFFF0000u));
    }
    f.p[0][e] = __builtin_amdgcn_perm(__float_as_uint(v[2 * e + 1]), __float_as_uint(v[2 * e]), 0x07060302u);
    f.p[1][e] = __builtin_amdgcn_perm(lo[1], lo[0], 0x07060302u);
  }
  return f;
}
// The power of a byte.
__device__ __forceinline__ float power(uint32_t byte) { return __uint_as_float(byte << 23); }

// A tile in LDS: R elements from a row to the next, PL from a part to the next; TURN: its pieces turned, R of them whole.
template <int N, int R, int PL, bool TURN = false>
struct Tile {
  bf16* t;
  // row row0 + lane%16, step s of 32 columns
  __device__ __forceinline__ Frag<N> rows(int row0, int s) const {
    const int lane = threadIdx.x % 64;
    const bf16* p = t + (row0 + lane % 16) * R + (TURN ? 8 * ((4 * s + lane / 16) ^ turn<R>(lane % 16)) : 32 * s + 8 * (lane / 16));
    Frag<N> f;
#pragma unroll
    for (int i = 0; i < N; ++i) f.p[i] = *reinterpret_cast<const u32x4*>(p + i * PL);
    return f;
  }
  // column 16 cb + lane%16 of a tile in spot() order, step s of 32 rows; of one that lies as it is, column
  // 32 (cb/2) + 8 (lane%16/4) + 4 (cb%2) + lane%4
  __device__ __forceinline__ Frag<N> cols(int cb, int s) const {
    const int lane = threadIdx.x % 64, row = 4 * (lane / 16) + (lane % 16) / 4;
    const bf16* p = t + (32 * s + row) * R + 4 * (cb % 2) +
                    (TURN ? 8 * ((4 * (cb / 2) + lane % 4) ^ turn<R>(row)) : 32 * (cb / 2) + 8 * (lane % 4));
    Frag<N> f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const u32x2 a = lds_read_tr16(p + i * PL), b = lds_read_tr16(p + i * PL + 16 * R);
      f.p[i] = u32x4{a[0], a[1], b[0], b[1]};
    }
    return f;
  }
  // columns c .. c + 3 (a quad) of a row in spot() order
  __device__ __forceinline__ f32x4 four(int row, int c) const {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = N - 1; i >= 0; --i) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(t + row * R + spot(c) + i * PL);
      v += f32x4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xFFFF0000u), __uint_as_float(w[1] << 16),
                 __uint_as_float(w[1] & 0xFFFF0000u)};
    }
    return v;
  }
};

// C rows of W channels on their way from memory to a tile: 16-byte pieces that wait in registers.  WHOLE: rows are whole
// 16-byte pieces, no shorter apart than they are long and within 32-bit offsets: buffer loads, whose range drops the rows
// that are not there (loads under branches wait for one another).  Else they are gathered element by element.
template <typename T, int C, int W, int NT, bool WHOLE>
struct Rows {
  static constexpr int VE = 16 / (int)sizeof(T), PR = W / VE, NV = C * PR / NT, RPI = NT / PR;
  static_assert(C * PR % NT == 0 && NT % PR == 0, "whole pieces and rows to every thread");
  u32x4 v[NV];
  // rows 0 .. cnt-1 of base, `width` of the channels exist; the others are zero
  __device__ __forceinline__ void load(const T* base, int64_t stride, int width, int cnt) {
    const int r0 = (int)threadIdx.x / PR, c = (int)threadIdx.x % PR * VE;
    if constexpr (WHOLE) {  // the range ends behind the last row
      const rsrc_t rs = make_rsrc_wave(base, ((int64_t)(cnt - 1) * stride + width) * (int64_t)sizeof(T));
      const int sb = (int)stride * (int)sizeof(T), off = r0 * sb + c * (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = bload128(rs, c < width ? off + i * RPI * sb : kOut);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int r = r0 + i * RPI;
        T e[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) e[j] = r < cnt && c + j < width ? base[(int64_t)r * stride + c + j] : (T)0.f;
        __builtin_memcpy(&v[i], e, 16);
      }
    }
  }
  // into a tile of R elements a row, in spot() order or as they are
  template <int R, int PL, bool SPOT>
  __device__ __forceinline__ void store(bf16* lds) const {
    const int c = (int)threadIdx.x % PR * VE;
    bf16* to = lds + (int)threadIdx.x / PR * R;
#pragma unroll
    for (int i = 0; i < NV; ++i, to += RPI * R) {
      if constexpr (sizeof(T) == 4) {
        uint32_t a[3], b[3];
        split<3>(__uint_as_float(v[i][0]), __uint_as_float(v[i][1]), a);
        split<3>(__uint_as_float(v[i][2]), __uint_as_float(v[i][3]), b);
#pragma unroll
        for (int j = 0; j < 3; ++j) *reinterpret_cast<u32x2*>(to + (SPOT ? spot(c) : c) + j * PL) = u32x2{a[j], b[j]};
      } else {
        constexpr int N = parts_of<T>();
        u32x4 w[N];
        if constexpr (N == 1) {
          w[0] = v[i];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t ab[2];
            split<2>(Mma16<T>::to_f(v[i][e] & 0xFFFFu), Mma16<T>::to_f(v[i][e] >> 16), ab);
            w[0][e] = ab[0];
            w[1][e] = ab[1];
          }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if constexpr (SPOT) {
            *reinterpret_cast<u32x2*>(to + spot(c) + j * PL) = u32x2{w[j][0], w[j][1]};
            *reinterpret_cast<u32x2*>(to + spot(c + 4) + j * PL) = u32x2{w[j][2], w[j][3]};
          } else {
            *reinterpret_cast<u32x4*>(to + c + j * PL) = w[j];
          }
        }
      }
    }
  }
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

// What each chunk needs of its own keys: a workgroup of four wavefronts to a chunk of one head, four workgroups to a CU.
// B4 T4096 H16 hd128 bf16 68 us for 277 MB (4.1 TB/s; a third slower before its products' factors came in quads, unbranched):
// what it waits for is the substitution's 16 steps and the barriers around them, and the four hide each other's.
template <typename T, int NP, int KP, bool WHOLE>
__global__ __launch_bounds__(256) void dr_prep(Args a) {
  constexpr int NI = parts_of<T>(), C = chunk_of(NP, KP), NB = C / 16, R = KP + 8, PL = C * R, RA = C + 4;
  constexpr int TILES = 2 * NI * PL * 2, MATS = 2 * C * RA * 4;
  __shared__ __align__(16) unsigned char mem[TILES > MATS ? TILES : MATS];
  // of each token: c in two parts, b, 1/|k|, 1/|q|, the factors of A's and P's rows 1/|k| and scale/|q| and of their columns b/|k|
  __shared__ __align__(16) float chi[C], clo[C], be[C], rk[C], rq[C], by[2][C], bk[C];
  bf16 *lk = reinterpret_cast<bf16*>(mem), *lq = lk + NI * PL;
  float (*A)[RA] = reinterpret_cast<float (*)[RA]>(mem), (*X)[RA] = A + C;
  const DrProblem& p = a.p;
  const int64_t blk = a.blk0 + blockIdx.x, n = blk % a.n, bh = blk / a.n, b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
  const int t0 = (int)n * C, len = length_of(p, b), t = threadIdx.x, lane = t % 64, g = lane / 16, col = lane % 16, wv = wave_id();
  if (t0 >= len) return;
  const int cnt = min(C, len - t0);
  {
    Rows<T, C, KP, 256, WHOLE> k, q;
    k.load((const T*)p.k + b * p.ks[0] + hk * p.ks[1] + (int64_t)t0 * p.ks[2], p.ks[2], (int)p.K, cnt);
    q.load((const T*)p.q + b * p.qs[0] + hk * p.qs[1] + (int64_t)t0 * p.qs[2], p.qs[2], (int)p.K, cnt);
    k.template store<R, PL, false>(lk);
    q.template store<R, PL, false>(lq);
  }
  if (wv == 0) {
    // a token to a lane; the sums in float64: their differences count to the last place
    const bool live = lane < cnt;
    float lam = live ? gate_at(p.g, p.gdtype, b * p.gs[0] + h * p.gs[1] + (t0 + lane) * p.gs[2]) : 0.f;
    lam = lam < -128.f ? -128.f : lam;  // e^-128 is nothing to float32, and differences stay finite
    double c = lam;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const double o = __shfl_up(c, m);
      if (lane >= m) c += o;
    }
    const float bt = live ? gate_at(p.b, p.gdtype, b * p.bs[0] + h * p.bs[1] + (t0 + lane) * p.bs[2]) : 0.f;
    if (lane < C) {
      chi[lane] = (float)c;
      clo[lane] = (float)(c - (double)(float)c);
      be[lane] = fabsf(bt) < kTiny ? kTiny : bt;
    }
  }
  __syncthreads();
  const Tile<NI, R, PL> tk{lk}, tq{lq};
  {
    constexpr int TPR = 256 / C, CH = KP / TPR;  // threads to a row, channels to a thread
    const int row = t / TPR, c0 = t % TPR * CH;
    float s[2] = {0.f, 0.f};
    if (p.normalize)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll 4
        for (int c = 0; c < CH; c += 8) {
          u32x4 w[NI];
#pragma unroll
          for (int i = 0; i < NI; ++i) w[i] = *reinterpret_cast<const u32x4*>((m ? lq : lk) + row * R + c0 + c + i * PL);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = 0.f, y = 0.f;
#pragma unroll
            for (int i = NI - 1; i >= 0; --i) {
              x += __uint_as_float(w[i][e] << 16);
              y += __uint_as_float(w[i][e] & 0xFFFF0000u);
            }
            s[m] += x * x + y * y;
          }
        }
#pragma unroll
    for (int m = 1; m < TPR; m *= 2) {
      s[0] += __shfl_xor(s[0], m);
      s[1] += __shfl_xor(s[1], m);
    }
    if (t % TPR == 0) {
      // rows from cnt on are no tokens: factors of zero keep them out of everything, also where eps is zero
      const float one = row < cnt ? 1.f : 0.f, ik = row < cnt && p.normalize ? 1.f / sqrtf(s[0] + p.eps) : one,
                  iq = row < cnt && p.normalize ? 1.f / sqrtf(s[1] + p.eps) : one;
      rk[row] = ik;
      rq[row] = iq;
      by[0][row] = ik;
      by[1][row] = p.scale * iq;
      bk[row] = be[row] * ik;
    }
  }
  // blocks on and below the diagonal, k k^T and q k^T, round the wavefronts
  constexpr int NBL = NB * (NB + 1) / 2, NU = (2 * NBL + 3) / 4;
  f32x4 acc[NU];
  auto unit = [&](int i, int& m, int& rb, int& cb) {  // of this wavefront
    const int u = wv + 4 * i, e = u - (u >= NBL ? NBL : 0);
    m = u >= NBL;
    rb = (e >= 1) + (e >= 3) + (e >= 6);
    cb = e - rb * (rb + 1) / 2;
    return u < 2 * NBL;
  };
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    int m, rb, cb;
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!unit(i, m, rb, cb)) continue;
#pragma unroll
    for (int s = 0; s < KP / 32; ++s) acc[i] = mma((m ? tq : tk).rows(16 * rb, s), tk.rows(16 * cb, s), acc[i]);
  }
  __syncthreads();  // the tiles have been read; rk and rq are there
  if (t < C) {
    float* vec = a.vec + blk * kVecs * C + t;
    const float G = expf(chi[t]) * (1.f + clo[t]), D = expf((chi[C - 1] - chi[t]) + (clo[C - 1] - clo[t]));
    vec[0] = chi[t];
    vec[C] = clo[t];
    vec[kB * C] = be[t];
    vec[kRk * C] = rk[t];
    vec[kRq * C] = rq[t];
    vec[kGk * C] = G * rk[t];
    vec[kDk * C] = D * bk[t];
    vec[kGq * C] = p.scale * G * rq[t];
  }
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    int m, rb, cb;
    if (!unit(i, m, rb, cb)) continue;
    const int j = 16 * cb + col, x = 16 * rb + 4 * g;
    const f32x4 hi = *reinterpret_cast<const f32x4*>(&chi[x]), lo = *reinterpret_cast<const f32x4*>(&clo[x]),
                row = *reinterpret_cast<const f32x4*>(&by[m][x]);
    const float hj = chi[j], lj = clo[j], kj = bk[j];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float c = ((hi[r] - hj) + (lo[r] - lj)) * 1.44269504088896f;
      acc[i][r] *= __builtin_amdgcn_exp2f(j < x + r + m ? c : -__builtin_inff()) * row[r] * kj;  // without a branch
      if (!m) A[x + r][j] = acc[i][r];
    }
  }
  __syncthreads();
  // (1 + A)^-1: the blocks on the diagonal column by column, those below from the diagonal outwards,
  // X_ij = -X_ii sum_{j<=l<i} A_il X_lj, on float32 matrix instructions
  if (wv < NB) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == col ? 1.f : 0.f;
#pragma unroll
      for (int l = 0; l < i; ++l) s -= A[16 * wv + i][16 * wv + l] * x[l];
      x[i] = s;
    }
    if (g == 0)
#pragma unroll
      for (int i = 0; i < 16; ++i) X[16 * wv + i][16 * wv + col] = x[i];
  }
#pragma unroll
  for (int d = 1; d < NB; ++d) {
    __syncthreads();
    if (wv < NB - d) {
      const int i = wv + d, j = wv;
      f32x4 m = {0.f, 0.f, 0.f, 0.f}, x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int l = 0; l < d; ++l)
#pragma unroll
        for (int s = 0; s < 4; ++s)
          m = __builtin_amdgcn_mfma_f32_16x16x4f32(A[16 * i + col][16 * (j + l) + 4 * s + g], X[16 * (j + l) + 4 * s + g][16 * j + col],
                                                   m, 0, 0, 0);
#pragma unroll
      for (int s = 0; s < 4; ++s) x = __builtin_amdgcn_mfma_f32_16x16x4f32(X[16 * i + col][16 * i + 4 * g + s], m[s], x, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) X[16 * i + 4 * g + r][16 * j + col] = -x[r];
    }
  }
  __syncthreads();
  // P takes A's place, and both leave in parts and in spot() order
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    int m, rb, cb;
    if (!unit(i, m, rb, cb) || !m) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) A[16 * rb + 4 * g + r][16 * cb + col] = acc[i][r];
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int e = t; e < C * C / 8; e += 256) {
      const int x = e / (C / 8), c = e % (C / 8) * 8, j0 = (c & ~31) | ((c & 24) >> 1);  // columns j0 .. j0+3 and 16 on of row x
      f32x4 v[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int j = j0 + 16 * w;
        v[w] = *reinterpret_cast<const f32x4*>(&(m ? A : X)[x][j]);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[w][r] = j + r > x ? 0.f : v[w][r];
      }
      const Frag<NP> f = pack<NP>(v[0], v[1]);
#pragma unroll
      for (int i = 0; i < NP; ++i)
        *reinterpret_cast<u32x4*>((m ? a.pp : a.tt) + ((blk * NP + i) * C + x) * C + c) = f.p[i];
    }
}

// A chunk's T or P on its way to LDS.
template <int NP, int C, int NT>
struct Square {
  static constexpr int NV = NP * C * C / 8 / NT;
  static_assert(NP * C * C / 8 % NT == 0, "whole pieces to every thread");
  u32x4 v[NV];
  __device__ __forceinline__ void load(const bf16* from) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = *reinterpret_cast<const u32x4*>(from + (threadIdx.x + i * NT) * 8);
  }
  __device__ __forceinline__ void store(bf16* lds) const {  // C + 8 elements a row
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (threadIdx.x + i * NT) * 8;
      *reinterpret_cast<u32x4*>(lds + e / C * (C + 8) + e % C) = v[i];
    }
  }
};

// Rows of halves (Rows<bf16>, as they are) over the powers of their columns into a tile of two parts.
template <int R, int PL, typename ROWS>
__device__ __forceinline__ void store_halves(const ROWS& rows, const f32x4 (&by)[2], bf16* lds) {
  bf16* to = lds + (int)threadIdx.x / ROWS::PR * R + (int)threadIdx.x % ROWS::PR * 8;
#pragma unroll
  for (int i = 0; i < ROWS::NV; ++i, to += ROWS::RPI * R) {
    float v[8];
    const Frag<2> f = halves(rows.v[i], by, v);
#pragma unroll
    for (int j = 0; j < 2; ++j) *reinterpret_cast<u32x4*>(to + j * PL) = f.p[j];
  }
}

// 16 columns of C rows as results lie: element r of v[rb] is row 16 rb + 4 (lane/16) + r, column lane%16.
template <typename T, int C, bool WHOLE>
struct Columns {
  typedef typename Unit<sizeof(T)>::type U;
  U v[C / 16][4];
  __device__ static __forceinline__ U load1(rsrc_t rs, int off, int more) {
    if constexpr (sizeof(T) == 2) return (U)__builtin_amdgcn_raw_buffer_load_b16(rs, off, more, 0);
    else return (U)__builtin_amdgcn_raw_buffer_load_b32(rs, off, more, 0);
  }
  // base: row 0 of this lane's column; cnt rows, `left` columns from the wavefront's first on
  __device__ __forceinline__ void load(const T* base, int64_t stride, int left, int cnt) {
    const int g = threadIdx.x % 64 / 16, col = threadIdx.x % 16;
    if constexpr (WHOLE) {
      const rsrc_t rs = make_rsrc_wave(base - col, ((int64_t)(cnt - 1) * stride + left) * (int64_t)sizeof(T));
      const int sb = (int)stride * (int)sizeof(T), off = col < left ? 4 * g * sb + col * (int)sizeof(T) : kOut - 64 * sb;
      if (cnt == C) {  // every row is there: the range need only drop columns, which it does without the scalar offset
#pragma unroll
        for (int rb = 0; rb < C / 16; ++rb)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[rb][r] = load1(rs, off, (16 * rb + r) * sb);
      } else {
#pragma unroll
        for (int rb = 0; rb < C / 16; ++rb)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[rb][r] = load1(rs, off + (16 * rb + r) * sb, 0);
      }
    } else {
#pragma unroll
      for (int rb = 0; rb < C / 16; ++rb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * rb + 4 * g + r;
          const T e = col < left && row < cnt ? base[row * stride] : (T)0.f;
          __builtin_memcpy(&v[rb][r], &e, sizeof(T));
        }
    }
  }
  __device__ __forceinline__ f32x4 get(int rb) const {
    f32x4 f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = (float)__builtin_bit_cast(T, v[rb][r]);
    return f;
  }
};
// Results of 16 rows (row0 ..) into such columns, rows below cnt.
template <typename T, bool WHOLE>
__device__ __forceinline__ void put_columns(T* base, int64_t stride, int left, int cnt, int row0, f32x4 y) {
  const int g = threadIdx.x % 64 / 16, col = threadIdx.x % 16;
  if constexpr (WHOLE) {
    const rsrc_t rs = make_rsrc_wave(base - col, ((int64_t)(cnt - 1) * stride + left) * (int64_t)sizeof(T));
    const int sb = (int)stride * (int)sizeof(T), off = col < left ? (row0 + 4 * g) * sb + col * (int)sizeof(T) : kOut - 4 * sb;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      BufUnit<sizeof(T)>::template store<false>(__builtin_bit_cast(typename Unit<sizeof(T)>::type, (T)y[r]), rs, off + r * sb);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col < left && row0 + 4 * g + r < cnt) base[(row0 + 4 * g + r) * stride] = (T)y[r];
  }
}

// An operand of 32 rows and this wavefront's 16 columns into [NP][rows][vp], `plane` elements a part; element e of a lane is
// row 8 g + e (states) or 16 (e/4) + 4 g + e%4 (tokens).  Neighbouring lanes trade halves, so that a store has two columns of
// a row (48 two-byte stores a chunk took 20% of the chain that keeps).
template <int NP, bool STATE>
__device__ __forceinline__ void keep(bf16* to, int vp, int64_t plane, const Frag<NP>& f) {
  const int g = threadIdx.x % 64 / 16, col = threadIdx.x % 16, odd = col % 2;
  const rsrc_t rs = make_rsrc_wave(to, ((NP - 1) * plane + 32 * vp) * 2);
  const int off = (((STATE ? 8 : 4) * g + odd) * vp + col - odd) * 2;
  const uint32_t sel = odd ? 0x03020706u : 0x05040100u;  // (the neighbour's, own) high halves, or (own, its) low halves
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t own = f.p[i][e], its = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)own, 0xB1, 0xF, 0xF, false);
      const int more = ((int)(i * plane) + (STATE ? 2 * e : 16 * (e / 2) + 2 * (e % 2)) * vp) * 2;
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_amdgcn_perm(its, own, sel), rs, off, more, 0);
    }
}

// A chunk's states (or their gradients) of this wavefront's columns into memory: halves, or the parts that are there.
template <typename T, int NP, int KP>
__device__ __forceinline__ void keep_state(bf16* to, uint8_t* exponents, int64_t ch, int vp, int n0, const f32x4 (&S)[KP / 16],
                                           const Frag<NP> (&parts)[KP / 32]) {
  if constexpr (kHalves<T, NP>) {
    const Half half(S);
#pragma unroll
    for (int s = 0; s < KP / 32; ++s) keep<1, true>(to + (ch * KP + 32 * s) * vp + n0, vp, 0, half(S[2 * s], S[2 * s + 1]));
    exponents[(ch * 4 + threadIdx.x % 64 / 16) * vp + n0 + threadIdx.x % 16] = (uint8_t)half.byte;
  } else {
#pragma unroll
    for (int s = 0; s < KP / 32; ++s) keep<NP, true>(to + (ch * NP * KP + 32 * s) * vp + n0, vp, (int64_t)KP * vp, parts[s]);
  }
}

// Nothing moves across the end of a phase: without it the compiler sinks a batch of operands to its use, which then waits.
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// A lane's part of a state: element r of S[kb] is channel 32 (kb/2) + 8 g + 4 (kb%2) + r of q and k, so that an operand of
// two results holds 8 neighbouring channels, as they lie in a row of a tile.
template <int KP>
__device__ __forceinline__ void load_state(f32x4 (&S)[KP / 16], const float* from, bool live, int K, int V) {
  const int g = threadIdx.x % 64 / 16;
#pragma unroll
  for (int kb = 0; kb < KP / 16; ++kb)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 32 * (kb / 2) + 8 * g + 4 * (kb % 2) + r;
      S[kb][r] = from && live && d < K ? from[d * V] : 0.f;
    }
}
template <int KP>
__device__ __forceinline__ void store_state(const f32x4 (&S)[KP / 16], float* to, int K, int V) {
  const int g = threadIdx.x % 64 / 16;
#pragma unroll
  for (int kb = 0; kb < KP / 16; ++kb)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 32 * (kb / 2) + 8 * g + 4 * (kb % 2) + r;
      if (d < K) to[d * V] = S[kb][r];
    }
}

// The chains' scales of a chunk on their way to LDS: G/|k|, D b/|k|, scale G/|q|; top: the whole chunk's decay's logarithm.
// Every thread loads and stores as many, those past the 3 C for their wavefront's sake (load_direct): 4 C lie in LDS.
template <int C, int NT>
struct Scales {
  static_assert(4 * C % NT == 0, "every wavefront loads scales and stores them");
  static constexpr int N = 4 * C / NT;
  float v[N], top = 0.f;
  __device__ __forceinline__ void load(const float* vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = i * NT + (int)threadIdx.x;
      v[i] = vec[kGk * C + (e < 3 * C ? e : 0)];
    }
    top = vec[C - 1];
  }
  __device__ __forceinline__ void store(float* lds) const {
#pragma unroll
    for (int i = 0; i < N; ++i) lds[i * NT + (int)threadIdx.x] = v[i];
  }
};

// C rows of W channels from memory into a turned tile, by loads that write LDS themselves (16 bytes a lane, 1 KB of the tile
// a wavefront): no registers hold them.  Rows from cnt on repeat the last one; their scales are zero.  Memory operations complete in order: a
// wavefront that has waited for a later load of its own has these in LDS too, and the barrier after that makes them
// everybody's.  That load is the scales', which every wavefront issues behind these and stores to LDS before the barrier.
// Waiting for all, stores among them, took half of the time of the chains that keep states.
template <int C, int W, int NW>
__device__ __forceinline__ void load_direct(const bf16* base, int64_t stride, int cnt, bf16* lds) {
  constexpr int PR = W / 8, N = C * PR / (NW * 64), RPL = (NW * 64) / PR;  // pieces of a row, loads, rows of a load
  constexpr int VAR = RPL < 16 ? 16 / RPL : 1;                 // loads after which the rows' turns repeat
  static_assert(C * PR % (NW * 64) == 0 && N % VAR == 0, "whole loads");
  const rsrc_t rs = make_rsrc_wave(base, ((int64_t)(cnt - 1) * stride + W) * 2);
  const int wv = wave_id(), lane = threadIdx.x % 64, sb = (int)stride * 2;
  const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) bf16*)lds + wv * 1024;
  auto place = [&](int i, int last) {
    const int row = ((i * NW + wv) * 64 + lane) / PR;
    return min(row, last) * sb + 16 * ((lane % PR) ^ turn<W>(row));
  };
  auto load = [&](int i, int off, int more) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to + i * NW * 1024), "v"(off),
                 "s"(rs), "s"(more)
                 : "m0", "memory");
  };
  if (cnt == C) {
#pragma unroll
    for (int i = 0; i < N; ++i) load(i, place(i % VAR, C), i / VAR * VAR * RPL * sb);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) load(i, place(i, cnt - 1), 0);
  }
}

// How rows reach the chains' tiles.
enum Mode { kGather, kWhole, kDirect };

// Tiles of one buffer that leave room for four workgroups on a CU, two wavefronts to a SIMD, where those of two leave two
// (bf16 with float32 results at 128 channels): with workgroups enough they hide each other's latencies, and the chains take
// rows through registers (B1 T32768 H16: outputs 416 -> 322 us, segments 405 -> 363; B2 T4096 H16 backward's segments 133 ->
// 93). With fewer the second buffer does (512 workgroups of outputs 113 us, 128 through registers), and in the backward's
// chain, whose registers are a wavefront's alone (250 us, 260).
template <typename T, int NP, int KP>
constexpr bool kShares = __is_same(T, bf16) && NP == 3 && KP == 128;

// What the chains share: the sizes of their tiles in LDS, k, q, T, P and the scales, twice where loads write them directly.
// The memory is asked for at the launch: with its size in sight the compiler takes one wavefront to a SIMD for granted, and
// 512 registers, of which half are accumulation registers, whose moves were 300 of 490 vector instructions a chunk.
template <typename T, int NP, int KP, int MODE>
struct ChainSize {
  static constexpr bool DIRECT = MODE == kDirect;
  static constexpr int NI = parts_of<T>(), C = chunk_of(NP, KP), NB = C / 16, R = KP + (DIRECT ? 0 : 24), PL = C * R,
                       RC = C + (DIRECT ? 0 : 8), PC = C * RC;
  // steps of an operands' batch, one ahead of the products: two parts' products of one step take as long as one part's of two
  static constexpr int STEPS = NP == 2 ? 1 : 2;
  static constexpr int BUF = DIRECT ? 2 : 1, KEYS = NI * PL, SQUARE = NP * PC;
  static constexpr int bytes(bool both) { return BUF * ((both ? 2 : 1) * (KEYS + SQUARE) * 2 + 4 * C * 4); }
  static constexpr int WAVES = DIRECT && NP == 2 || kShares<T, NP, KP> && MODE == kWhole ? 2 : 1;
};

// bf16 rows of whole tiles, where two buffers fit.
template <typename T, int NP, int KP>
constexpr bool kHasDirect = __is_same(T, bf16) && ChainSize<T, NP, KP, kDirect>::bytes(true) <= 160 * 1024;

// Tiles that leave room for one workgroup on a CU: four wavefronts to it instead of two, where there are columns for them.
template <typename T, int NP, int KP>
constexpr bool kHasFour = kHalves<T, NP> && KP == 128;

// The states from chunk to chunk, and o (kOutputs); or Z and the state before each chunk for the backward (kKeep); or all of
// these (kBoth); or what each segment but the last makes of the state before it (kAcross): its end from zero, and behind those
// columns its end from each unit vector without values.
//
// A chunk waits for the one before it, so a chain's time is its chunks': 3.7 us each at 128 x 128 in bf16, 4.5 with the
// states' stores (B4 T4096 H16: 64 chunks, 235 and 289 us).  Of that 0.9 us are matrix instructions and about half all
// instructions of a wavefront that has its SIMD to itself; the rest are latencies, of operands from LDS within a chunk, and of
// the next chunk's loads, for which a second buffer leaves the time of one chunk and LDS has no third.  With one part of each
// operand, another wavefront beside each for the outputs and one for the loads took 146 us for 180 without the stores, but the
// same 222 with them, and lost to four wavefronts where heads abound (B4 T2048 H32 forward 219 us for 175): not here.
enum What { kOutputs, kKeep, kBoth, kAcross };
template <typename T, int NP, int KP, int MODE, int WHAT, int NW>
__global__ __launch_bounds__(NW * 64, (ChainSize<T, NP, KP, MODE>::WAVES)) void dr_chain(Args a) {
  typedef ChainSize<T, NP, KP, MODE> Z;
  constexpr int NI = Z::NI, C = Z::C, NB = Z::NB, R = Z::R, PL = Z::PL, RC = Z::RC, PC = Z::PC;
  constexpr bool DIRECT = Z::DIRECT, WHOLE = MODE != kGather;
  constexpr bool OUT = WHAT == kOutputs || WHAT == kBoth, KEEP = WHAT == kKeep || WHAT == kBoth;  // !OUT: no q and no o
  extern __shared__ __align__(16) unsigned char chain_lds[];
  float (*lv)[4][C] = reinterpret_cast<float (*)[4][C]>(chain_lds);
  bf16 (*lk)[Z::KEYS] = reinterpret_cast<bf16 (*)[Z::KEYS]>(lv + Z::BUF);
  bf16 (*lt)[Z::SQUARE] = reinterpret_cast<bf16 (*)[Z::SQUARE]>(lk + Z::BUF);
  bf16 (*lq)[Z::KEYS] = reinterpret_cast<bf16 (*)[Z::KEYS]>(lt + Z::BUF);  // there if OUT
  bf16 (*lp)[Z::SQUARE] = reinterpret_cast<bf16 (*)[Z::SQUARE]>(lq + Z::BUF);
  const DrProblem& p = a.p;
  // columns: V's, and behind them those of the unit vectors
  const int nvb = (a.vp + (WHAT == kAcross ? KP : 0)) / (NW * 16), nseg = WHAT == kAcross ? a.nseg - 1 : a.nseg;
  int64_t blk = a.blk0 + xcd_remap(blockIdx.x, a.nblk);
  const int vb = (int)(blk % nvb);
  blk /= nvb;
  const int seg = (int)(blk % nseg);
  const int64_t bh = blk / nseg, b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
  const int lane = threadIdx.x % 64, g = lane / 16, col = lane % 16;
  const int n0 = vb * NW * 16 + wave_id() * 16, nn = n0 + col, K = (int)p.K, V = (int)p.V;
  const bool live = nn < V, unit = WHAT == kAcross && vb * NW * 16 >= a.vp;
  if (unit && seg == 0) return;  // the state before the first segment is known
  const int lo = seg * a.seg, len = min(length_of(p, b), lo + a.seg), whole = length_of(p, b);
  const T* q = (const T*)p.q + b * p.qs[0] + hk * p.qs[1];
  const T* k = (const T*)p.k + b * p.ks[0] + hk * p.ks[1];
  const T* v = (const T*)p.v + b * p.vs[0] + h * p.vs[1] + nn;
  T* o = (T*)p.o + b * p.os[0] + h * p.os[1] + n0;
  const int64_t sb = bh * K * V + nn;
  f32x4 S[KP / 16];
  const int64_t at0 = (bh * a.nseg + seg) * K * V + nn;
  if (unit) {
#pragma unroll
    for (int kb = 0; kb < KP / 16; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[kb][r] = 32 * (kb / 2) + 8 * g + 4 * (kb % 2) + r == nn - a.vp ? 1.f : 0.f;
  } else {
    const float* from = seg == 0 ? (p.s_in ? p.s_in + sb : nullptr) : WHAT == kAcross ? nullptr : a.start + at0;
    load_state<KP>(S, from, live, K, V);
  }
  Rows<T, C, KP, NW * 64, WHOLE> rk, rq;
  Square<NP, C, NW * 64> rt, rp;
  Columns<T, C, WHOLE> cv;
  Scales<C, NW * 64> vec;
  auto fetch = [&](int t0, int buf) {
    if (t0 >= len) return;
    const int cnt = min(C, len - t0);
    const int64_t ch = bh * a.n + t0 / C;
    const T *kt = k + (int64_t)t0 * p.ks[2], *qt = q + (int64_t)t0 * p.qs[2];
    const bf16 *tt = a.tt + ch * NP * C * C, *pt = a.pp + ch * NP * C * C;
    if constexpr (DIRECT) {
      load_direct<C, KP, NW>(kt, p.ks[2], cnt, lk[buf]);
      load_direct<NP * C, C, NW>(tt, C, NP * C, lt[buf]);
      if (OUT) {
        load_direct<C, KP, NW>(qt, p.qs[2], cnt, lq[buf]);
        load_direct<NP * C, C, NW>(pt, C, NP * C, lp[buf]);
      }
    } else {
      rk.load(kt, p.ks[2], K, cnt);
      rt.load(tt);
      if (OUT) {
        rq.load(qt, p.qs[2], K, cnt);
        rp.load(pt);
      }
    }
    cv.load(v + (int64_t)t0 * p.vs[2], p.vs[2], unit ? 0 : V - n0, cnt);
    vec.load(a.vec + ch * kVecs * C);
  };
  auto arrive = [&](int buf) {  // what fetch() left in registers
    if constexpr (!DIRECT) {
      rk.template store<R, PL, false>(lk[buf]);
      rt.store(lt[buf]);
      if (OUT) {
        rq.template store<R, PL, false>(lq[buf]);
        rp.store(lp[buf]);
      }
    }
    vec.store(lv[buf][0]);
  };
  fetch(lo, 0);
  f32x4 x[NB];
  auto arrived = [&](int buf) {
    arrive(buf);
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) x[rb] = cv.get(rb);
  };
  arrived(0);
  int buf = 0;
  for (int t0 = lo; t0 < len; t0 += C, buf ^= DIRECT) {
    const int cnt = min(C, len - t0);
    const int64_t ch = bh * a.n + t0 / C;
    __syncthreads();  // this chunk is there (and the other buffer has been read)
    const Tile<NI, R, PL, DIRECT> tk{lk[buf]}, tq{lq[buf]};
    const Tile<NP, RC, PC, DIRECT> tt{lt[buf]}, tp{lp[buf]};
    const float (*sc)[C] = lv[buf];
    const float gc = expf(vec.top);
    fetch(t0 + C, buf ^ DIRECT);
    f32x4 y[NB];
    // X = V - G k S
    constexpr int ST = Z::STEPS;
    Frag<NI> even[ST][NB], odd[ST][NB];
    auto rows = [&](const Tile<NI, R, PL, DIRECT>& t, Frag<NI> (&f)[ST][NB], int s) {
#pragma unroll
      for (int i = 0; i < ST; ++i)
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) f[i][rb] = t.rows(16 * rb, s + i);
      phase();
    };
    rows(tk, even, 0);
    Frag<NP> sf[KP / 32];
#pragma unroll
    for (int s = 0; s < KP / 32; ++s) sf[s] = pack<NP>(S[2 * s], S[2 * s + 1]);
    if constexpr (KEEP) keep_state<T, NP, KP>(a.s, a.es, ch, a.vp, n0, S, sf);
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) y[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
    Frag<NP> tr[NB][NB / 2];
    auto square = [&](const Tile<NP, RC, PC, DIRECT>& t) {
#pragma unroll
      for (int rb = 0; rb < NB; ++rb)
#pragma unroll
        for (int s = 0; s <= rb / 2; ++s) tr[rb][s] = t.rows(16 * rb, s);
      phase();
    };
#pragma unroll
    for (int s = 0; s < KP / 32; s += ST) {
      Frag<NI> (&now)[ST][NB] = s / ST % 2 ? odd : even, (&then)[ST][NB] = s / ST % 2 ? even : odd;
      if (s + ST < KP / 32) rows(tk, then, s + ST);
      else square(tt);
#pragma unroll
      for (int i = 0; i < ST; ++i)
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) y[rb] = mma(now[i][rb], sf[s + i], y[rb]);
      phase();
    }
    // operands of k^T: batches of 8, the step of 32 tokens first
    constexpr int KN = KP / 16, NK = KN * (C / 32);
    Frag<NI> kc[2][NK < 8 ? NK : 8];
    auto keys = [&](int e0) {
#pragma unroll
      for (int e = 0; e < 8 && e < NK; ++e) kc[e0 / 8 % 2][e] = tk.cols((e0 + e) % KN, (e0 + e) / KN);
      phase();
    };
    if (ST > 1) keys(0);
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) x[rb] -= *reinterpret_cast<const f32x4*>(&sc[0][16 * rb + 4 * g]) * y[rb];
    Frag<NP> f[C / 32], d[C / 32];
#pragma unroll
    for (int s = 0; s < C / 32; ++s) f[s] = pack<NP>(x[2 * s], x[2 * s + 1]);
    // Z = T X
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) x[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NB / 2; ++s)
#pragma unroll
      for (int rb = 2 * s; rb < NB; ++rb) x[rb] = mma(tr[rb][s], f[s], x[rb]);
    if (ST == 1) keys(0);  // two parts' T has left its registers by now
#pragma unroll
    for (int kb = 0; kb < KN; ++kb) S[kb] *= gc;
#pragma unroll
    for (int s = 0; s < C / 32; ++s) {
      f[s] = pack<NP>(x[2 * s], x[2 * s + 1]);
      if constexpr (KEEP && !kHalves<T, NP>) keep<NP, false>(a.z + (ch * NP * C + 32 * s) * a.vp + n0, a.vp, (int64_t)C * a.vp, f[s]);
      d[s] = pack<NP>(x[2 * s] * *reinterpret_cast<const f32x4*>(&sc[1][32 * s + 4 * g]),
                      x[2 * s + 1] * *reinterpret_cast<const f32x4*>(&sc[1][32 * s + 16 + 4 * g]));
    }
    if constexpr (KEEP && kHalves<T, NP>) {
      const Half half(x);
#pragma unroll
      for (int s = 0; s < C / 32; ++s) keep<1, false>(a.z + (ch * C + 32 * s) * a.vp + n0, a.vp, 0, half(x[2 * s], x[2 * s + 1]));
      a.ez[(ch * 4 + g) * a.vp + nn] = (uint8_t)half.byte;
    }
    phase();
    // S <- G_C S + k^T D b Z
#pragma unroll
    for (int e0 = 0; e0 < NK; e0 += 8) {
      if (e0 + 8 < NK) keys(e0 + 8);
      else if (OUT) rows(tq, even, 0);
#pragma unroll
      for (int e = 0; e < 8 && e < NK; ++e) {
        const int kb = (e0 + e) % KN, s = (e0 + e) / KN;
        S[kb] = mma(kc[e0 / 8 % 2][e], d[s], S[kb]);
      }
      phase();
    }
    // O^T = G S^T q^T + Z^T P^T: four neighbouring channels of a token in a lane
    if constexpr (OUT) {
#pragma unroll
      for (int rb = 0; rb < NB; ++rb) y[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KP / 32; s += ST) {
        Frag<NI> (&now)[ST][NB] = s / ST % 2 ? odd : even, (&then)[ST][NB] = s / ST % 2 ? even : odd;
        if (s + ST < KP / 32) rows(tq, then, s + ST);
        else square(tp);
#pragma unroll
        for (int i = 0; i < ST; ++i)
#pragma unroll
          for (int rb = 0; rb < NB; ++rb) y[rb] = mma(sf[s + i], now[i][rb], y[rb]);
        phase();
      }
#pragma unroll
      for (int rb = 0; rb < NB; ++rb) y[rb] *= sc[2][16 * rb + col];
#pragma unroll
      for (int s = 0; s < NB / 2; ++s)
#pragma unroll
        for (int rb = 2 * s; rb < NB; ++rb) y[rb] = mma(f[s], tr[rb][s], y[rb]);
      if constexpr (WHOLE) {
        const int st = (int)p.os[2] * (int)sizeof(T);
        const rsrc_t rs = make_rsrc_wave(o + (int64_t)t0 * p.os[2], ((int64_t)(cnt - 1) * p.os[2] + V - n0) * (int64_t)sizeof(T));
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
          const float e[4] = {y[rb][0], y[rb][1], y[rb][2], y[rb][3]};
          bstore_vals<T, 4>(rs, 4 * g < V - n0 ? (16 * rb + col) * st + 4 * g * (int)sizeof(T) : kOut, e);
        }
      } else {
#pragma unroll
        for (int rb = 0; rb < NB; ++rb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * rb + col < cnt && n0 + 4 * g + r < V) o[(int64_t)(t0 + 16 * rb + col) * p.os[2] + 4 * g + r] = (T)y[rb][r];
      }
    }
    // waited for where its loads were issued, in one iteration: stores since then need not have ended
    if (t0 + C < len) {
      if (!DIRECT) __syncthreads();  // this chunk has been read
      arrived(buf ^ DIRECT);
    }
  }
  if (unit) store_state<KP>(S, a.trans + (bh * a.nseg + seg) * KP * KP + nn - a.vp, KP, KP);
  if (!live) return;
  if (WHAT == kAcross) store_state<KP>(S, a.start + at0 + K * V, K, V);
  if (!OUT) return;
  if (p.s_out && (lo < whole ? whole <= lo + a.seg : seg == 0 && whole == 0)) store_state<KP>(S, p.s_out + sb, K, V);
  for (int64_t t = max(whole, lo) + g; t < min(p.T, (int64_t)lo + a.seg); t += 4) o[t * p.os[2] + col] = (T)0.f;
}

// The states' gradients from the last chunk on, and dv; ACROSS: only what each segment but the first makes of them from zero
// (from the state after it they come by the transpose of what the forward found).  As the forward's, with twice its products
// that the state waits for: 4.2 us a chunk at 128 x 128 in bf16, 267 us at B4 T4096 H16.
template <typename T, int NP, int KP, int MODE, bool ACROSS, int NW>
__global__ __launch_bounds__(NW * 64, (ACROSS || MODE == kDirect ? ChainSize<T, NP, KP, MODE>::WAVES : 1)) void dr_chain_bwd(Args a) {
  typedef ChainSize<T, NP, KP, MODE> Z;
  constexpr int NI = Z::NI, C = Z::C, NB = Z::NB, R = Z::R, PL = Z::PL, RC = Z::RC, PC = Z::PC;
  constexpr bool DIRECT = Z::DIRECT, WHOLE = MODE != kGather;
  extern __shared__ __align__(16) unsigned char chain_lds[];
  float (*lv)[4][C] = reinterpret_cast<float (*)[4][C]>(chain_lds);
  bf16 (*lk)[Z::KEYS] = reinterpret_cast<bf16 (*)[Z::KEYS]>(lv + Z::BUF);
  bf16 (*lt)[Z::SQUARE] = reinterpret_cast<bf16 (*)[Z::SQUARE]>(lk + Z::BUF);
  bf16 (*lq)[Z::KEYS] = reinterpret_cast<bf16 (*)[Z::KEYS]>(lt + Z::BUF);
  bf16 (*lp)[Z::SQUARE] = reinterpret_cast<bf16 (*)[Z::SQUARE]>(lq + Z::BUF);
  const DrProblem& p = a.p;
  const int nvb = a.vp / (NW * 16), nseg = ACROSS ? a.nseg - 1 : a.nseg;
  int64_t blk = a.blk0 + xcd_remap(blockIdx.x, a.nblk);
  const int vb = (int)(blk % nvb);
  blk /= nvb;
  const int seg = (int)(blk % nseg) + ACROSS;
  const int64_t bh = blk / nseg, b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
  const int lane = threadIdx.x % 64, g = lane / 16, col = lane % 16;
  const int n0 = vb * NW * 16 + wave_id() * 16, nn = n0 + col, K = (int)p.K, V = (int)p.V;
  const bool live = nn < V;
  const int lo = seg * a.seg, len = min(length_of(p, b), lo + a.seg), whole = length_of(p, b);
  const T* q = (const T*)p.q + b * p.qs[0] + hk * p.qs[1];
  const T* k = (const T*)p.k + b * p.ks[0] + hk * p.ks[1];
  const T* d_o = (const T*)p.d_o + b * p.dos[0] + h * p.dos[1] + nn;
  T* dv = (T*)p.dv + b * p.dvs[0] + h * p.dvs[1] + nn;
  const int64_t sb = bh * K * V + nn;
  f32x4 S[KP / 16];
  const int64_t at0 = (bh * a.nseg + seg) * K * V + nn;
  const float* from = seg == a.nseg - 1 ? (p.ds_in ? p.ds_in + sb : nullptr) : ACROSS ? nullptr : a.dstart + at0;
  load_state<KP>(S, from, live, K, V);
  Rows<T, C, KP, NW * 64, WHOLE> rk, rq;
  Square<NP, C, NW * 64> rt, rp;
  Columns<T, C, WHOLE> cd;
  Scales<C, NW * 64> vec;
  auto fetch = [&](int t0, int buf) {
    if (t0 < lo) return;
    const int cnt = min(C, len - t0);
    const int64_t ch = bh * a.n + t0 / C;
    const T *kt = k + (int64_t)t0 * p.ks[2], *qt = q + (int64_t)t0 * p.qs[2];
    const bf16 *tt = a.tt + ch * NP * C * C, *pt = a.pp + ch * NP * C * C;
    if constexpr (DIRECT) {
      load_direct<C, KP, NW>(kt, p.ks[2], cnt, lk[buf]);
      load_direct<NP * C, C, NW>(tt, C, NP * C, lt[buf]);
      load_direct<C, KP, NW>(qt, p.qs[2], cnt, lq[buf]);
      load_direct<NP * C, C, NW>(pt, C, NP * C, lp[buf]);
    } else {
      rk.load(kt, p.ks[2], K, cnt);
      rt.load(tt);
      rq.load(qt, p.qs[2], K, cnt);
      rp.load(pt);
    }
    cd.load(d_o + (int64_t)t0 * p.dos[2], p.dos[2], V - n0, cnt);
    vec.load(a.vec + ch * kVecs * C);
  };
  auto arrive = [&](int buf) {  // what fetch() left in registers
    if constexpr (!DIRECT) {
      rk.template store<R, PL, false>(lk[buf]);
      rt.store(lt[buf]);
      rq.template store<R, PL, false>(lq[buf]);
      rp.store(lp[buf]);
    }
    vec.store(lv[buf][0]);
  };
  const int first = (len + C - 1) / C * C - C;  // lo is whole chunks: below it where no token is
  fetch(first, 0);
  f32x4 x[NB];
  auto arrived = [&](int buf) {
    arrive(buf);
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) x[rb] = cd.get(rb);
  };
  arrived(0);
  int buf = 0;
  for (int t0 = first; t0 >= lo; t0 -= C, buf ^= DIRECT) {
    const int cnt = min(C, len - t0);
    const int64_t ch = bh * a.n + t0 / C;
    __syncthreads();  // this chunk is there (and the other buffer has been read)
    const Tile<NI, R, PL, DIRECT> tk{lk[buf]}, tq{lq[buf]};
    const Tile<NP, RC, PC, DIRECT> tt{lt[buf]}, tp{lp[buf]};
    const float (*sc)[C] = lv[buf];
    const float gc = expf(vec.top);
    fetch(t0 - C, buf ^ DIRECT);
    auto at = [&](int m, int row) { return *reinterpret_cast<const f32x4*>(&sc[m][row + 4 * g]); };
    constexpr int ST = Z::STEPS;
    Frag<NI> even[ST][NB], odd[ST][NB];
    auto rows = [&](Frag<NI> (&f)[ST][NB], int s) {
#pragma unroll
      for (int i = 0; i < ST; ++i)
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) f[i][rb] = tk.rows(16 * rb, s + i);
      phase();
    };
    rows(even, 0);
    Frag<NP> sf[KP / 32];
    Frag<NP> gd[C / 32], f[C / 32];
    Frag<NI> df[C / 32];
#pragma unroll
    for (int s = 0; s < KP / 32; ++s) sf[s] = pack<NP>(S[2 * s], S[2 * s + 1]);
    if constexpr (!ACROSS) keep_state<T, NP, KP>(a.ds, a.eds, ch, a.vp, n0, S, sf);
#pragma unroll
    for (int s = 0; s < C / 32; ++s) {
      df[s] = pack<NI>(x[2 * s], x[2 * s + 1]);
      gd[s] = pack<NP>(x[2 * s] * at(2, 32 * s), x[2 * s + 1] * at(2, 32 * s + 16));
    }
    // Y = P^T dO + b D k dS
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) x[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
    Frag<NP> tc[NB][NB / 2];
    auto square = [&](const Tile<NP, RC, PC, DIRECT>& t) {
#pragma unroll
      for (int rb = 0; rb < NB; ++rb)
#pragma unroll
        for (int s = rb / 2; s < NB / 2; ++s) tc[rb][s] = t.cols(rb, s);
      phase();
    };
#pragma unroll
    for (int s = 0; s < KP / 32; s += ST) {
      Frag<NI> (&now)[ST][NB] = s / ST % 2 ? odd : even, (&then)[ST][NB] = s / ST % 2 ? even : odd;
      if (s + ST < KP / 32) rows(then, s + ST);
      else square(tp);
#pragma unroll
      for (int i = 0; i < ST; ++i)
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) x[rb] = mma(now[i][rb], sf[s + i], x[rb]);
      phase();
    }
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) x[rb] *= at(1, 16 * rb);
#pragma unroll
    for (int s = 0; s < NB / 2; ++s)
#pragma unroll
      for (int rb = 0; rb < 2 * s + 2; ++rb) x[rb] = mma(tc[rb][s], df[s], x[rb]);
    phase();
    // dS <- G_C dS + q^T G dO - k^T G dX: its first part, beside dX = T^T Y
    square(tt);
    constexpr int KN = KP / 16, NK = KN * (C / 32);
    Frag<NI> kc[2][NK < 8 ? NK : 8];
    auto keys = [&](const Tile<NI, R, PL, DIRECT>& t, int e0) {
#pragma unroll
      for (int e = 0; e < 8 && e < NK; ++e) kc[e0 / 8 % 2][e] = t.cols((e0 + e) % KN, (e0 + e) / KN);
      phase();
    };
    keys(tq, 0);
#pragma unroll
    for (int s = 0; s < C / 32; ++s) f[s] = pack<NP>(x[2 * s], x[2 * s + 1]);
#pragma unroll
    for (int kb = 0; kb < KN; ++kb) S[kb] *= gc;
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) x[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NB / 2; ++s)
#pragma unroll
      for (int rb = 0; rb < 2 * s + 2; ++rb) x[rb] = mma(tc[rb][s], f[s], x[rb]);
    phase();
    constexpr int NBATCH = (NK + 7) / 8;
#pragma unroll
    for (int i = 0; i < 2 * NBATCH; ++i) {  // q's batches, then k's
      const int e0 = i % NBATCH * 8, slot = i % 2;
      auto load = [&](int j) {
#pragma unroll
        for (int e = 0; e < 8 && e < NK; ++e)
          kc[j % 2][e] = (j < NBATCH ? tq : tk).cols((j % NBATCH * 8 + e) % KN, (j % NBATCH * 8 + e) / KN);
        phase();
      };
      if (i + 1 < 2 * NBATCH) load(i + 1);
#pragma unroll
      for (int e = 0; e < 8 && e < NK; ++e) {
        const int kb = (e0 + e) % KN, s = (e0 + e) / KN;
        S[kb] = mma(kc[slot][e], i < NBATCH ? gd[s] : f[s], S[kb]);
      }
      if (i == 0) {
#pragma unroll
        for (int rb = 0; rb < NB; ++rb)
          if (!ACROSS) put_columns<T, WHOLE>(dv + (int64_t)t0 * p.dvs[2], p.dvs[2], V - n0, cnt, 16 * rb, x[rb]);
#pragma unroll
        for (int s = 0; s < C / 32; ++s) {
          if (!ACROSS && !kHalves<T, NP>) keep<NP, false>(a.x + (ch * NP * C + 32 * s) * a.vp + n0, a.vp, (int64_t)C * a.vp, pack<NP>(x[2 * s], x[2 * s + 1]));
          f[s] = pack<NP>(-x[2 * s] * at(0, 32 * s), -x[2 * s + 1] * at(0, 32 * s + 16));
        }
      }
      phase();
    }
    if (t0 >= lo + C) {  // as in the forward
      if (!DIRECT) __syncthreads();
      arrived(buf ^ DIRECT);
    }
  }
  if (!live) return;
  if (ACROSS) return store_state<KP>(S, a.dstart + at0 - K * V, K, V);
  if (p.ds_out && seg == 0) store_state<KP>(S, p.ds_out + sb, K, V);
  for (int64_t t = max(whole, lo) + g; t < min(p.T, (int64_t)lo + a.seg); t += 4) dv[t * p.dvs[2]] = (T)0.f;
}

// From segment to segment, a workgroup to 16 columns of a head and a quarter of the rows to a wavefront:
// start[s + 1] += trans[s] start[s], or with gradients dstart[s - 1] += trans[s]^T dstart[s], on float32 matrix instructions
// (16x16x4).  A step waits for the one before, so what it reads of the transitions is on its way by then, up to 128 channels
// (one wavefront to the columns, which read as it went, took 9 us a segment at 128 channels and 45 at 256).
template <int KP, bool BWD>
__global__ __launch_bounds__(256) void dr_across(Args a) {
  constexpr int RB = KP / 64, KB = KP / 16;
  __shared__ __align__(16) float lds[2][16][KP + 4];  // states, by column
  const DrProblem& p = a.p;
  const int nvb = a.vp / 16, K = (int)p.K, V = (int)p.V, lane = threadIdx.x % 64, g = lane / 16, col = lane % 16, wv = wave_id();
  const int64_t blk = a.blk0 + blockIdx.x, bh = blk / nvb;
  const int nn = (int)(blk % nvb) * 16 + col;
  float* st = (BWD ? a.dstart : a.start) + bh * a.nseg * K * V + nn;
  const int64_t kv = (int64_t)K * V;
  auto load = [&](f32x4 (&S)[RB], const float* from) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * (wv * RB + i) + 4 * g + r;
        S[i][r] = nn < V && d < K ? from[d * V] : 0.f;
      }
  };
  auto share = [&](int buf, const f32x4 (&S)[RB]) {
#pragma unroll
    for (int i = 0; i < RB; ++i) *reinterpret_cast<f32x4*>(&lds[buf][col][16 * (wv * RB + i) + 4 * g]) = S[i];
  };
  auto segment = [&](int i) { return BWD ? a.nseg - 1 - i : i; };
  auto row = [&](f32x4 (&m)[KB], int i, int rb) {  // a block of rows of the transition of step i
    const float* M = a.trans + (bh * a.nseg + segment(i)) * KP * KP;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      if constexpr (BWD) {
#pragma unroll
        for (int r = 0; r < 4; ++r) m[kb][r] = M[(16 * kb + 4 * g + r) * KP + 16 * rb + col];
      } else {
        m[kb] = *reinterpret_cast<const f32x4*>(M + (16 * rb + col) * KP + 16 * kb + 4 * g);
      }
    }
  };
  constexpr bool AHEAD = KP <= 128;
  f32x4 S[RB], N[RB], m[AHEAD ? RB : 1][KB];
  load(S, st + segment(1) * kv);
  share(1, S);
  if (AHEAD)
#pragma unroll
    for (int i = 0; i < RB; ++i) row(m[AHEAD ? i : 0], 1, wv * RB + i);
  for (int i = 1; i < a.nseg - 1; ++i) {
    float* to = st + (segment(i) + (BWD ? -1 : 1)) * kv;
    load(N, to);
    __syncthreads();
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      f32x4 (&mr)[KB] = m[AHEAD ? rb : 0];
      if (!AHEAD) row(mr, i, wv * RB + rb);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(&lds[i % 2][col][16 * kb + 4 * g]);
#pragma unroll
        for (int r = 0; r < 4; ++r) N[rb] = __builtin_amdgcn_mfma_f32_16x16x4f32(mr[kb][r], s[r], N[rb], 0, 0, 0);
      }
      if (AHEAD && i + 1 < a.nseg - 1) row(mr, i + 1, wv * RB + rb);
    }
    share((i + 1) % 2, N);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * (wv * RB + rb) + 4 * g + r;
        if (nn < V && d < K) to[d * V] = N[rb][r];
      }
  }
}

// Gradients of q, k and the gates, chunk by chunk: the value heads of one key head to a workgroup, a quarter of the
// channels to a wavefront.  With the rows' norms in E's place (rq_i rk_j for P, rk_i rk_j for N) the sums are those of q and
// k themselves, before their part along the row is taken out.  Results lie turned over, four neighbouring channels of a
// token in a lane: sums over a row are of a lane's own and three others', and a store has 8 bytes.  ONE: one value head to a
// key head, whose sums need no registers of their own.  The memory path bounds it, and the halves' way into parts: B4 T4096
// H16 hd128 bf16 212 us for 0.74 GB, of which the states and their gradients are 0.27 (3.5 TB/s; 177 from one part of each, which
// needs no way); with two value heads to a key head, whose sums leave one workgroup to a CU for two, 566 us for B2 T8192 H32
// (1.3 GB, 2.3 TB/s).
template <typename T, int NP, int KP, bool WHOLE, bool ONE>
__global__ __launch_bounds__(256, ONE && KP <= 128 && parts_of<T>() == 1 ? 2 : 1) void dr_grads(Args a) {
  constexpr int NI = parts_of<T>(), C = chunk_of(NP, KP), NB = C / 16, R = KP + 8, PL = C * R, RC = C + 8, PC = C * RC;
  constexpr bool HALF = kHalves<T, NP>;
  // columns of v at once: 64 where LDS then has room for two workgroups and registers have too
  constexpr int PIECE = HALF && ONE && KP <= 128 ? 64 : 128, NX = HALF ? 1 : NP, ND = planes(HALF, NP);
  constexpr int NCB = KP / 64, RV = PIECE + 8, PV = C * RV, NU = NB * NB / 4;
  constexpr int ROWS = (NI + NP + NX) * PV, KEYS = 2 * NI * PL;
  __shared__ __align__(16) bf16 mem[ROWS > KEYS ? ROWS : KEYS], lm[2 * NP * PC];
  __shared__ __align__(16) float lv[kVecs][C];
  __shared__ float diag[C], red[3][4][C], total[4], along[2][C];
  __shared__ __align__(16) float powers[2][4][HALF ? PIECE : 4];  // of the states' and their gradients' lanes
  const Tile<NI, RV, PV> to{mem};
  const Tile<NP, RV, PV> tz{mem + NI * PV};
  const Tile<NX, RV, PV> tx{mem + (NI + NP) * PV};
  const Tile<NI, R, PL> tk{mem}, tq{mem + NI * PL};
  const Tile<NP, RC, PC> pe{lm}, ne{lm + NP * PC};  // row j, column i
  const DrProblem& p = a.p;
  const int64_t blk = a.blk0 + blockIdx.x, n = blk % a.n, bhk = blk / a.n, b = bhk / p.Hk, hk = bhk % p.Hk;
  const int t0 = (int)n * C, len = length_of(p, b), cnt = min(C, max(len - t0, 0)), rows = min(C, (int)p.T - t0), t = threadIdx.x;
  const int K = (int)p.K, V = (int)p.V, group = ONE ? 1 : (int)(p.H / p.Hk), lane = t % 64, g = lane / 16, col = lane % 16;
  const int wv = wave_id();
  T* dq_ = (T*)p.dq + b * p.dqs[0] + hk * p.dqs[1] + (int64_t)t0 * p.dqs[2];
  T* dk_ = (T*)p.dk + b * p.dks[0] + hk * p.dks[1] + (int64_t)t0 * p.dks[2];
  f32x4 sq[NB][NCB], sk[NB][NCB];
#pragma unroll
  for (int rb = 0; rb < NB; ++rb)
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) sq[rb][cb] = sk[rb][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (t < C) along[0][t] = along[1][t] = 0.f;
  if (cnt == 0) {  // no token of the sequence: zeros
    for (int hd = 0; hd < group; ++hd)
      if (t < rows) {
        const int64_t h = hk * group + hd;
        put_gate(p.dg, p.gdtype, b * p.dgs[0] + h * p.dgs[1] + (t0 + t) * p.dgs[2], 0.f);
        put_gate(p.db, p.gdtype, b * p.dbs[0] + h * p.dbs[1] + (t0 + t) * p.dbs[2], 0.f);
      }
    for (int e = t; e < rows * K; e += 256) {
      dq_[(int64_t)(e / K) * p.dqs[2] + e % K] = (T)0.f;
      dk_[(int64_t)(e / K) * p.dks[2] + e % K] = (T)0.f;
    }
    return;
  }
  for (int hd = 0; hd < group; ++hd) {
    const int64_t h = hk * group + hd, bh = b * p.H + h, ch = bh * a.n + n;
    const T* d_o = (const T*)p.d_o + b * p.dos[0] + h * p.dos[1] + (int64_t)t0 * p.dos[2];
    const T* dv = (const T*)p.dv + b * p.dvs[0] + h * p.dvs[1] + (int64_t)t0 * p.dvs[2];
    if (hd > 0) __syncthreads();  // the head before has been read
    f32x4 dq[NB][NCB], dr[NB][NCB], dw[NB][NCB];
#pragma unroll
    for (int rb = 0; rb < NB; ++rb)
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) dq[rb][cb] = dr[rb][cb] = dw[rb][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
    // dO Z^T and dX Z^T: a block of rows (i) to a wavefront and all blocks of columns (j), those above the diagonal too,
    // which cost less than the branches that would leave them out; with two blocks of rows one block to a wavefront
    const int rbu = NB == 4 ? wv : wv % 2;
    f32x4 accp[NU], accn[NU];
#pragma unroll
    for (int i = 0; i < NU; ++i) accp[i] = accn[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float dot = 0.f;
    for (int v0 = 0; v0 < a.vp; v0 += PIECE) {
      const int width = min(PIECE, a.vp - v0);
      if (v0 > 0) __syncthreads();
      Frag<ND> fs[2][NCB], fd[2][NCB];  // the states of a step and the next, as they lie in memory
      auto states = [&](int s) {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
          const int64_t at = ch * ND * KP * a.vp + (int64_t)(wv * NCB * 16 + 16 * cb + col) * a.vp + v0 + 32 * s + 8 * g;
#pragma unroll
          for (int i = 0; i < ND; ++i) {
            fs[s % 2][cb].p[i] = *reinterpret_cast<const u32x4*>(a.s + at + (int64_t)i * KP * a.vp);
            fd[s % 2][cb].p[i] = *reinterpret_cast<const u32x4*>(a.ds + at + (int64_t)i * KP * a.vp);
          }
        }
      };
      {
        Rows<T, C, PIECE, 256, WHOLE> ro, rv;
        Rows<bf16, C, PIECE, 256, true> rz[HALF ? 1 : 2 * NP];
        ro.load(d_o + v0, p.dos[2], V - v0, cnt);
        if constexpr (HALF) rv.load(dv + v0, p.dvs[2], V - v0, cnt);
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          rz[i].load(a.z + (ch * ND + i) * C * a.vp + v0, a.vp, width, C);
          if constexpr (!HALF) rz[NP + i].load(a.x + (ch * NP + i) * C * a.vp + v0, a.vp, width, C);
        }
        u32x2 ez = {0, 0};
        uint32_t ep[HALF ? 2 * PIECE / 64 : 1];
        if constexpr (HALF) {  // exponents: Z's of this thread's columns (its rows are of one lane's kind), the states' shared
          const int c0 = t % (PIECE / 8) * 8, kind = t / (PIECE / 8) % 16 / 4;
          static_assert(256 / (PIECE / 8) % 16 == 0, "a thread's rows");
          if (c0 < width) ez = *reinterpret_cast<const u32x2*>(a.ez + (ch * 4 + kind) * a.vp + v0 + c0);
#pragma unroll
          for (int i = 0; i < 2 * PIECE / 64; ++i) {
            const int e = i * 256 + t, c = e % PIECE, m = e / PIECE;
            ep[i] = c < width ? (m < 4 ? a.es : a.eds)[(ch * 4 + m % 4) * a.vp + v0 + c] : 0;
          }
        }
        float vec[(kVecs * C + 255) / 256];
        if (v0 == 0)
#pragma unroll
          for (int i = 0; i * 256 < kVecs * C; ++i) vec[i] = a.vec[ch * kVecs * C + i * 256 + t];
        states(0);
        ro.template store<RV, PV, false>(mem);
        if constexpr (HALF) {
          rv.template store<RV, PV, false>(mem + (NI + NP) * PV);
          const f32x4 by[2] = {{power(ez[0] & 0xFF), power(ez[0] >> 8 & 0xFF), power(ez[0] >> 16 & 0xFF), power(ez[0] >> 24)},
                               {power(ez[1] & 0xFF), power(ez[1] >> 8 & 0xFF), power(ez[1] >> 16 & 0xFF), power(ez[1] >> 24)}};
          store_halves<RV, PV>(rz[0], by, mem + NI * PV);
#pragma unroll
          for (int i = 0; i < 2 * PIECE / 64; ++i) (&powers[0][0][0])[i * 256 + t] = power(ep[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 2 * NP; ++i) rz[i].template store<RV, PV, false>(mem + (NI + i) * PV);
        }
        if (v0 == 0)
#pragma unroll
          for (int i = 0; i * 256 < kVecs * C; ++i) lv[0][i * 256 + t] = vec[i];
      }
      __syncthreads();
#pragma unroll
      for (int s = 0; s < PIECE / 32; ++s) {
        if (s * 32 >= width) break;
        if ((s + 1) * 32 < width) states(s + 1);
        Frag<NP> gs[NCB], gd[NCB];
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
          if constexpr (HALF) {
            auto by = [&](int m) { return &powers[m][((wv * NCB + cb) % 2 * 16 + col) / 8][32 * s + 8 * g]; };  // of this channel's lanes
            float x[8], y[8];
            f32x4 w[2];
            __builtin_memcpy(w, __builtin_assume_aligned(by(0), 16), 32);
            gs[cb] = halves(fs[s % 2][cb].p[0], w, x);
            __builtin_memcpy(w, __builtin_assume_aligned(by(1), 16), 32);
            gd[cb] = halves(fd[s % 2][cb].p[0], w, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) dot += x[e] * y[e];
          } else {
            gs[cb] = fs[s % 2][cb];
            gd[cb] = fd[s % 2][cb];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x[2] = {0.f, 0.f}, y[2] = {0.f, 0.f};
#pragma unroll
              for (int i = NP - 1; i >= 0; --i) {
                x[0] += __uint_as_float(gs[cb].p[i][e] << 16);
                x[1] += __uint_as_float(gs[cb].p[i][e] & 0xFFFF0000u);
                y[0] += __uint_as_float(gd[cb].p[i][e] << 16);
                y[1] += __uint_as_float(gd[cb].p[i][e] & 0xFFFF0000u);
              }
              dot += x[0] * y[0] + x[1] * y[1];
            }
          }
        }
        const Frag<NI> uo = to.rows(16 * rbu, s);
        const Frag<NX> ux = tx.rows(16 * rbu, s);
        if constexpr (NB == 2) {
          const Frag<NP> uz = tz.rows(16 * (wv / 2), s);
          accp[0] = mma(uo, uz, accp[0]);
          accn[0] = mma(ux, uz, accn[0]);
        }
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
          const Frag<NI> ro = to.rows(16 * rb, s);
          const Frag<NX> rx = tx.rows(16 * rb, s);
          const Frag<NP> rz = tz.rows(16 * rb, s);
          if constexpr (NB == 4) {
            accp[rb] = mma(uo, rz, accp[rb]);
            accn[rb] = mma(ux, rz, accn[rb]);
          }
#pragma unroll
          for (int cb = 0; cb < NCB; ++cb) {
            dq[rb][cb] = mma(gs[cb], ro, dq[rb][cb]);
            dr[rb][cb] = mma(gs[cb], rx, dr[rb][cb]);
            dw[rb][cb] = mma(gd[cb], rz, dw[rb][cb]);
          }
        }
      }
    }
    Rows<T, C, KP, 256, WHOLE> rk, rq;
    rk.load((const T*)p.k + b * p.ks[0] + hk * p.ks[1] + (int64_t)t0 * p.ks[2], p.ks[2], K, cnt);
    rq.load((const T*)p.q + b * p.qs[0] + hk * p.qs[1] + (int64_t)t0 * p.qs[2], p.qs[2], K, cnt);
    // the pairs' gradients with their decays, strengths and norms, as operands
    {
      auto at = [&](int m) { return *reinterpret_cast<const f32x4*>(&lv[m][16 * rbu + 4 * g]); };
      const f32x4 hi = at(0), lo = at(1), ki = at(kRk), qi = at(kRq) * p.scale;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const int cb = NB == 4 ? i : wv / 2, j = 16 * cb + col;
        const float hj = lv[0][j], lj = lv[1][j], kj = lv[kRk][j] * lv[kB][j];
        f32x4 vp, vn;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int x = 16 * rbu + 4 * g + r;
          // e^(c_i - c_j) by the instruction (one last place); above the diagonal the difference is not negative, and unused
          const float E = kj * __builtin_amdgcn_exp2f(((hi[r] - hj) + (lo[r] - lj)) * 1.44269504088896f);
          vp[r] = j <= x ? qi[r] * E * accp[i][r] : 0.f;
          vn[r] = j < x ? -ki[r] * E * accn[i][r] : 0.f;
          if (!HALF && x == j) diag[x] = accn[i][r];
        }
        const int where = j * RC + spot(16 * rbu + 4 * g);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          uint32_t w0[NP], w1[NP];
          split<NP>(m ? vn[0] : vp[0], m ? vn[1] : vp[1], w0);
          split<NP>(m ? vn[2] : vp[2], m ? vn[3] : vp[3], w1);
#pragma unroll
          for (int l = 0; l < NP; ++l) *reinterpret_cast<u32x2*>(lm + (m * NP + l) * PC + where) = u32x2{w0[l], w1[l]};
        }
      }
    }
    __syncthreads();  // the rows have been read, the pairs are there
    rk.template store<R, PL, true>(mem);
    rq.template store<R, PL, true>(mem + NI * PL);
    __syncthreads();
    float kept = expf(lv[0][C - 1]) * dot, sums[3][NB];
    Frag<NI> fk[NCB][C / 32], fq[NCB][C / 32];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
      for (int s = 0; s < C / 32; ++s) {
        fk[cb][s] = tk.cols(wv * NCB + cb, s);
        fq[cb][s] = tq.cols(wv * NCB + cb, s);
      }
#pragma unroll
    for (int rb = 0; rb < NB; ++rb) {
      const int i = 16 * rb + col;
      const float gq = lv[kGq][i], gk = -lv[kGk][i], dk = lv[kDk][i];
      sums[0][rb] = sums[1][rb] = sums[2][rb] = 0.f;
      f32x4 kv[NCB], qv[NCB];
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        kv[cb] = tk.four(i, 16 * (wv * NCB + cb) + 4 * g);
        qv[cb] = tq.four(i, 16 * (wv * NCB + cb) + 4 * g);
        dq[rb][cb] *= gq;
        dr[rb][cb] *= gk;
        dw[rb][cb] *= dk;
#pragma unroll
        for (int r = 0; r < 4; ++r) kept += kv[cb][r] * dw[rb][cb][r];
      }
#pragma unroll
      for (int s = 0; s < C / 32; ++s) {
        if (s <= rb / 2) {
          const Frag<NP> fp = pe.cols(rb, s), fn = ne.cols(rb, s);
#pragma unroll
          for (int cb = 0; cb < NCB; ++cb) {
            dq[rb][cb] = mma(fk[cb][s], fp, dq[rb][cb]);
            dr[rb][cb] = mma(fk[cb][s], fn, dr[rb][cb]);
          }
        }
        if (s >= rb / 2) {
          const Frag<NP> fp = pe.rows(16 * rb, s), fn = ne.rows(16 * rb, s);
#pragma unroll
          for (int cb = 0; cb < NCB; ++cb) {
            dw[rb][cb] = mma(fq[cb][s], fp, dw[rb][cb]);
            dw[rb][cb] = mma(fk[cb][s], fn, dw[rb][cb]);
          }
        }
      }
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sums[0][rb] += qv[cb][r] * dq[rb][cb][r];
          sums[1][rb] += kv[cb][r] * dr[rb][cb][r];
          sums[2][rb] += kv[cb][r] * dw[rb][cb][r];
        }
        sq[rb][cb] += dq[rb][cb];
        sk[rb][cb] += dr[rb][cb] + dw[rb][cb];
      }
    }
#pragma unroll
    for (int m = 0; m < 3; ++m)
#pragma unroll
      for (int rb = 0; rb < NB; ++rb) {
        float s = sums[m][rb];
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (g == 0) red[m][wv][16 * rb + col] = s;
      }
#pragma unroll
    for (int i = 1; i < 64; i *= 2) kept += __shfl_xor(kept, i);
    if (lane == 0) total[wv] = kept;
    __syncthreads();
    if (wv == 0) {
      const int i = lane < C ? lane : 0;
      float s[3];
#pragma unroll
      for (int j = 0; j < 3; ++j) s[j] = (red[j][0][i] + red[j][1][i]) + (red[j][2][i] + red[j][3][i]);
      if (lane < C) {
        along[0][i] += s[0];
        along[1][i] += s[1] + s[2];
      }
      float c = lane < C ? s[0] + (s[1] - s[2]) : 0.f;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {  // sums over the tokens from this one on
        const float o = __shfl_down(c, d);
        if (lane + d < 64) c += o;
      }
      if (lane < rows) {
        const bool in = lane < cnt;
        c += (total[0] + total[1]) + (total[2] + total[3]);
        const float be = lv[kB][i];
        put_gate(p.dg, p.gdtype, b * p.dgs[0] + h * p.dgs[1] + (t0 + lane) * p.dgs[2], in ? c : 0.f);
        put_gate(p.db, p.gdtype, b * p.dbs[0] + h * p.dbs[1] + (t0 + lane) * p.dbs[2], in ? (HALF ? s[2] : diag[i]) / be : 0.f);
      }
    }
  }
  __syncthreads();
  auto out = [&](T* base, int64_t stride, int i, int c, f32x4 v) {  // rows from cnt on are zero
    if constexpr (WHOLE) {
      const rsrc_t rs = make_rsrc_wave(base, ((int64_t)(rows - 1) * stride + K) * (int64_t)sizeof(T));
      const float e[4] = {v[0], v[1], v[2], v[3]};
      bstore_vals<T, 4>(rs, c < K ? i * (int)stride * (int)sizeof(T) + c * (int)sizeof(T) : kOut, e);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (i < rows && c + r < K) base[(int64_t)i * stride + c + r] = (T)v[r];
    }
  };
#pragma unroll
  for (int rb = 0; rb < NB; ++rb) {
    const int i = 16 * rb + col;
    const float rki = lv[kRk][i], rqi = lv[kRq][i];
    const float ak = p.normalize ? rki * rki * along[1][i] : 0.f, aq = p.normalize ? rqi * rqi * along[0][i] : 0.f;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      const int c = 16 * (wv * NCB + cb) + 4 * g;
      const f32x4 x = sq[rb][cb] - tq.four(i, c) * aq, y = sk[rb][cb] - tk.four(i, c) * ak, zero = {0.f, 0.f, 0.f, 0.f};
      out(dq_, p.dqs[2], i, c, i < cnt ? x : zero);
      out(dk_, p.dks[2], i, c, i < cnt ? y : zero);
    }
  }
}

// The launches of a type and a number of parts (instantiated in delta_<type>.hip).
enum Stage { kPrep, kAhead, kCarry, kChain, kChainKeep, kKeepStates, kAheadBwd, kCarryBwd, kChainBwd, kGrads };
template <typename T, int NP>
hipError_t launch(Stage st, const Args& a, int mode, hipStream_t stream) {
  auto run = [&](auto kernel, int threads, int lds) {
    kernel<<<(unsigned)a.nblk, threads, lds, stream>>>(a);
    return hipGetLastError();
  };
  auto chain = [&](auto kp, auto m, auto w) {
    constexpr int KP = decltype(kp)::value, M = decltype(m)::value, NW = decltype(w)::value;
    typedef ChainSize<T, NP, KP, M> Z;
    switch (st) {
      case kAhead: return run(dr_chain<T, NP, KP, M, kAcross, NW>, NW * 64, Z::bytes(false));
      case kChain: return run(dr_chain<T, NP, KP, M, kOutputs, NW>, NW * 64, Z::bytes(true));
      case kChainKeep: return run(dr_chain<T, NP, KP, M, kBoth, NW>, NW * 64, Z::bytes(true));
      case kKeepStates: return run(dr_chain<T, NP, KP, M, kKeep, NW>, NW * 64, Z::bytes(false));
      case kAheadBwd: return run(dr_chain_bwd<T, NP, KP, M, true, NW>, NW * 64, Z::bytes(true));
      default: return run(dr_chain_bwd<T, NP, KP, M, false, NW>, NW * 64, Z::bytes(true));
    }
  };
  constexpr std::integral_constant<int, 2> two;
  constexpr std::integral_constant<int, 4> four;
  auto pick = [&](auto kp, auto w) {
    constexpr int KP = decltype(kp)::value;
    constexpr bool W = decltype(w)::value;
    if (st == kPrep) return run(dr_prep<T, NP, KP, W>, 256, 0);
    if (st == kCarry) return run(dr_across<KP, false>, 256, 0);
    if (st == kCarryBwd) return run(dr_across<KP, true>, 256, 0);
    if (st == kGrads)
      return a.p.H == a.p.Hk ? run(dr_grads<T, NP, KP, W, true>, 256, 0) : run(dr_grads<T, NP, KP, W, false>, 256, 0);
    if constexpr (W && kHasDirect<T, NP, KP>)
      if (mode == kDirect && a.p.K == KP &&
          !(kShares<T, NP, KP> && st != kChainBwd && a.blocks > (st == kChain || st == kChainKeep ? 512 : 256))) {
        if constexpr (kHasFour<T, NP, KP>)
          if (a.nw == 4) return chain(kp, std::integral_constant<int, kDirect>(), four);
        return chain(kp, std::integral_constant<int, kDirect>(), two);
      }
    if constexpr (kHasFour<T, NP, KP>)
      if (a.nw == 4) return chain(kp, std::integral_constant<int, W ? kWhole : kGather>(), four);
    return chain(kp, std::integral_constant<int, W ? kWhole : kGather>(), two);
  };
  auto size = [&](auto w) {
    switch (cover((int)a.p.K)) {
      case 64: return pick(std::integral_constant<int, 64>(), w);
      case 128: return pick(std::integral_constant<int, 128>(), w);
      default: return pick(std::integral_constant<int, 256>(), w);
    }
  };
  return mode != kGather ? size(std::true_type()) : size(std::false_type());
}
extern template hipError_t launch<bf16, 2>(Stage, const Args&, int, hipStream_t);
extern template hipError_t launch<bf16, 3>(Stage, const Args&, int, hipStream_t);
extern template hipError_t launch<fp16, 2>(Stage, const Args&, int, hipStream_t);
extern template hipError_t launch<fp16, 3>(Stage, const Args&, int, hipStream_t);
extern template hipError_t launch<float, 3>(Stage, const Args&, int, hipStream_t);

}  // namespace dr
}  // namespace dc
