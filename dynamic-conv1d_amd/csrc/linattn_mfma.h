// Linear attention with a decay for each head, in chunks of tokens on matrix
// cores (include/dynconv_layer.h).  One pass (LaPass) is, for each head,
//
//   S_t = g S_{t-1} + skv k_t^T v_t,    o_t = so q_t S_t
//
// and over a chunk of C tokens with the state S before it, i, j = 0 .. C-1:
//
//   o_i = so ( g^{i+1} q_i S + sum_{j<=i} g^{i-j} (q_i . k_j) skv v_j )
//   S  <- g^C S + sum_j k_j^T (skv g^{C-1-j} v_j)
//
// A chunk that is not full holds its tokens in its last rows, behind rows of zeros,
// so that the weights of k^T v are those of every chunk.
//
// Four matrix products: scores, scores * v, q * S, k^T * v.  The forward is one
// pass; dq, dk and dv are passes on other tensors (linattn.hip), those of dk and
// dv against time, where the tokens are loaded in turned order and all else is
// alike.  The state that enters a pass against time (the gradient of the final
// state) meets its first token without a decay.
//
// Layout.  A workgroup takes one segment of one head's tokens, chunk after
// chunk, and NW * 32 columns of v; a wavefront keeps its 32 columns of S in
// float32 accumulators for the whole segment.  v_mfma_f32_32x32x16 leaves
// element (row, col) of its result in lane col + 32 ((row/4) % 2), register
// row%4 + 4 (row/8); an operand wants 8 values of the summed index in a lane.
// Every product here sums in the order that results come in (step s: 16 s +
// 8 (e/4) + 4 half + e%4 for element e), so scores and S go from results to
// operands without leaving their lane: scores are formed as k q^T (column i in
// lane i), S as k^T v (column n in lane n), o as (v^T scores^T + S^T q^T), whose
// column i sits in lane i with four neighbouring channels to a store.  The blocks
// of scores go round the wavefronts, through LDS, lane by lane as they are.  q and k
// rows lie in LDS so that a lane's 8 values of that order are neighbours (16-byte
// reads; two 8-byte reads took twice the LDS's time), v and k columns are read
// through transposing reads.
//
// Precision.  Scores and S are rounded to the inputs' type as operands (relative
// 2^-8 / 2^-11 of single terms, below the rounding of o); the products that make
// S take v g^{C-1-j} in two parts of the type (16 or 22 bits), bf16 in three where
// the state is returned, which so is a float32 result.  fp16 operands are lifted to
// the upper end of the type by powers of two that the float32 sums leave again:
// each token's scores and each column's v g^{C-1-j} by its own, the 32 columns of S
// of a wavefront by one (what is below 2^-28 of their largest value loses digits in
// q S, not in S).  float32 inputs are products of three bf16 parts throughout (Parts).
// All sums and S are float32.
//
// Measured at B2 H32 T8192, 128 x 128, bf16 (134 MB a tensor), four segments: the states' launch 63 us (3.2 TB/s of the
// k and v of three segments), the carry 8, the forward's chunks 133 (0.55 GB past the L2, 4.2 TB/s), the backward's three
// passes 308 (1.40 GB, 4.5 TB/s), with the backward's own states 590 in all.  The backward is near the rate of the memory
// path for what it moves: dk's and dv's passes walk a segment side by side and share their loads, dq's walks it the other
// way round and meets them in the middle only, so seven tensors are read past the L2 where four exist.  Loads alone take
// 42, 73 and 163, stores 20 and 60-78 more.  Matrix instructions fill 22% of the SIMDs' cycles in the forward's chunks and
// 31% in the backward's, vector instructions 28% and 38%.  In fp16 the lifts take 5-6% (B1 H16 T32768: chunks 146 ->
// 153 us, states 68 -> 74).
//
// An infinity or a NaN stays out of the tokens before its own, also within a chunk: scores of later tokens are selected
// away, not multiplied by zero, and v's elements that are not finite are taken out of the products of the diagonal blocks
// and added token by token (a branch that finite values do not take).
#pragma once

#include <type_traits>

#include "lowrank_mfma.h"
#include "layer_launch.h"

namespace dc {
namespace la {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// Kernel arguments: the problem, segments of seg tokens (a multiple of the
// chunk), and the states before each segment, [B * H][nseg][K * V] per set.
struct Args {
  LaProblem p;
  int npass, seg, nseg, nvb, nkb;
  int blk0, nblk;  // workgroups of this launch, of all
  bool returned;  // a state formed by this launch is the caller's result
  // what a pass starts its segments from / a state pass writes: one set of states (null: one segment, s_in / s_out)
  float* states[kLaMaxPasses];
};

// Tokens of a chunk: 64, or 32 in float32, whose tiles are three planes (64 would pass the LDS).
__host__ __device__ constexpr int chunk_tokens(int es) { return es == 4 ? 32 : 64; }

// Rows of a state that a workgroup forms in the states' launch: 64, so that three workgroups fit a CU whatever K is.
constexpr int kStateRows = 64;

// Where channel c of a row of q or k lies in LDS: of each 16 channels the second and third quads change places, so that
// the 8 channels of a lane's half, 4 half .. + 3 and 8 + 4 half .. + 3, are neighbours.
__host__ __device__ constexpr int quad(int c) { return (c & ~12) | ((c & 4) << 1) | ((c & 8) >> 1); }

template <typename T> struct Ops {  // 16-bit types
  typedef u32x4 Frag;
  typedef T Lds;  // elements of the tiles in LDS, in one plane
  static constexpr int kPlanes = 1;
  static constexpr bool kSplit = true, kNarrow = __is_same(T, fp16);  // two parts; float32 values may not fit
  __device__ static __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    if constexpr (__is_same(T, bf16))
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  }
  // this lane's half of 16 channels of a row: p points at the first of them
  __device__ static __forceinline__ Frag rows(const T* p, int half, int = 0) { return *reinterpret_cast<const Frag*>(p + 8 * half); }
  // column lane%32 of 16 rows: p points at (row 0, column 0) of the 16 x 32 block, rows rs elements apart; TURNED: the
  // rows' channels lie in quad() order
  template <bool TURNED>
  __device__ static __forceinline__ Frag cols(const T* p, int rs, int lane, int = 0) {
    const int c = 4 * (lane % 4);
    const T* q = p + (4 * (lane / 32) + (lane % 16) / 4) * rs + 16 * ((lane / 16) % 2) + (TURNED ? quad(c) : c);
    const u32x2 a = lds_read_tr16(q), b = lds_read_tr16(q + 8 * rs);
    return Frag{a[0], a[1], b[0], b[1]};
  }
  __device__ static __forceinline__ Frag pack(const float* v) {
    return Frag{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])};
  }
  __device__ static __forceinline__ void unpack(Frag f, float* v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = Mma16<T>::to_f(elem16(f, e));
  }
  // sign bits of the halves of a word that are infinite or NaN, and others that mean nothing
  __device__ static __forceinline__ uint32_t odd_bits(uint32_t w) {
    return __is_same(T, bf16) ? (w & 0x7F807F80u) + 0x00800080u : (w & 0x7C007C00u) + 0x04000400u;
  }
  __device__ static __forceinline__ bool odd(Frag f) {
    return (odd_bits(f[0]) | odd_bits(f[1]) | odd_bits(f[2]) | odd_bits(f[3])) & 0x80008000u;
  }
  __device__ static __forceinline__ Frag keep_finite(Frag f, Frag by) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] &= ~(((odd_bits(by[i]) & 0x80008000u) >> 15) * 0xFFFFu);
    return f;
  }
  __device__ static __forceinline__ Frag finite(Frag f) { return keep_finite(f, f); }
  // a lane's operand in LDS, 64 lanes to a plane
  __device__ static __forceinline__ void put(u32x4* p, int lane, Frag f) { p[lane] = f; }
  __device__ static __forceinline__ Frag get(const u32x4* p, int lane) { return p[lane]; }
};

// float32 as a sum of three bf16 (8 bits each: all 24 of them, over bf16's range, which is float32's).  A product is the
// six products of parts down to 2^-16 of it, so it is as good as float32's own, at 6 matrix instructions of 32 cycles for 8
// of 64 (v_mfma_f32_32x32x2): float32 training of B3 T1537 H10 hd100 went from 315 to 260 us.
struct Parts {
  struct Frag { u32x4 p[3]; };
  typedef bf16 Lds;
  static constexpr int kPlanes = 3;
  static constexpr bool kSplit = false, kNarrow = false;
  __device__ static __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
    typedef Ops<bf16> O;
    c = O::mma(a.p[2], b.p[0], c);  // the smallest first
    c = O::mma(a.p[0], b.p[2], c);
    c = O::mma(a.p[1], b.p[1], c);
    c = O::mma(a.p[1], b.p[0], c);
    c = O::mma(a.p[0], b.p[1], c);
    return O::mma(a.p[0], b.p[0], c);
  }
  // two floats into their parts, a word of two for each
  __device__ static __forceinline__ void split(float a, float b, uint32_t (&w)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      w[i] = pack2<bf16>(a, b);
      a -= __uint_as_float(w[i] << 16);
      b -= __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ static __forceinline__ Frag rows(const bf16* p, int half, int plane) {
    return Frag{{Ops<bf16>::rows(p, half), Ops<bf16>::rows(p + plane, half), Ops<bf16>::rows(p + 2 * plane, half)}};
  }
  template <bool TURNED>
  __device__ static __forceinline__ Frag cols(const bf16* p, int rs, int lane, int plane) {
    return Frag{{Ops<bf16>::cols<TURNED>(p, rs, lane), Ops<bf16>::cols<TURNED>(p + plane, rs, lane),
                 Ops<bf16>::cols<TURNED>(p + 2 * plane, rs, lane)}};
  }
  __device__ static __forceinline__ Frag pack(const float* v) {
    Frag f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t w[3];
      split(v[2 * e], v[2 * e + 1], w);
#pragma unroll
      for (int i = 0; i < 3; ++i) f.p[i][e] = w[i];
    }
    return f;
  }
  __device__ static __forceinline__ void unpack(const Frag& f, float* v) {
    float u[8];
    Ops<bf16>::unpack(f.p[2], v);
#pragma unroll
    for (int i = 1; i >= 0; --i) {
      Ops<bf16>::unpack(f.p[i], u);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += u[e];
    }
  }
  // the first part of an infinity is one, and of a NaN
  __device__ static __forceinline__ bool odd(const Frag& f) { return Ops<bf16>::odd(f.p[0]); }
  __device__ static __forceinline__ Frag finite(const Frag& f) {
    typedef Ops<bf16> O;
    return Frag{{O::finite(f.p[0]), O::keep_finite(f.p[1], f.p[0]), O::keep_finite(f.p[2], f.p[0])}};
  }
  __device__ static __forceinline__ void put(u32x4* p, int lane, const Frag& f) {
#pragma unroll
    for (int i = 0; i < 3; ++i) p[i * 64 + lane] = f.p[i];
  }
  __device__ static __forceinline__ Frag get(const u32x4* p, int lane) {
    return Frag{{p[lane], p[64 + lane], p[128 + lane]}};
  }
};
template <typename T> struct OpsOf { typedef Ops<T> type; };
template <> struct OpsOf<float> { typedef Parts type; };

// float32 on float32 matrix instructions (the lowrank step, whose products are few).
template <> struct Ops<float> {
  struct Frag { float v[8]; };
  __device__ static __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
    return c;
  }
  template <bool TURNED>
  __device__ static __forceinline__ Frag cols(const float* p, int rs, int lane) {
    static_assert(!TURNED, "plain order");
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = p[(8 * (e / 4) + 4 * (lane / 32) + e % 4) * rs + lane % 32];
    return f;
  }
  __device__ static __forceinline__ Frag pack(const float* v) {
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = v[e];
    return f;
  }
};

// Elements from a row of a tile to the next in LDS.  Measured over 16 bytes of padding by 16, eight wavefronts: row
// reads of 16 bytes take 2048 cycles a KB of reads without padding, 370 with an odd multiple of 16 bytes; transposing
// reads 4 cycles each from 32 bytes on, under 3 with 64.  Rows of q and k take 48, v's (only read by columns) 64.
template <typename T, int N, bool TURNED>
constexpr int row_elems() {
  return N + (sizeof(T) == 4 ? 16 : !TURNED ? (N % 128 == 0 ? 64 : 32) : N % 128 == 0 ? 48 : 16) / (int)sizeof(T);
}

constexpr int kOut = 0x7FFFFFF0;  // a byte offset past every buffer's range

// g^k, g = 2^lam2; g^0 = 1 also where lam2 is minus infinity.
__device__ __forceinline__ float power(float lam2, int k) { return k == 0 ? 1.f : exp2f(lam2 * (float)k); }

// The end of a phase: what it has read of LDS is read again by the next one, and nothing moves across.  Without it the
// compiler keeps operands for the following phases, and spills.
__device__ __forceinline__ void phase() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// One tile of C rows of N channels on its way from memory to LDS, in 16-byte
// pieces, which wait in registers through the chunk before.  WHOLE: every piece of
// a row lies inside or outside of it, 16-byte aligned, rows within 32-bit offsets of
// each other: buffer loads, whose range drops the rows past `end`.  Otherwise
// pieces are gathered element by element.
template <typename T, int C, int N, int NT, bool WHOLE>
struct Tile {
  static constexpr int VE = 16 / (int)sizeof(T), PR = N / VE, NV = C * PR / NT, RPI = NT / PR;
  static_assert(C * PR % NT == 0 && NT % PR == 0, "whole pieces and rows to every thread");
  u32x4 v[NV];
  // the tile's last row is token `end` - 1 (or p0 + C - 1), rows before token p0 are zero; token p of a head sits at row p
  // of `base`, or turn - p where turn >= 0
  __device__ __forceinline__ void load(const T* base, int64_t stride, int width, int p0, int end, int turn) {
    const int n = min(end - p0, C), r0 = (int)threadIdx.x / PR - (C - n), c = ((int)threadIdx.x % PR) * VE;
    if constexpr (WHOLE) {
      // the range holds the n tokens: the rows before them fall in front of it, or (turned) behind
      const T* first = base + (int64_t)(turn >= 0 ? turn - (p0 + n - 1) : p0) * stride;
      const int sb = (int)stride * (int)sizeof(T);
      const rsrc_t rs = make_rsrc_wave<(int64_t(1) << 30)>(first, ((int64_t)(n - 1) * stride + width) * (int64_t)sizeof(T));
      const int step = turn >= 0 ? -sb : sb;
      const int off = (turn >= 0 ? (n - 1 - r0) * sb : r0 * sb) + c * (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = bload128(rs, c < width ? off + i * RPI * step : kOut);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int r = r0 + i * RPI;
        v[i] = u32x4{0, 0, 0, 0};
        if (r >= 0 && c < width) {
          const T* q = base + (int64_t)(turn >= 0 ? turn - p0 - r : p0 + r) * stride + c;
          T e[VE];
#pragma unroll
          for (int j = 0; j < VE; ++j) e[j] = c + j < width ? q[j] : (T)0.f;
          __builtin_memcpy(&v[i], e, 16);
        }
      }
    }
  }
  // TURNED: channels in quad() order; planes `plane` elements apart
  template <typename O, bool TURNED>
  __device__ __forceinline__ void store(typename O::Lds* lds, int plane) const {
    typedef typename O::Lds L;
    const int c = ((int)threadIdx.x % PR) * VE;
    L* to = lds + (int)threadIdx.x / PR * row_elems<L, N, TURNED>() + (TURNED ? quad(c) : c);
#pragma unroll
    for (int i = 0; i < NV; ++i, to += RPI * row_elems<L, N, TURNED>()) {
      if constexpr (O::kPlanes == 3) {
        uint32_t a[3], b[3];
        O::split(__uint_as_float(v[i][0]), __uint_as_float(v[i][1]), a);
        O::split(__uint_as_float(v[i][2]), __uint_as_float(v[i][3]), b);
#pragma unroll
        for (int j = 0; j < 3; ++j) *reinterpret_cast<u32x2*>(to + j * plane) = u32x2{a[j], b[j]};
      } else if constexpr (TURNED) {  // two quads, which part
        *reinterpret_cast<u32x2*>(to) = u32x2{v[i][0], v[i][1]};
        *reinterpret_cast<u32x2*>(to + 8) = u32x2{v[i][2], v[i][3]};
      } else {
        *reinterpret_cast<u32x4*>(to) = v[i];
      }
    }
  }
};

// The largest of N values.
template <int N>
__device__ __forceinline__ float largest(const float* v, float m = 0.f) {
#pragma unroll
  for (int i = 0; i < N; i += 2) m = fmaxf(fmaxf(m, fabsf(v[i])), fabsf(v[i + 1]));
  return m;
}
template <int N>
__device__ __forceinline__ void scale(float* v, float by) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] *= by;
}

// fp16 operands whose largest value m may lie anywhere in float32's range: the exponent that brings it between 2^14 and
// 2^15, so that what is down to 2^-28 of it keeps all of the type's bits.  (An infinity or a NaN gives any: its products
// are not finite either way.)
__device__ __forceinline__ int lift_of(float m) { return min(15 - __builtin_amdgcn_frexp_expf(m), 120); }
__device__ __forceinline__ float two_to(int n) { return __builtin_ldexpf(1.f, n); }
// The larger of a lane's value and its partner's, 32 lanes on.
__device__ __forceinline__ float pair_max(float m) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// The exponent of a lane's largest value m, far below all others where m is zero or not finite, and its largest over the
// wavefront.
__device__ __forceinline__ int exponent_of(float m) {
  return m > 0.f && m < __builtin_inff() ? __builtin_amdgcn_frexp_expf(m) : -1000;
}
__device__ __forceinline__ int wave_max(int e) {
  auto dpp = [&](auto ctrl) { return max(e, __builtin_amdgcn_update_dpp(0, e, decltype(ctrl)::value, 0xF, 0xF, false)); };
  e = dpp(std::integral_constant<int, 0xB1>());   // pairs
  e = dpp(std::integral_constant<int, 0x4E>());   // quads
  e = dpp(std::integral_constant<int, 0x141>());  // the mirrored lane of 8
  e = dpp(std::integral_constant<int, 0x140>());  // of 16
  return max(max(__builtin_amdgcn_readlane(e, 0), __builtin_amdgcn_readlane(e, 16)),
             max(__builtin_amdgcn_readlane(e, 32), __builtin_amdgcn_readlane(e, 48)));
}
// The largest magnitude of a lane's 8 fp16 values (NaN where one is).
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float largest16(u32x4 f) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, f[i] & 0x7FFF7FFFu));
  return (float)__builtin_bit_cast(_Float16, (uint16_t)max(m[0], m[1]));
}

// A diagonal block's products with the elements of v that are not finite, for the tokens from theirs on: v points at
// (token 0, column 0), p at the block's scores.
template <typename O, int PL>
__device__ __forceinline__ void add_odd(float* acc, const typename O::Lds* v, int rs, const u32x4* p, int lane) {
  typedef typename O::Lds L;
  const int half = lane / 32, col = lane % 32;
#pragma unroll 1
  for (int j = 0; j < 32; ++j) {
    const uint16_t* pj = reinterpret_cast<const uint16_t*>(p + j / 16 * PL * 64 + j / 4 % 2 * 32 + col);
    const float pv = Mma16<L>::to_f(pj[j % 16 / 8 * 4 + j % 4]);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float x = Mma16<L>::to_f(reinterpret_cast<const uint16_t*>(v)[j * rs + 8 * (r / 4) + 4 * half + r % 4]);
      acc[r] += j <= col && !(fabsf(x) < __builtin_inff()) ? pv * x : 0.f;
    }
  }
}

// Wavefronts on a SIMD that leave a kernel's registers unspilled.
constexpr int waves_per_simd(int es, int kp, int nw, bool states) {
  return es == 4 || kp > 128 || (kp == 128 && nw == 2) ? 1 : states ? 3 : 2;
}

// STATES: only the state after each segment, from zero, for states[pass], KP of its rows to a workgroup.  RETURNED: a state that is formed here is the
// caller's result (three parts in bf16; in every kernel they cost the common one 10% by spilled registers).
template <typename T, int KP, int NW, int C, bool WHOLE, bool STATES, bool RETURNED>
__global__ __launch_bounds__(NW * 64, waves_per_simd(sizeof(T), KP, NW, STATES)) void la_chunks(Args A) {
  typedef typename OpsOf<T>::type O;
  typedef typename O::Frag Frag;
  typedef typename O::Lds L;
  constexpr int NT = NW * 64, NB = C / 32, KB = KP / 32, RK = row_elems<L, KP, true>(), RV = row_elems<L, NW * 32, false>();
  constexpr int PL = O::kPlanes, PK = C * RK, PV = C * RV;  // planes of a tile, elements from one to the next
  __shared__ __align__(16) L sk[PL * PK];
  __shared__ __align__(16) L sv[PL * PV];
  // q, and once it has been read o
  constexpr int RO = NW * 32 + 16 / (int)sizeof(T), QB = PL * PK * (int)sizeof(L), OB = C * RO * (int)sizeof(T);
  __shared__ __align__(16) unsigned char sqo[STATES ? 16 : QB > OB ? QB : OB];
  L* const sq = reinterpret_cast<L*>(sqo);
  T* const so = reinterpret_cast<T*>(sqo);
  // scores as operands: blocks of 32 x 32 on and below the diagonal, two steps of a lane's 8; in fp16 each token's are
  // lifted (lift_of), and sback brings them back
  constexpr int NP = NB * (NB + 1) / 2;
  __shared__ u32x4 sp[STATES ? 1 : NP * 2 * PL * 64];
  __shared__ float sback[O::kNarrow && !STATES ? NP * 32 : 1];

  // the passes of one segment run side by side: what one reads, the others find in the last-level cache
  int blk = A.blk0 + xcd_remap(blockIdx.x, A.nblk);
  const int vb = blk % A.nvb;
  blk /= A.nvb;
  const int k0 = STATES ? blk % A.nkb * KP : 0;  // first row of the state
  if (STATES) blk /= A.nkb;
  const int pass = blk % A.npass;
  blk /= A.npass;
  const LaPass& P = A.p.pass[pass];
  const int seg = P.rev ? A.nseg - 1 - blk % A.nseg : blk % A.nseg, bh = blk / A.nseg;
  const int b = bh / (int)A.p.H, hd = bh % (int)A.p.H;
  const int lane = threadIdx.x % 64, half = lane / 32, col = lane % 32, wv = wave_id();
  const int n0 = vb * NW * 32 + wv * 32;  // first column of this wavefront
  if (vb * NW * 32 >= P.V || k0 >= P.K) return;
  if (STATES && seg == A.nseg - 1 && !P.s_out) return;  // nothing reads the last segment's
  const bool mine = n0 < P.V;
  const float lam = A.p.log_decay[hd], lam2 = lam * 1.44269504088896f;
  const int T_ = (int)A.p.T;
  const int len = A.p.lengths ? min(max(A.p.lengths[b], 0), T_) : T_;
  const int lo = seg * A.seg, top = min(T_, lo + A.seg), hi = min(len, top);
  const int turn = P.rev ? len - 1 : -1;
  const T* k = (const T*)P.k + b * P.ks[0] + hd * P.ks[1] + k0;
  const T* v = (const T*)P.v + b * P.vs[0] + hd * P.vs[1] + vb * NW * 32;
  const T* q = (const T*)P.q + b * P.qs[0] + hd * P.qs[1];
  T* o = (T*)P.o + b * P.os[0] + hd * P.os[1];
  const int vw = P.V - vb * NW * 32;

  float* states = A.states[pass];
  if (states) states += ((int64_t)bh * A.nseg + seg) * P.K * P.V;
  const int64_t sbase = (int64_t)bh * P.K * P.V;

  // element (a, n0 + col) of a state of this head, a = row + 4 half, through a buffer of the state's range
  const int K = P.K, V = P.V, srow = (int)P.s_row * 4, scol = (int)P.s_col * 4, srange = K * V * 4;
  auto at = [=](int a, int c) {
    const int off = a * srow + c * scol;
    return ((a < K) & (c < V)) ? off : kOut;
  };
  f32x16 S[KB];
  {
    const float* from = STATES ? nullptr : states ? states : P.s_in ? P.s_in + sbase : nullptr;
    const rsrc_t rs = make_rsrc_wave(from, from ? srange : 0);  // no state: zeros
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        S[kb][r] = __uint_as_float(bload32(rs, at(k0 + kb * 32 + 8 * (r / 4) + 4 * half + r % 4, n0 + col)));
  }

  // weights that every full chunk has, element e of a step (or register r of a result) at row(e): of the last 16
  // tokens for S, and of a score on the diagonal
  auto row = [&](int e) { return 8 * (e / 4) + 4 * half + e % 4; };
  float vlast[8], diag[STATES ? 1 : 16];
#pragma unroll
  for (int e = 0; e < 8; ++e) vlast[e] = P.skv * power(lam2, 15 - row(e));
  if constexpr (!STATES)
#pragma unroll
    for (int r = 0; r < 16; ++r) diag[r] = P.skv * P.so * power(lam2, max(col - row(r), 0));
  const float g16 = power(lam2, 16), gcol = P.so * power(lam2, col + 1);
  const float gC = power(lam2, C);

  constexpr bool three = __is_same(T, bf16) && RETURNED;
  // fp16: S is held times 2^ex; smax: the exponent of a column's largest value; skv_top: v's largest weight in its 16 tokens
  int ex = 0, smax = -1000;
  const float skv_top = fabsf(P.skv) * fmaxf(1.f, power(lam2, 15));

  // tiles on their way: the next chunk's (STATES with the one after it too: 62 -> 67 us at B2 H32 T8192 hd128)
  Tile<T, C, KP, NT, WHOLE> tk, tq;
  Tile<T, C, NW * 32, NT, WHOLE> tv;
  auto fetch_k = [&](int p) { if (p < hi) tk.load(k, P.ks[2], P.K - k0, p, hi, turn); };
  auto fetch_v = [&](int p) { if (p < hi) tv.load(v, P.vs[2], vw, p, hi, turn); };
  auto fetch_q = [&](int p) { if (!STATES && p < hi) tq.load(q, P.qs[2], P.K, p, hi, turn); };
  fetch_k(lo);
  fetch_v(lo);
  fetch_q(lo);
  for (int p0 = lo; p0 < hi; p0 += C) {
    __syncthreads();  // the chunk before has been read
    tk.template store<O, true>(sk, PK);
    tv.template store<O, false>(sv, PV);
    if constexpr (!STATES) tq.template store<O, true>(sq, PK);
    __syncthreads();
    // the next loads go out a tile at a time between the phases: twelve at once hold a wavefront up for 1100 cycles
    fetch_k(p0 + C);
    if (STATES) fetch_v(p0 + C);
    if (STATES && !mine) continue;
    const int cl = min(C, hi - p0), shift = C - cl;  // tokens of this chunk: its last rows
    const int early = P.rev && p0 == 0 ? 1 : 0;      // the entering state meets the first token without a decay
    // opaque, or the compiler forms every product of these weights before the loop, and spills
    float g1 = g16;
    asm volatile("" : "+v"(g1));
    float* const Sf = reinterpret_cast<float*>(S);

    if constexpr (!STATES) {
      // the blocks of scores go round the wavefronts: 0 (0, 0), 1 (1, 0), 2 (1, 1); those of zero rows are not used
      for (int blk = wv; blk < NP; blk += NW) {
        const int ib = blk > 0, jb = blk > 1;
        if (jb * 32 + 31 < shift) continue;
        f32x16 sc = {};
#pragma unroll
        for (int s = 0; s < KP / 16; ++s)
          sc = O::mma(O::rows(sk + (jb * 32 + col) * RK + s * 16, half, PK), O::rows(sq + (ib * 32 + col) * RK + s * 16, half, PK), sc);
        float t[16];
        if (blk == 1) {  // by way of the block's last token: g^{i-j} = g^{col+1} g^{31-j}, the first factor with o
#pragma unroll
          for (int r = 0; r < 16; ++r) t[r] = sc[r] * (r < 8 ? vlast[r] * g1 : vlast[r - 8]);
        } else {
          const int later = col - 4 * half;
#pragma unroll
          for (int r = 0; r < 16; ++r) t[r] = 8 * (r / 4) + r % 4 <= later ? sc[r] * diag[r] : 0.f;
        }
        if constexpr (O::kNarrow) {
          const int n = lift_of(pair_max(largest<16>(t)));
          scale<16>(t, two_to(n));
          sback[blk * 32 + col] = two_to(-n);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) O::put(sp + (blk * 2 + s) * PL * 64, lane, O::pack(t + 8 * s));
      }

      phase();
      fetch_v(p0 + C);
      f32x16 acc[NB] = {};
      // fp16: the wavefront's columns of S lifted together, by one power of two, which leaves again with o's factors (one of
      // each column's own would stand in the rows of o: 16 registers and 32 products more, 8% of the launch)
      float up = 1.f, back = 1.f;
      if constexpr (O::kNarrow) {
        smax = exponent_of(largest<KB * 16>(Sf)) - ex;
        const int n = min(15 - wave_max(smax), 120);
        up = two_to(min(n - ex, 120));
        back = two_to(-n);
      }
#pragma unroll
      for (int s = 0; s < KP / 16; ++s) {
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = O::kNarrow ? Sf[s * 8 + e] * up : Sf[s * 8 + e];
        const Frag sf = O::pack(t);
#pragma unroll
        for (int ib = 0; ib < NB; ++ib) acc[ib] = O::mma(sf, O::rows(sq + (ib * 32 + col) * RK + s * 16, half, PK), acc[ib]);
      }
      __syncthreads();  // the scores are there, and q has been read
      fetch_q(p0 + C);
      if (!mine) continue;
#pragma unroll
      for (int ib = 0; ib < NB; ++ib) {
        if (ib * 32 + 31 < shift) continue;
        float* const af = reinterpret_cast<float*>(&acc[ib]);
        // by: what the sum is multiplied with later on, and these products with it
        auto add = [&](int jb, float by) {
          const int blk = ib + jb;
          Frag vf[2];
#pragma unroll
          for (int s = 0; s < 2; ++s) vf[s] = O::template cols<false>(sv + (jb * 2 + s) * 16 * RV + wv * 32, RV, lane, PV);
          const bool late = jb == ib && __any(O::odd(vf[0]) | O::odd(vf[1]));
          if (late) {
            vf[0] = O::finite(vf[0]);
            vf[1] = O::finite(vf[1]);
          }
          // lifted scores: sums of their own, brought back by token
          f32x16 own = {};
          f32x16& sum = O::kNarrow ? own : acc[ib];
          float* const sf = reinterpret_cast<float*>(&sum);
#pragma unroll
          for (int s = 0; s < 2; ++s) sum = O::mma(vf[s], O::get(sp + (blk * 2 + s) * PL * 64, lane), sum);
          if (late) add_odd<O, PL>(sf, sv + jb * 32 * RV + wv * 32, RV, sp + blk * 2 * PL * 64, lane);
          if constexpr (O::kNarrow) {
            const float back = sback[blk * 32 + col] * by;
#pragma unroll
            for (int r = 0; r < 16; ++r) af[r] = fmaf(sf[r], back, af[r]);
          }
        };
        if (ib > 0 && shift < 32) {  // the state and the block before by way of its last token: g^{i+1} = g^{32} g^{col+1}
          if constexpr (O::kNarrow) {
            scale<16>(af, power(lam2, 32 - early - shift) * gcol * back);
            add(0, gcol);
          } else {
            scale<16>(af, power(lam2, 32 - early - shift));
            add(0, 1.f);
            scale<16>(af, gcol);
          }
        } else {
          scale<16>(af, P.so * power(lam2, max(ib * 32 + col + 1 - early - shift, 0)) * back);
        }
        add(ib, 1.f);
#pragma unroll
        for (int g = 0; g < 4; ++g) store_vals<T, 4>(so + (ib * 32 + col) * RO + wv * 32 + 8 * g + 4 * half, af + 4 * g);
      }
      // o leaves by way of LDS, in 16-byte pieces of a row (the pieces that the wavefront's 32 columns have)
      constexpr int VE = 16 / (int)sizeof(T), PR = 32 / VE, RPI = 64 / PR;
      const int r0 = lane / PR - shift, c = lane % PR * VE;
      const T* from = so + lane / PR * RO + wv * 32 + c;
      if constexpr (WHOLE) {
        // rows in front of the chunk's tokens fall out of the range, as they do in Tile
        const int64_t st = P.os[2];
        const int sb = (int)st * (int)sizeof(T), step = turn >= 0 ? -RPI * sb : RPI * sb;
        const T* first = o + (turn >= 0 ? turn - (p0 + cl - 1) : p0) * st + n0;
        const rsrc_t rs = make_rsrc_wave(const_cast<T*>(first), ((cl - 1) * st + P.V - n0) * (int64_t)sizeof(T));
        const int off = (turn >= 0 ? cl - 1 - r0 : r0) * sb + c * (int)sizeof(T);
#pragma unroll
        for (int it = 0; it < C / RPI; ++it)
          bstore128<false>(*reinterpret_cast<const u32x4*>(from + it * RPI * RO), rs, n0 + c < P.V ? off + it * step : kOut);
      } else {
#pragma unroll
        for (int it = 0; it < C / RPI; ++it) {
          const int i = r0 + it * RPI;
          T* to = o + (int64_t)(turn >= 0 ? turn - p0 - i : p0 + i) * P.os[2] + n0 + c;
#pragma unroll
          for (int j = 0; j < VE; ++j)
            if (i >= 0 && n0 + c + j < P.V) to[j] = from[it * RPI * RO + j];
        }
      }
    }

    phase();
    // S <- g^cl S + k^T (skv g^{C-1-row} v).  In fp16 S is held times 2^ex, each column by itself, so that the chunk's
    // weighted v come between 2^14 and 2^15 (by a bound of each 16 tokens, which weights below it only lower by g^15)
    float lift = 1.f;
    if constexpr (O::kNarrow) {
      float m = 0.f, g = skv_top;
#pragma unroll
      for (int s = C / 16 - 1; s >= 0; --s, g *= g1)
        m = fmaxf(m, largest16(O::template cols<false>(sv + s * 16 * RV + wv * 32, RV, lane, PV)) * g);
      // S itself stays within float32: a large one asks for no more of v
      const int n = min(min(lift_of(pair_max(m)), 64), 100 - smax);
      scale<KB * 16>(Sf, power(lam2, cl - early) * two_to(n - ex));
      lift = two_to(n);
      ex = n;
    } else {
      scale<KB * 16>(Sf, cl == C && !early ? gC : power(lam2, cl - early));
    }
#pragma unroll
    for (int s = 0; s < C / 16; ++s) {
      float t[8], g = lift;  // g^{C-16-16s}
#pragma unroll
      for (int i = s + 1; i < C / 16; ++i) g *= g1;
      O::unpack(O::template cols<false>(sv + s * 16 * RV + wv * 32, RV, lane, PV), t);
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] *= vlast[e] * g;
      const Frag v1 = O::pack(t);
      Frag v2, v3;
      if constexpr (O::kSplit) {
        float u[8];
        O::unpack(v1, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] -= u[e];
        v2 = O::pack(t);
        if (three) {
          O::unpack(v2, u);
#pragma unroll
          for (int e = 0; e < 8; ++e) t[e] -= u[e];
          v3 = O::pack(t);
        }
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const Frag kf = O::template cols<true>(sk + s * 16 * RK + kb * 32, RK, lane, PK);
        S[kb] = O::mma(kf, v1, S[kb]);
        if constexpr (O::kSplit) S[kb] = O::mma(kf, v2, S[kb]);
        if (three) S[kb] = O::mma(kf, v3, S[kb]);
      }
    }
  }

  // the final state of a head in one segment, or the segment's own
  float* to = STATES ? states : states ? nullptr : P.s_out ? P.s_out + sbase : nullptr;
  if (to) {
    float g = !STATES && P.rev && len > 0 ? power(lam2, 1) : 1.f;
    if constexpr (O::kNarrow) g *= two_to(-ex);
    const rsrc_t rs = make_rsrc_wave(to, srange);
    // opaque to the compiler, which would otherwise keep the offsets of the first
    // state's loads in registers through the whole segment (100 spilled registers)
    int h4 = 4 * half, c = n0 + col;
    asm volatile("" : "+v"(h4), "+v"(c));
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        BufUnit<4>::template store<false>(__float_as_uint(S[kb][r] * g), rs, at(k0 + kb * 32 + 8 * (r / 4) + h4 + r % 4, c));
  }
  if constexpr (!STATES) {  // rows past the sequence's length
    constexpr int VE = 16 / (int)sizeof(T), PR = NW * 32 / VE;
    const int c = (int)threadIdx.x % PR * VE;
    for (int t = max(len, lo) + (int)threadIdx.x / PR; t < top; t += NT / PR) {
      T* to = o + t * P.os[2] + vb * NW * 32 + c;
      if (WHOLE && c < vw) *reinterpret_cast<u32x4*>(to) = u32x4{0, 0, 0, 0};
      if constexpr (!WHOLE)
        for (int j = 0; j < VE; ++j)
          if (c + j < vw) to[j] = (T)0.f;
    }
  }
}

// The kernel of a type for these sizes (instantiated in linattn_<type>.hip).
template <typename T, int KP, int NW, bool STATES>
void launch_dims(const Args& a, bool whole, hipStream_t st) {
  constexpr int C = chunk_tokens(sizeof(T));
  constexpr bool B16 = __is_same(T, bf16);
  auto run = [&](auto kernel) { kernel<<<(unsigned)a.nblk, NW * 64, 0, st>>>(a); };
  if (B16 && a.returned) run(whole ? la_chunks<T, KP, NW, C, true, STATES, B16> : la_chunks<T, KP, NW, C, false, STATES, B16>);
  else run(whole ? la_chunks<T, KP, NW, C, true, STATES, false> : la_chunks<T, KP, NW, C, false, STATES, false>);
}
template <typename T>
hipError_t launch(const Args& a, int kp, int nw, bool whole, bool states, hipStream_t st) {
  if (states) nw == 2 ? launch_dims<T, kStateRows, 2, true>(a, whole, st) : launch_dims<T, kStateRows, 4, true>(a, whole, st);
  else if (kp == 64) nw == 2 ? launch_dims<T, 64, 2, false>(a, whole, st) : launch_dims<T, 64, 4, false>(a, whole, st);
  else if (kp == 128) nw == 2 ? launch_dims<T, 128, 2, false>(a, whole, st) : launch_dims<T, 128, 4, false>(a, whole, st);
  else launch_dims<T, 256, 4, false>(a, whole, st);
  return hipGetLastError();
}
extern template hipError_t launch<bf16>(const Args&, int, int, bool, bool, hipStream_t);
extern template hipError_t launch<fp16>(const Args&, int, int, bool, bool, hipStream_t);
extern template hipError_t launch<float>(const Args&, int, int, bool, bool, hipStream_t);

}  // namespace la
}  // namespace dc
