// The gated delta rule over whole sequences (include/dynconv_layer.h).
//
//   S' = a S,   u = b (v - k S'),   S <- S' + k^T u,   o = scale q S
//
// in chunks of C tokens.  With the state S before a chunk, c_i the sum of its logarithms of decays up to token i,
// G_i = e^{c_i}, E_ij = e^{c_i - c_j}, D_i = e^{c_C - c_i}, and q, k normed and q scaled:
//
//   A_ij = E_ij k_i.k_j b_j (j < i),   P_ij = E_ij q_i.k_j b_j (j <= i),   T = (1 + A)^-1
//   X = V - G k S,   Z = T X (what the state gets wrong of each token, u = b Z),   O = G q S + P Z,   S <- G_C S + k^T D b Z
//
// and backward, dS the gradient of the state after the chunk, Y that of Z:
//
//   Y = P^T dO + b D k dS,   dX = T^T Y = dV,   dS <- G_C dS + q^T G dO - k^T G dX
//   dP = dO Z^T b (j <= i),   N = -dX Z^T b (j < i)                                    (b of the columns)
//   dq = G dO S^T + (dP E) k
//   W  = (dP E)^T q + D b Z dS^T + (N E)^T k,   R = -G dX S^T + (N E) k,   dk = W + R
//   db_i = (dX_i . Z_i) / b_i = k_i.W_i / b_i (the former where dX keeps more bits than dv)
//   dc_i = q_i.dq_i + k_i.(R_i - W_i),   dc_C += <S after the chunk, dS>;   dlog_decay_i = sum_{l >= i} dc_l
//
// Launches: what each chunk needs of its own keys (T, P and the decays); the states from chunk to chunk with the outputs, and
// in the backward with Z and the states themselves; the same against time for the states' gradients; and the gradients chunk
// by chunk.  A b below 2^-60 counts as that, so that db has its quotient: dX is b times a gradient, and what is summed in
// dX.Z stays a normal float32 where it is above 2^-66 without b (with U = b Z kept instead of Z it was b^2 times that, and
// nothing was left of gradients below 2^-29).
#include "delta_mfma.h"

namespace dc {
namespace {

using dr::Args;
using dr::Stage;

// Parts of what is computed (delta_mfma.h).
int np_of(const DrProblem& p) { return p.dtype == kFP32 || p.precise ? 3 : 2; }
// Halves in memory (delta_mfma.h).
bool halves(const DrProblem& p) { return p.dtype == kBF16 && !p.precise; }
int chunk(const DrProblem& p) { return dr::chunk_of(np_of(p), dr::cover((int)p.K)); }

// How the chains are cut: segments of the tokens, where heads and columns leave CUs idle (one launch finds what each makes of
// the state before it, a second carries the states across, and the chains run side by side), and wavefronts of a workgroup
// where its tiles leave room for one on a CU.  The least estimated time: per chunk of a chain `us`, 0.8 of that without
// outputs (with the unit vectors' columns, twice as many where K is V), in rounds of the workgroups that fit (small tiles
// let wavefronts share SIMDs, at 0.65 of a round for another), and the launches.  Measured, bf16, us (* is what it takes):
// forward of B1 H16 T8192 hd128, 1 segment 427, 2 383, 4 231, 8 176 *, 16 202; B1 H2 T16384 hd128, 8 205, 16 151, 26 154 *,
// 32 159; B1 H16 T32768 hd128 with its state, 1 2845, 4 1530, 8 950, 16 816 *; B1 H4 T2048 hd256, 1 237, 4 141 *, 8 147,
// 16 235 (its transitions are carried at 12 us a segment).
// Training of B4 H32 T2048 hd128: workgroups of 2 wavefronts 864, of 4 624 *; of B4 H16 T4096, 2 818 *, 4 891.
struct Cut {
  int nseg, nw;
};
Cut cut_of(const DrProblem& p, int C, int np) {
  const int kp = dr::cover((int)p.K), vp = ((int)p.V + 31) / 32 * 32;
  const int64_t chunks = (p.T + C - 1) / C, heads = p.B * p.H;
  const bool one = halves(p) && kp >= 128;  // workgroup on a CU; elsewhere two
  const bool shares = np == 3 && kp == 128 && p.dtype == kBF16;  // two or, of more than 512, four (delta_mfma.h)
  double best = -1;
  Cut cut{1, 2};
  for (int nw = 2; nw <= (one && kp == 128 && vp % 64 == 0 ? 4 : 2); nw += 2) {
    auto rounds = [&](double wgs, bool small) {
      if (shares && !small) return wgs <= 512 ? 1 : 1.6 * wgs / 1024 > 0.6 + wgs / 1024 ? 1.6 * wgs / 1024 : 0.6 + wgs / 1024;
      return small ? (wgs <= 512 ? 1 : 0.35 + 0.65 * wgs / 512) : __builtin_ceil(wgs / (one ? 256 : 512));
    };
    const double us = (shares ? 3.2 : 2.8) * (nw == 4 ? 1.25 : 1);
    const int cols = nw * 16;
    for (int s = 1; s <= 64 && (s == 1 || s <= chunks); ++s) {
      const int64_t len = (chunks + s - 1) / s;
      if (s > 1 && (chunks + len - 1) / len != s) continue;  // the same segments as fewer
      double t = us * len * rounds((double)heads * s * (vp / cols), np == 3 && kp == 64);
      if (s > 1)
        t += (shares ? 0.65 : 0.8) * us * len * rounds((double)heads * (s - 1) * ((vp + kp) / cols), true) +
             (shares ? 5 + 3 * s : 15 + (kp == 256 && np == 2 ? 12 : 2) * s);
      if (best < 0 || t < best) {
        best = t;
        cut = {s, nw};
      }
    }
  }
  return cut;
}

// The workspace: of the forward vec, T, P and the segments' states, of the backward dX, where it is not dv, and the states'
// gradients; Z and the states with their exponents, of the forward where it keeps them, else of the backward (the exponents, a
// byte for 8 to 64 values, have room in both, so that keeping moves Z and the states alone).
struct Plan {
  int64_t n, vec, sq, rows, st, ex, cut, trans;  // chunks of a head; bytes of each array
  int vp, seg, nseg, nw;
  bool kept, from_dv;
  explicit Plan(const DrProblem& p) {
    const int C = chunk(p), np = np_of(p);
    n = (p.T + C - 1) / C;
    vp = ((int)p.V + 31) / 32 * 32;
    const int64_t chunks = p.B * p.H * n;
    vec = chunks * dr::kVecs * C * 4;
    sq = chunks * np * C * C * 2;
    const int nd = dr::planes(halves(p), np);
    rows = chunks * nd * C * vp * 2;
    const int kp = dr::cover((int)p.K);
    st = chunks * nd * kp * vp * 2;
    ex = halves(p) ? chunks * 4 * vp : 0;
    const Cut cut_ = cut_of(p, C, np);
    nseg = cut_.nseg;
    nw = cut_.nw;
    seg = (int)((n + nseg - 1) / nseg) * C;
    cut = nseg > 1 ? (p.B * p.H * nseg * p.K * p.V * 4 + 15) / 16 * 16 : 0;
    trans = nseg > 1 ? p.B * p.H * nseg * kp * kp * 4 : 0;
    from_dv = halves(p);
    // saves the backward a launch: training of B4 H16 T4096 hd128 in bf16 956 -> 816 us for 201 MB, 0.75 of q, k, v and o;
    // of B2 T2048 with 8 | 16 heads of 64 x 128 and float32 gates 48 of 377 us would take 3.6 times their memory
    kept = p.keep && rows + st <= 2 * p.B * p.T * (p.Hk * 2 * p.K + p.H * 2 * p.V) * dtype_size(p.dtype);
  }
  int64_t fwd() const { return vec + 2 * sq + trans + cut + 2 * ex + (kept ? rows + st : 0); }
  int64_t bwd() const { return (kept ? 0 : rows + st) + (from_dv ? 0 : rows) + st + 3 * ex + cut; }
};

Args args_of(const DrProblem& p, bool bwd) {
  const Plan pl(p);
  Args a{};
  a.p = p;
  a.n = pl.n;
  a.vp = pl.vp;
  a.seg = pl.seg;
  a.nseg = pl.nseg;
  a.nw = pl.nw;
  char* f = static_cast<char*>(bwd && p.fwd_ws ? const_cast<void*>(p.fwd_ws) : p.ws);
  a.vec = reinterpret_cast<float*>(f);
  a.tt = reinterpret_cast<bf16*>(f + pl.vec);
  a.pp = reinterpret_cast<bf16*>(f + pl.vec + pl.sq);
  a.trans = reinterpret_cast<float*>(f + pl.vec + 2 * pl.sq);
  f += pl.vec + 2 * pl.sq + pl.trans;
  a.start = reinterpret_cast<float*>(f);
  f += pl.cut;
  uint8_t* ex = reinterpret_cast<uint8_t*>(f);
  f += 2 * pl.ex;
  char* w = static_cast<char*>(p.ws) + (p.fwd_ws ? 0 : pl.fwd());  // the backward's
  char* kept = pl.kept ? f : w;
  a.z = reinterpret_cast<bf16*>(kept);
  a.s = reinterpret_cast<bf16*>(kept + pl.rows);
  a.kept = pl.kept;
  if (bwd) {
    if (!pl.kept) w += pl.rows + pl.st;
    a.x = reinterpret_cast<bf16*>(w);
    if (!pl.from_dv) w += pl.rows;
    a.ds = reinterpret_cast<bf16*>(w);
    a.eds = reinterpret_cast<uint8_t*>(w + pl.st);
    if (!pl.kept) ex = a.eds + pl.ex;
    a.dstart = reinterpret_cast<float*>(w + pl.st + 3 * pl.ex);
  }
  a.es = ex;
  a.ez = ex + pl.ex;
  return a;
}

// Rows no shorter apart than they are long, 64 of them within 32-bit offsets.
bool slim(const int64_t (&st)[3], int64_t width, int es) { return st[2] >= width && st[2] * es < (1 << 24); }
// And whole 16-byte pieces.
bool whole16(const void* t, const int64_t (&st)[3], int64_t width, int es) {
  const int64_t n = 16 / es;
  return reinterpret_cast<uintptr_t>(t) % 16 == 0 && st[0] % n == 0 && st[1] % n == 0 && st[2] % n == 0 && width % n == 0 &&
         slim(st, width, es);
}

// whole: rows are whole pieces; then the chains' loads write LDS themselves where they can.
hipError_t run(Stage st, Args a, bool whole, int64_t blocks) {
  const int mode = whole ? dr::kDirect : dr::kGather;
  const DrProblem& p = a.p;
  constexpr int64_t most = most_workgroups(256);
  a.blocks = blocks;
  for (a.blk0 = 0; a.blk0 < blocks; a.blk0 += most) {
    a.nblk = (int)(blocks - a.blk0 < most ? blocks - a.blk0 : most);
    const hipError_t e = p.dtype == kFP32 ? dr::launch<float, 3>(st, a, mode, p.stream)
                         : p.dtype == kFP16 && p.precise ? dr::launch<fp16, 3>(st, a, mode, p.stream)
                         : p.dtype == kFP16              ? dr::launch<fp16, 2>(st, a, mode, p.stream)
                         : p.precise                     ? dr::launch<bf16, 3>(st, a, mode, p.stream)
                                                         : dr::launch<bf16, 2>(st, a, mode, p.stream);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Workgroups of the chains over `seg` segments, and `more` columns beside V's.
int64_t columns(const Args& a, int seg, int more = 0) { return a.p.B * a.p.H * seg * ((a.vp + more) / (a.nw * 16)); }

// What the chunks need of their own keys, and the states before the segments.
hipError_t ahead(const Args& a, bool keys, bool values) {
  const DrProblem& p = a.p;
  hipError_t e = run(dr::kPrep, a, keys, p.B * p.H * a.n);
  if (a.nseg == 1 || e != hipSuccess) return e;
  e = run(dr::kAhead, a, keys && values, columns(a, a.nseg - 1, dr::cover((int)p.K)));
  return e != hipSuccess || a.nseg == 2 ? e : run(dr::kCarry, a, true, p.B * p.H * (a.vp / 16));
}

}  // namespace

int64_t dr_ws_bytes(const DrProblem& p, int bwd) {
  const Plan pl(p);
  return (bwd == 2 ? 0 : pl.fwd()) + (bwd ? pl.bwd() : 0);
}

hipError_t dr_fwd(const DrProblem& p) {
  const Args a = args_of(p, false);
  const int es = dtype_size(p.dtype);
  const bool w = whole16(p.q, p.qs, p.K, es) && whole16(p.k, p.ks, p.K, es), v = slim(p.vs, p.V, es);
  const hipError_t e = ahead(a, w, v);
  return e != hipSuccess ? e : run(a.kept ? dr::kChainKeep : dr::kChain, a, w && v && whole16(p.o, p.os, p.V, es), columns(a, a.nseg));
}

hipError_t dr_bwd(const DrProblem& p) {
  const Args a = args_of(p, true);
  const int es = dtype_size(p.dtype);
  const bool w = whole16(p.q, p.qs, p.K, es) && whole16(p.k, p.ks, p.K, es), v = slim(p.vs, p.V, es);
  hipError_t e = p.fwd_ws ? hipSuccess : ahead(a, w, v);
  if (e == hipSuccess && !(p.fwd_ws && a.kept)) e = run(dr::kKeepStates, a, w && v, columns(a, a.nseg));
  const bool d = w && slim(p.dos, p.V, es) && slim(p.dvs, p.V, es);
  if (e == hipSuccess && a.nseg > 1) e = run(dr::kAheadBwd, a, d, columns(a, a.nseg - 1));
  if (e == hipSuccess && a.nseg > 2) e = run(dr::kCarryBwd, a, true, p.B * p.H * (a.vp / 16));
  if (e == hipSuccess) e = run(dr::kChainBwd, a, d, columns(a, a.nseg));
  const bool g = w && whole16(p.d_o, p.dos, p.V, es) && whole16(p.dv, p.dvs, p.V, es) && whole16(p.dq, p.dqs, p.K, es) &&
                 whole16(p.dk, p.dks, p.K, es);
  return e != hipSuccess ? e : run(dr::kGrads, a, g, p.B * p.Hk * a.n);
}

}  // namespace dc
