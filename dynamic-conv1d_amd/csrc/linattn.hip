// Linear attention with a decay for each head: passes, segments and launches
// (kernels: linattn_mfma.h).
//
//   S_t = g S_{t-1} + k_t^T v_t,    o_t = s q_t S_t,    g = exp(log_decay[h])
//
// The forward is one pass of this recurrence; the backward is three more, each
// the same recurrence on other tensors:
//   dq_t = s (S_t do_t)             forward in time on (do, v, k): state S^T
//   dk_t = (dS_t v_t)               against time on (v, do, q): state dS^T
//   dv_t = (k_t dS_t)               against time on (k, q, do): state dS
// with dS_t = g dS_{t+1} + s q_t^T do_t.  The gradient of the final state enters
// dS at the last token without a factor, and g dS_0 is the initial state's.
//
// Where batch x heads leave CUs idle, tokens are cut into segments: one launch
// forms each segment's state from zero (k and v are read), a second carries the
// states from segment to segment, the third runs the chunks of every segment from
// its state.  dk and dv walk the same states, turned over.
#include "layer_launch.h"
#include "linattn_mfma.h"

namespace dc {
namespace {

using la::Args;

int cover(int n) { return n <= 64 ? 64 : n <= 128 ? 128 : 256; }

struct Cut {
  int seg, nseg;
};

// Sets of segment states: the forward's one; the backward's two (dq's, and dv's that dk shares).
int sets_of(const LaProblem& p) { return p.npass == 3 ? 2 : 1; }

// Workgroups of a pass that a CU holds at once: by registers two wavefronts on a SIMD in 16 bits up to 128 channels, else
// one; by LDS three tiles each.
int resident(const LaPass& p, int dtype) {
  const int kp = cover(p.K), nw = p.V <= 64 ? 2 : 4;
  if (dtype == kFP32) return nw == 2 && kp == 64 ? 2 : 1;
  if (kp == 256) return 1;
  return nw == 4 ? 2 : kp == 64 ? 4 : 3;
}

// Segments of a problem: the count with the least estimated time, in units of a round of chunks on every CU.  A launch
// takes whole rounds of resident workgroups; segments cost the states' launch (0.4 of a chunk's time for each of its
// chunks, measured 72 us against 172) and carrying them (one unit for 25 MB).  Against filling 512 workgroups by division
// alone: B2 H32 T8192 hd128 backward 9 rounds of 12 chunks for 576 workgroups, now 3 of 16.
Cut cut_of(const LaProblem& p) {
  const int C = la::chunk_tokens(dtype_size(p.dtype), cover(p.pass[0].K));
  const int64_t chunks = (p.T + C - 1) / C;
  const int sets = sets_of(p);
  double best = 0;
  int64_t seg = chunks;
  for (int64_t n = 1; n <= 128 && n <= (chunks + 1) / 2; ++n) {
    const int64_t len = (chunks + n - 1) / n;
    if (n > 1 && (chunks + len - 1) / len != n) continue;  // the same segments as fewer
    double t = 0, wgs = 0;
    for (int i = 0; i < p.npass; ++i) {
      const LaPass& a = p.pass[i];
      const double w = (double)p.B * p.H * n * ((a.V + 127) / 128) / (256 * resident(a, p.dtype));
      wgs += w;
      if (n > 1 && (p.npass == 1 || i != 1)) t += 0.4 * (w < 1 ? 1 : w) * len;
    }
    t += (wgs <= 1 ? 1 : __builtin_ceil(wgs)) * len;
    if (n > 1) t += 1 + 4e-8 * sets * 4 * (double)p.B * p.H * n * p.pass[0].K * p.pass[0].V;
    if (n == 1 || t < best) {
      best = t;
      seg = len;
    }
  }
  if (seg < 1) seg = 1;
  return {(int)(seg * C), (int)(chunks > 0 ? (chunks + seg - 1) / seg : 1)};
}

// States from segment to segment: states[s] <- the state before segment s.
struct Carry {
  const float* log_decay;
  const int32_t* lengths;
  float* states[2];
  const float* s_in[2];
  float* s_out[2];
  int rev[2];
  int64_t H, T, n;  // n: elements of a state
  int seg, nseg;
};

__global__ __launch_bounds__(256) void la_carry(Carry A) {
  const int set = blockIdx.z, rev = A.rev[set];
  const int64_t bh = blockIdx.y, e = ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (e >= A.n) return;
  const int T = (int)A.T;
  const int len = A.lengths ? min(max(A.lengths[bh / A.H], 0), T) : T;
  const double lam = A.log_decay[bh % A.H];
  float* st = A.states[set] + bh * A.nseg * A.n + e;
  float run = A.s_in[set] ? A.s_in[set][bh * A.n + e] : 0.f;
  const float full = (float)exp(lam * A.seg);
  for (int s = 0; s < A.nseg; ++s) {
    const bool last = s == A.nseg - 1;
    const float own = last && !A.s_out[set] ? 0.f : st[s * A.n];
    st[s * A.n] = run;
    const int cnt = min(max(len - s * A.seg, 0), A.seg) - (rev && s == 0 && len > 0 ? 1 : 0);
    const float g = cnt == 0 ? 1.f : cnt == A.seg ? full : (float)exp(lam * cnt);
    run = g * run + own;
  }
  if (A.s_out[set]) A.s_out[set][bh * A.n + e] = rev && len > 0 ? (float)(run * exp(lam)) : run;
}

// Rows of whole 16-byte pieces, 64 of which stay within the 2^30 bytes of a buffer's range.
bool whole16(const void* t, const int64_t (&st)[3], int width, int es) {
  const int64_t n = 16 / es;
  return reinterpret_cast<uintptr_t>(t) % 16 == 0 && st[0] % n == 0 && st[1] % n == 0 && st[2] % n == 0 && width % n == 0 &&
         st[2] >= width && st[2] * es < (1 << 24);
}

// Rows of every tensor of a pass are whole 16-byte pieces.
bool whole(const LaPass& a, int es, bool states) {
  return whole16(a.k, a.ks, a.K, es) && whole16(a.v, a.vs, a.V, es) &&
         (states || (whole16(a.q, a.qs, a.K, es) && whole16(a.o, a.os, a.V, es)));
}

// The passes whose kernel is the same go in one launch.
hipError_t launch(const LaProblem& p, const Cut& c, float* const* states_of, bool states) {
  const int es = dtype_size(p.dtype);
  bool done[kLaMaxPasses] = {};
  for (int i = 0; i < p.npass; ++i) {
    if (done[i]) continue;
    Args a{};
    a.p = p;
    a.seg = c.seg;
    a.nseg = c.nseg;
    const int kp = cover(p.pass[i].K), nw = p.pass[i].V <= 64 ? 2 : 4;
    const bool w = whole(p.pass[i], es, states);
    a.nvb = 1;
    for (int j = i; j < p.npass; ++j) {
      const LaPass& b = p.pass[j];
      if (done[j] || cover(b.K) != kp || (b.V <= 64 ? 2 : 4) != nw || whole(b, es, states) != w) continue;
      done[j] = true;
      a.p.pass[a.npass] = b;
      a.states[a.npass++] = c.nseg > 1 ? states_of[j] : nullptr;
      a.returned |= b.s_out && states == (c.nseg > 1);
      const int nvb = (b.V + nw * 32 - 1) / (nw * 32);
      if (nvb > a.nvb) a.nvb = nvb;
    }
    const int64_t nblk = p.B * p.H * c.nseg * a.nvb;
    if (nblk > 0x7fffffff) return hipErrorInvalidValue;
    a.nblk = (int)nblk;
    hipError_t e;
    switch (p.dtype) {
      case kBF16: e = la::launch<bf16>(a, kp, nw, w, states, p.stream); break;
      case kFP16: e = la::launch<fp16>(a, kp, nw, w, states, p.stream); break;
      default: e = la::launch<float>(a, kp, nw, w, states, p.stream); break;
    }
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

int64_t la_ws_bytes(const LaProblem& p) {
  const Cut c = cut_of(p);
  if (c.nseg == 1) return 0;
  return sets_of(p) * p.B * p.H * c.nseg * (int64_t)p.pass[0].K * p.pass[0].V * (int64_t)sizeof(float);
}

hipError_t la_run(const LaProblem& p) {
  const Cut c = cut_of(p);
  float* of[kLaMaxPasses] = {};
  if (c.nseg > 1) {
    const int sets = sets_of(p);
    const int64_t n = (int64_t)p.pass[0].K * p.pass[0].V, set = p.B * p.H * c.nseg * n;
    float* ws = static_cast<float*>(p.ws);
    of[0] = ws;
    of[1] = of[2] = ws + set;
    // a set's states are formed by the pass whose state lies row by row: dq's k and v change places, dv's stay
    LaProblem f = p;
    f.npass = sets;
    if (sets == 2) f.pass[1] = p.pass[2];
    Carry y{};
    for (int i = 0; i < sets; ++i) {
      LaPass& a = f.pass[i];
      if (a.s_col != 1) {
        const LaPass t = a;
        a.k = t.v; a.v = t.k;
        for (int d = 0; d < 3; ++d) {
          a.ks[d] = t.vs[d];
          a.vs[d] = t.ks[d];
        }
        a.K = t.V; a.V = t.K; a.s_row = t.s_col; a.s_col = 1;
      }
      y.states[i] = of[i];
      y.s_in[i] = a.s_in;
      y.s_out[i] = a.s_out;
      y.rev[i] = a.rev;
    }
    hipError_t e = launch(f, c, of, true);
    if (e != hipSuccess) return e;
    y.log_decay = p.log_decay;
    y.lengths = p.lengths;
    y.H = p.H; y.T = p.T; y.n = n;
    y.seg = c.seg; y.nseg = c.nseg;
    la_carry<<<dim3((unsigned)((n + 255) / 256), (unsigned)(p.B * p.H), (unsigned)sets), 256, 0, p.stream>>>(y);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return launch(p, c, of, false);
}

}  // namespace dc
