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

// Channels of q and k that a kernel holds, and wavefronts of 32 columns of v: two for up to 64 columns, but not at 256
// channels, where four share the loads that two have no registers for.  Channels between the sizes are computed as zeros.
// What that costs, B2 H32 T4096, bf16, forward + backward, us: 32 channels 77 + 91, 64 80 + 103, 96 96 + 176, 128 108 +
// 207, 192 282 + 729, 256 318 + 776; and rows that are not whole 16-byte pieces, which are loaded element by element: 100
// channels 311 + 589.  float32: 32 208 + 356, 64 217 + 366, 96 290 + 702, 100 300 + 714, 128 309 + 730, 192 903 + 2351, 256
// 965 + 2445.
int cover(int n) { return n <= 64 ? 64 : n <= 128 ? 128 : 256; }
int waves(int V, int kp) { return V <= 64 && kp <= 128 ? 2 : 4; }

struct Cut {
  int seg, nseg;
};

// Time of one chunk of a workgroup that has a CU to itself, in us, measured with one segment (float32's chunks have 32
// tokens, the others' 64).  Two workgroups on a CU take nearly twice as long.
double chunk_us(int K, int dtype) {
  const int kp = cover(K);
  const double t = kp == 64 ? 2.4 : kp == 128 ? 3.5 : 6.5;
  return dtype == kFP32 ? 1.8 * t : t;
}

// Segments of a problem, the forward's and the backward's alike: the count with the least estimated time of the forward.
// The chunks run in rounds of one workgroup to a CU; segments cost 0.6 of a chunk's time to form each of their states, all
// but the last one's, the carrying of float32 states at 4.5 TB/s, two launches, and the start of their workgroups.
// Measured, forward + backward, us (* is what the estimate takes): B2 H32 T8192 hd128 bf16, 4 segments 202 + 391 *,
// 8 215 + 402, 3 243 + 456, 1 455 + 550; B1 H8 T700 hd128, 1 segment 40 + 42, 6 24 + 32, 11 24 + 33 *; B8 H32 T4096 hd64,
// 1 segment 172 + 274 *, 2 195 + 446; B3 H10 T1537 hd100 float32, 7 segments 80 + 179 *, 17 85 + 185, 1 312 + 322.
Cut cut_of(const LaProblem& p) {
  // dq's pass of a backward has K and V the other way round: the same cut
  const int K = p.npass == 3 ? p.pass[0].V : p.pass[0].K, V = p.npass == 3 ? p.pass[0].K : p.pass[0].V;
  const int C = la::chunk_tokens(dtype_size(p.dtype));
  const int64_t chunks = (p.T + C - 1) / C;
  const double heads = (double)p.B * p.H, wgs = heads * ((V + 127) / 128), us = chunk_us(K, p.dtype);
  double best = 0;
  int64_t seg = chunks < 1 ? 1 : chunks;
  for (int64_t n = 1; n <= 128 && n <= chunks; ++n) {
    const int64_t len = (chunks + n - 1) / n;
    if ((chunks + len - 1) / len != n) continue;  // the same segments as fewer
    double t = (us * len + 3) * __builtin_ceil(wgs * n / 256);
    if (n > 1) t += 5 + (0.6 * us * len + 2) * __builtin_ceil(wgs * (n - 1) / 256) + heads * n * K * V * 8 / 4.5e6;
    if (n == 1 || t < best) {
      best = t;
      seg = len;
    }
  }
  return {(int)(seg * C), (int)(chunks > 0 ? (chunks + seg - 1) / seg : 1)};
}

// States from segment to segment: states[s] <- the state before segment s.  A thread to an element, which it reads and
// writes once per segment: bound by memory (64 heads, 4 segments, 128 x 128: 34 MB in 7.7 us).
constexpr int kAhead = 8;  // segments' states on their way at once: one by one, 45 segments of 4 heads took 15 us
struct Carry {
  const float* log_decay;
  const int32_t* lengths;
  float* states[2];
  const float* s_in[2];
  float* s_out[2];
  int rev[2];
  int64_t H, T, n;  // n: elements of a state
  int64_t bh0;      // first head of the launch
  int seg, nseg;
};

__global__ __launch_bounds__(256) void la_carry(Carry A) {
  const int set = blockIdx.z, rev = A.rev[set];
  const int64_t bh = A.bh0 + blockIdx.y, e = ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (e >= A.n) return;
  const int T = (int)A.T;
  const int len = A.lengths ? min(max(A.lengths[bh / A.H], 0), T) : T;
  const double lam = A.log_decay[bh % A.H];
  float* st = A.states[set] + bh * A.nseg * A.n + e;
  float run = A.s_in[set] ? A.s_in[set][bh * A.n + e] : 0.f;
  const float full = (float)exp(lam * A.seg);
  for (int s0 = 0; s0 < A.nseg; s0 += kAhead) {
    float own[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int s = s0 + i, end = A.s_out[set] ? A.nseg : A.nseg - 1;
      own[i] = s < end ? st[s * A.n] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int s = s0 + i;
      if (s == A.nseg) break;
      st[s * A.n] = run;
      const int cnt = min(max(len - s * A.seg, 0), A.seg) - (rev && s == 0 && len > 0 ? 1 : 0);
      const float g = cnt == 0 ? 1.f : cnt == A.seg ? full : (float)exp(lam * cnt);
      run = g * run + own[i];
    }
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
    const int kp = states ? la::kStateRows : cover(p.pass[i].K), nw = waves(p.pass[i].V, kp);
    const bool w = whole(p.pass[i], es, states);
    a.nvb = a.nkb = 1;
    for (int j = i; j < p.npass; ++j) {
      const LaPass& b = p.pass[j];
      if (done[j] || (!states && cover(b.K) != kp) || waves(b.V, kp) != nw || whole(b, es, states) != w) continue;
      done[j] = true;
      a.p.pass[a.npass] = b;
      a.states[a.npass++] = c.nseg > 1 ? states_of[j] : nullptr;
      a.returned |= b.s_out && states == (c.nseg > 1);
      const int nvb = (b.V + nw * 32 - 1) / (nw * 32);
      if (nvb > a.nvb) a.nvb = nvb;
      const int nkb = states ? (b.K + kp - 1) / kp : 1;
      if (nkb > a.nkb) a.nkb = nkb;
    }
    const int64_t nblk = p.B * p.H * c.nseg * a.nvb * a.nkb * a.npass;
    if (nblk > 0x7fffffff) return hipErrorInvalidValue;
    for (int64_t b0 = 0; b0 < nblk; b0 += most_workgroups(nw * 64)) {
      a.blk0 = (int)b0;
      a.nblk = (int)(nblk - b0 < most_workgroups(nw * 64) ? nblk - b0 : most_workgroups(nw * 64));
      hipError_t e;
      switch (p.dtype) {
        case kBF16: e = la::launch<bf16>(a, kp, nw, w, states, p.stream); break;
        case kFP16: e = la::launch<fp16>(a, kp, nw, w, states, p.stream); break;
        default: e = la::launch<float>(a, kp, nw, w, states, p.stream); break;
      }
      if (e != hipSuccess) return e;
    }
  }
  return hipSuccess;
}

}  // namespace

// Sets of states before each segment: the forward's one, and for the backward dv's, that dk shares, behind dq's, which is
// the forward's, in its workspace, where the caller has kept it.
int64_t la_ws_bytes(const LaProblem& p, bool fwd_states) {
  const Cut c = cut_of(p);
  if (c.nseg == 1) return 0;
  return (p.npass == 3 && !fwd_states ? 2 : 1) * p.B * p.H * c.nseg * (int64_t)p.pass[0].K * p.pass[0].V * (int64_t)sizeof(float);
}

hipError_t la_run(const LaProblem& p) {
  const Cut c = cut_of(p);
  float* of[kLaMaxPasses] = {};
  if (c.nseg > 1) {
    const int64_t n = (int64_t)p.pass[0].K * p.pass[0].V;
    float* ws = static_cast<float*>(p.ws);
    of[0] = ws;
    if (p.npass == 3) {
      of[1] = of[2] = p.fwd_states ? ws : ws + p.B * p.H * c.nseg * n;
      if (p.fwd_states) of[0] = const_cast<float*>(p.fwd_states);
    }
    // the passes that form states, and where
    LaProblem f = p;
    float* at[2];
    f.npass = 0;
    Carry y{};
    for (int i = 0; i < p.npass; i += 2) {
      if (i == 0 && p.npass == 3 && p.fwd_states) continue;
      LaPass& a = f.pass[f.npass];
      a = p.pass[i];
      if (a.s_col != 1) {  // dq's state lies turned over: its k and v change places
        const LaPass t = a;
        a.k = t.v; a.v = t.k;
        for (int d = 0; d < 3; ++d) {
          a.ks[d] = t.vs[d];
          a.vs[d] = t.ks[d];
        }
        a.K = t.V; a.V = t.K; a.s_row = t.s_col; a.s_col = 1;
      }
      at[f.npass] = y.states[f.npass] = of[i];
      y.s_in[f.npass] = a.s_in;
      y.s_out[f.npass] = a.s_out;
      y.rev[f.npass++] = a.rev;
    }
    hipError_t e = launch(f, c, at, true);
    if (e != hipSuccess) return e;
    y.log_decay = p.log_decay;
    y.lengths = p.lengths;
    y.H = p.H; y.T = p.T; y.n = n;
    y.seg = c.seg; y.nseg = c.nseg;
    const unsigned per = 65535;  // heads to a launch: the grid's second axis
    for (int64_t h0 = 0; h0 < p.B * p.H; h0 += per) {
      y.bh0 = h0;
      const unsigned nh = (unsigned)(p.B * p.H - h0 < per ? p.B * p.H - h0 : per);
      la_carry<<<dim3((unsigned)((n + 255) / 256), nh, (unsigned)f.npass), 256, 0, p.stream>>>(y);
      if ((e = hipGetLastError()) != hipSuccess) return e;
    }
  }
  return launch(p, c, of, false);
}

}  // namespace dc
