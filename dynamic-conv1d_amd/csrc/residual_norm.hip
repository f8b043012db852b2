// Residual norm: the plan of a launch (kernels: residual_norm.h).
#include <initializer_list>

#include "residual_norm.h"

namespace dc {
namespace {

using gn::kWaves;
using rn::Args;
using rn::Plan;

bool all_aligned(std::initializer_list<const void*> ts, int bytes) {
  for (const void* t : ts)
    if (reinterpret_cast<uintptr_t>(t) % bytes != 0) return false;
  return true;
}

// A row of up to 1024 channels lies in a wavefront, a longer one in the workgroup.
bool wide(const RnProblem& p) { return p.D > 1024; }

// Row blocks: eight workgroups to a CU in the forward, two in the backward (its registers leave room for one or two, and its
// partial sums grow with them: 1024 instead of 512 cost 4 us of 230 at 16384 x 4096, 4 of 25 at 4611 x 1000), and no more
// than there are rows.
int64_t blocks(const RnProblem& p, bool bwd) {
  const int64_t want = bwd ? 512 : 2048, most = wide(p) ? p.M : (p.M + kWaves - 1) / kWaves;
  return want < most ? want : most;
}

Plan plan_of(const RnProblem& p, bool bwd) {
  const int es = dtype_size(p.dtype), xs = dtype_size(p.xdtype);
  Plan pl{};
  pl.wide = wide(p);
  // 16-byte pieces where rows are whole in them and start on one (8-byte pieces, else single channels)
  pl.vec = 1;
  for (const int bytes : {16, 8}) {
    const int vec = bytes / es, xb = vec * xs < 16 ? vec * xs : 16;
    if (p.D % vec == 0 && all_aligned({p.branch, p.gate, p.dy, p.y, p.dbranch, p.dgate}, bytes) &&
        all_aligned({p.x, p.h, p.dh, p.dx}, xb)) {
      pl.vec = vec;
      break;
    }
  }
  const int64_t lanes = pl.wide ? 256 : 64, pieces = (p.D + pl.vec - 1) / pl.vec;
  pl.nv = (int)((pieces + lanes - 1) / lanes);
  pl.gy = blocks(p, bwd);
  return pl;
}

hipError_t run(bool bwd, const RnProblem& p, const Args& a, const Plan& pl) {
  const bool wide_x = p.xdtype == kFP32;
  switch (p.dtype) {
    case kBF16: return rn::launch_vec<bf16>(bwd, a, pl, wide_x, p.stream);
    case kFP16: return rn::launch_vec<fp16>(bwd, a, pl, wide_x, p.stream);
    default: return rn::launch_vec<float>(bwd, a, pl, wide_x, p.stream);
  }
}

Args args_of(const RnProblem& p, const Plan& pl) {
  Args a{};
  a.g.M = p.M; a.g.D = p.D; a.g.size = (int)p.D; a.g.lanes = pl.wide ? 256 : 64;
  a.g.wide_params = p.pdtype == kFP32;
  a.g.param_pieces = all_aligned({p.weight, p.branch_weight, p.scale}, 16);
  a.g.eps = p.eps; a.g.act = p.act;
  a.x = p.x; a.branch = p.branch; a.weight = p.weight; a.branch_weight = p.branch_weight; a.gate = p.gate; a.scale = p.scale;
  a.dy = p.dy; a.dh = p.dh; a.y = p.y; a.h = p.h; a.dx = p.dx; a.dbranch = p.dbranch; a.dgate = p.dgate;
  a.constant = p.constant;
  return a;
}

}  // namespace

int64_t rn_bwd_ws_bytes(const RnProblem& p) { return 3 * blocks(p, true) * p.D * (int64_t)sizeof(float); }

hipError_t rn_fwd(const RnProblem& p) {
  const Plan pl = plan_of(p, false);
  return run(false, p, args_of(p, pl), pl);
}

hipError_t rn_bwd(const RnProblem& p) {
  const Plan pl = plan_of(p, true);
  Args a = args_of(p, pl);
  const int64_t n = pl.gy * p.D;
  a.pw = p.dweight ? p.ws : nullptr;
  a.pb = p.dbranch_weight ? p.ws + n : nullptr;
  a.ps = p.dscale ? p.ws + 2 * n : nullptr;
  const hipError_t e = run(true, p, a, pl);
  if (e != hipSuccess) return e;
  const PartialReduce r[3] = {{a.pw, p.D, (int)pl.gy, p.dweight ? p.D : 0, p.dweight},
                              {a.pb, p.D, (int)pl.gy, p.dbranch_weight ? p.D : 0, p.dbranch_weight},
                              {a.ps, p.D, (int)pl.gy, p.dscale ? p.D : 0, p.dscale}};
  return reduce_partials_multi(r, 3, p.pdtype, p.stream);
}

}  // namespace dc
