// Group norm: the plan of a launch (kernels: group_norm.h).
#include <initializer_list>

#include "group_norm.h"

namespace dc {
namespace {

using gn::GnArgs;
using gn::kWaves;
using gn::Plan;

constexpr int kMaxGroup = 4096;  // channels of a group: at most 16 to a lane

// Alignment that every tensor has (0: none has been given).
bool all_aligned(std::initializer_list<const void*> ts, int bytes) {
  for (const void* t : ts)
    if (reinterpret_cast<uintptr_t>(t) % bytes != 0) return false;
  return true;
}

Plan plan_of(const GnProblem& p) {
  const int es = dtype_size(p.dtype);
  const int64_t size = p.D / p.groups;
  Plan pl{};
  // 16-byte pieces where a group is whole in them and every row starts on one (8-byte pieces, else single channels)
  pl.vec = 1;
  for (const int bytes : {16, 8}) {
    if (size % (bytes / es) == 0 && all_aligned({p.x, p.gate, p.dy, p.y, p.dx, p.dgate}, bytes)) {
      pl.vec = bytes / es;
      break;
    }
  }
  const int64_t pieces = (size + pl.vec - 1) / pl.vec;
  pl.lanes = 1;
  while (pl.lanes < 64 && pl.lanes < pieces) pl.lanes *= 2;
  if (pieces > 128) pl.lanes = 256;
  const int64_t per = (pieces + pl.lanes - 1) / pl.lanes;
  pl.nv = 1;
  while (pl.nv < per) pl.nv *= 2;
  const bool wide = pl.lanes > 64;
  pl.gx = (unsigned)(wide ? p.groups : (p.groups + 64 / pl.lanes - 1) / (64 / pl.lanes));
  // row blocks: enough wavefronts for every SIMD of 256 CUs eight times over in the forward, four times in the backward
  // (its partial sums grow with them), and no more than there are rows
  const int64_t waves = p.dy ? 4096 : 8192, rows = wide ? 1 : kWaves;
  const int64_t want = (waves + pl.gx * kWaves - 1) / (pl.gx * kWaves), most = (p.M + rows - 1) / rows;
  pl.gy = want < most ? want : most;
  return pl;
}

hipError_t run(bool bwd, const GnProblem& p, const Plan& pl, const GnArgs& a) {
  switch (p.dtype) {
    case kBF16: return gn::launch_vec<bf16>(bwd, a, pl, p.stream);
    case kFP16: return gn::launch_vec<fp16>(bwd, a, pl, p.stream);
    default: return gn::launch_vec<float>(bwd, a, pl, p.stream);
  }
}

GnArgs args_of(const GnProblem& p, const Plan& pl) {
  GnArgs a{};
  a.x = p.x; a.weight = p.weight; a.bias = p.bias; a.gate = p.gate; a.dy = p.dy;
  a.y = p.y; a.dx = p.dx; a.dgate = p.dgate;
  a.M = p.M; a.D = p.D; a.size = (int)(p.D / p.groups); a.lanes = pl.lanes;
  a.wide_params = p.pdtype == kFP32; a.param_pieces = all_aligned({p.weight, p.bias}, 16); a.eps = p.eps; a.act = p.act;
  return a;
}

}  // namespace

bool gn_shape_ok(const GnProblem& p) { return p.D / p.groups <= kMaxGroup; }

// Partial sums of dw and db for every row block.  The plan of aligned tensors, or of
// single channels where there are more row blocks of those.
int64_t gn_bwd_ws_bytes(const GnProblem& p) {
  static const char kAligned[16] __attribute__((aligned(256))) = {0};
  GnProblem q = p;
  q.x = q.dy = kAligned;
  q.gate = nullptr;
  q.y = q.dx = q.dgate = nullptr;
  int64_t gy = plan_of(q).gy;
  for (const int off : {8, 2}) {
    q.x = kAligned + off;
    const int64_t n = plan_of(q).gy;
    gy = n > gy ? n : gy;
  }
  return 2 * gy * p.D * (int64_t)sizeof(float);
}

hipError_t gn_fwd(const GnProblem& p) {
  const Plan pl = plan_of(p);
  return run(false, p, pl, args_of(p, pl));
}

hipError_t gn_bwd(const GnProblem& p) {
  const Plan pl = plan_of(p);
  GnArgs a = args_of(p, pl);
  a.pw = p.dweight ? p.ws : nullptr;
  a.pb = p.dbias ? p.ws + pl.gy * p.D : nullptr;
  const hipError_t e = run(true, p, pl, a);
  if (e != hipSuccess) return e;
  const PartialReduce r[2] = {{a.pw, p.D, (int)pl.gy, p.dweight ? p.D : 0, p.dweight},
                              {a.pb, p.D, (int)pl.gy, p.dbias ? p.D : 0, p.dbias}};
  return reduce_partials_multi(r, 2, p.pdtype, p.stream);
}

}  // namespace dc
