// Dispatch of the norms over channels and the joins between residual
// blocks: the shape of a launch, and how a backward pass splits its rows.

#include <algorithm>

#include "rownorm.h"

namespace yams {

void join_fwd(int dt, const JoinDesc& d, hipStream_t s) {
  if (d.rows == 0 || d.C == 0) return;
  const RowShape r = row_shape(d.C);
  const int64_t blocks = (d.rows + r.BT / r.TPR - 1) / (r.BT / r.TPR);
  // a few blocks for each CU: more would only load the parameters again
  const int grid = int(std::min<int64_t>(blocks, 2048 * 256 / r.BT));
  DT_SWITCH(dt, {
    typedef TP<kDT> T;
    FwdArgs<T> a;
    a.h = static_cast<const T*>(d.h.p);
    a.x = static_cast<const T*>(d.x.p);
    a.g = static_cast<const T*>(d.g.p);
    a.hs = d.h.stride;
    a.xs = d.x.stride;
    a.gs = d.g.stride;
    a.hk = d.hk;
    a.xk = d.xk;
    a.gk = d.gk;
    a.w = d.w;
    a.b = d.b;
    a.scale = d.scale;
    a.w2 = d.w2;
    a.b2 = d.b2;
    a.y = static_cast<T*>(d.y);
    a.u = static_cast<T*>(d.u);
    a.rows = d.rows;
    a.C = d.C;
    a.G = ceil_div(d.C, kGroup);
    a.TPR = r.TPR;
    a.read = read_of(d.C);
    a.gate_act = d.gate_act;
    a.post = d.post;
    a.next = d.next;
    a.eps = d.eps;
    a.alpha = d.alpha;
    a.inv_c = 1.f / float(d.C);
    a.group = fast_div(unsigned(d.group_rows));
    const bool kept = d.hk.codes != nullptr || d.xk.codes != nullptr;
    join_fwd_launch<kDT>(a, r, d.layer, d.h.p != nullptr, d.gate, kept, grid,
                         s);
  });
}

namespace {

struct BwdPlan {
  RowShape r;
  int64_t groups, group_rows, part_rows;
  int parts, grid;
};

BwdPlan bwd_plan(int dt, const JoinDesc& d) {
  BwdPlan b;
  b.r = row_shape(d.C);
  const bool shared = d.gate == GATE_GROUP;
  b.group_rows = shared ? d.group_rows : d.rows;
  b.groups = d.rows / b.group_rows;
  const int rpb = b.r.BT / b.r.TPR;
  // the blocks that the chip holds at once, by the registers of the kernels
  // (bwd_waves(); two waves a SIMD for fp32 with what LayerNorm and a gate
  // take: 20000 x 1536 318 -> 254 us with 512 blocks for 768); fewer where a
  // block would get under four steps.  Runs shorter than a step leave teams
  // idle, so that they get blocks of their own (512 runs of 3 x 16: 915 us
  // with 6 blocks, 9.5 with 512).
  const bool has_h = d.h.p != nullptr || d.hk.codes != nullptr;
  const bool four = b.r.BT >= 512 || !has_h ||
                    (!d.layer && dt != DT_F32 && !shared);
  const bool two = dt == DT_F32 && d.layer && d.gate != GATE_NONE;
  const int64_t most = 256 * (four ? 1024 : two ? 512 : 768) / b.r.BT;
  const int64_t steps = b.groups * ((b.group_rows + rpb - 1) / rpb);
  const int64_t blocks = std::min<int64_t>(
      most, std::max<int64_t>({1, steps / 4,
                               b.group_rows < rpb ? b.groups : 0}));
  if (b.groups >= blocks) {
    b.parts = 1;
    b.part_rows = b.group_rows;
    b.grid = int(blocks);
  } else {
    const int64_t parts = (blocks + b.groups - 1) / b.groups;
    b.part_rows = std::max<int64_t>((b.group_rows + parts - 1) / parts, 1);
    b.part_rows = (b.part_rows + rpb - 1) / rpb * rpb;
    b.parts = int((b.group_rows + b.part_rows - 1) / b.part_rows);
    b.grid = int(b.groups * b.parts);
  }
  return b;
}

}  // namespace

int64_t join_bwd_ws(int dt, const JoinDesc& d) {
  if (d.rows == 0 || d.C == 0) return 0;
  const BwdPlan b = bwd_plan(dt, d);
  const int64_t Cp = (d.C + 3) / 4 * 4;
  int64_t n = b.grid == 1 ? 0 : b.grid * __builtin_popcount(d.want) * Cp;
  if (d.gate == GATE_GROUP && b.parts > 1)
    n += int64_t(b.parts) * b.groups * d.C;
  return n;
}

void join_bwd(int dt, const JoinDesc& d, hipStream_t s) {
  if (d.rows == 0 || d.C == 0) return;
  const BwdPlan b = bwd_plan(dt, d);
  const RowShape& r = b.r;
  const int64_t Cp = (d.C + 3) / 4 * 4;
  const int nsums = __builtin_popcount(d.want);
  const bool one = b.grid == 1;  // one row of partial sums is the sum
  DT_SWITCH(dt, {
    typedef TP<kDT> T;
    BwdArgs<T> a;
    a.h = static_cast<const T*>(d.h.p);
    a.x = static_cast<const T*>(d.x.p);
    a.g = static_cast<const T*>(d.g.p);
    a.dy = static_cast<const T*>(d.dy.p);
    a.du = static_cast<const T*>(d.du.p);
    a.hs = d.h.stride;
    a.xs = d.x.stride;
    a.gs = d.g.stride;
    a.dys = d.dy.stride;
    a.dus = d.du.stride;
    a.hk = d.hk;
    a.xk = d.xk;
    a.gk = d.gk;
    a.w = d.w;
    a.b = d.b;
    a.scale = d.scale;
    a.w2 = d.w2;
    a.dh = static_cast<T*>(d.dh);
    a.dx = static_cast<T*>(d.dx);
    a.dg = static_cast<T*>(d.dg);
    a.ws = one ? d.sums : d.ws;
    a.wsg = d.ws + (one ? 0 : int64_t(b.grid) * nsums * Cp);
    a.rows = d.rows;
    a.group_rows = b.group_rows;
    a.groups = b.groups;
    a.part_rows = b.part_rows;
    a.parts = b.parts;
    a.C = d.C;
    a.Cp = int(Cp);
    a.G = ceil_div(d.C, kGroup);
    a.TPR = r.TPR;
    a.read = read_of(d.C);
    a.gate_act = d.gate_act;
    a.post = d.post;
    a.next = d.next;
    a.want = d.want;
    a.eps = d.eps;
    a.alpha = d.alpha;
    a.inv_c = 1.f / float(d.C);
    const bool has_h = d.h.p != nullptr || d.hk.codes != nullptr;
    const bool kept = d.hk.codes != nullptr || d.xk.codes != nullptr;
    join_bwd_launch<kDT>(a, r, d.layer, has_h, d.gate, kept, b.grid, s);
    if (d.gate == GATE_GROUP && b.parts > 1 && d.dg != nullptr)
      gate_fold_launch<kDT>(a.wsg, a.dg, b.groups * d.C, b.parts, s);
  });
  if (nsums > 0 && !one)
    slab_reduce(d.ws, d.sums, nsums * Cp, b.grid, s);
}

}  // namespace yams
