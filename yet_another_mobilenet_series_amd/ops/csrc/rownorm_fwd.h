// Forward of the norms over channels and of the joins between residual
// blocks: y = x + scale * a(gate) * N1(h), u = N2(y), one pass.
//
// A row stays in registers from its load to its stores: each input is
// read once and each output written once, and the 8-bit forms for the
// backward pass come out of the same registers.  Bound by memory.
// Measured (bf16, kept in 8 bits): rms norm of 32768 x 2048 in 60 us, 5.6
// TB/s; join of 16384 x 4096 with a gate and the next norm, 167 us, 5.3 TB/s.
#pragma once

#include "rownorm.h"

namespace yams {

namespace {

// KEPT: the 8-bit forms of h, x and a gate of every row are written too
// (x's only where the next norm's gradient will need it)
template <int DT, int BT, int NV, bool LAYER, bool HAS_H, int GATE, bool KEPT>
__global__ __launch_bounds__(BT) void join_fwd_kernel(
    FwdArgs<TP<DT>> p) {
  constexpr unsigned kSize = unsigned(sizeof(TP<DT>));
  __shared__ float red[6 * (BT / 64)];
  // without h there is nothing else (a loop that might skip all uses of what
  // it loads waits for the last row's stores)
  const bool next = !HAS_H || p.next;
  int turn = 0;
  const int TPR = p.TPR, RPB = BT / TPR;
  const int t = int(threadIdx.x) & (TPR - 1);
  const unsigned team = threadIdx.x / unsigned(TPR);
  const Chunks<NV> chunks(p.C, t, TPR);
  const auto &n = chunks.n, &col = chunks.col;
  float w[NV][8], b[NV][8] = {}, s[NV][8], w2[NV][8], b2[NV][8] = {};
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[j][e] = 1.f;
      s[j][e] = 1.f;
      w2[j][e] = 1.f;
    }
    if (HAS_H) {
      if (p.w != nullptr) load_chunk<DT_F32>(p.w + col[j], n[j], w[j]);
      if (LAYER && p.b != nullptr)
        load_chunk<DT_F32>(p.b + col[j], n[j], b[j]);
      if (p.scale != nullptr)
        load_chunk<DT_F32>(p.scale + col[j], n[j], s[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[j][e] *= p.alpha;
    }
    if (p.w2 != nullptr) load_chunk<DT_F32>(p.w2 + col[j], n[j], w2[j]);
    if (LAYER && p.b2 != nullptr)
      load_chunk<DT_F32>(p.b2 + col[j], n[j], b2[j]);
  }
  // byte offsets of this lane from the first row of the block's step
  const unsigned oh = team * unsigned(p.hs) * kSize;
  const unsigned ox = team * unsigned(p.xs) * kSize;
  const unsigned og = team * unsigned(p.gs) * kSize;
  const unsigned oc = team * unsigned(p.C), oe = team * unsigned(p.G);

  struct Raw {
    RawChunk<DT, false> x[NV], h[NV], g[NV];
  };
  // rows of a team that has none are the first team's
  auto load_row = [&](Raw& q, int64_t base) {
    if (base >= p.rows) return;
    const bool live = base + team < p.rows;
    const unsigned lh = live ? oh : 0u, lx = live ? ox : 0u;
    unsigned lg = live ? og : 0u;
    const TP<DT>* g = p.g + base * p.gs;
    if (GATE == GATE_GROUP) {
      const unsigned at = p.group.div(unsigned(base));
      const unsigned run = p.group.div(unsigned(base) + (live ? team : 0u));
      g = p.g + int64_t(at) * p.gs;
      lg = (run - at) * unsigned(p.gs) * kSize;
    }
    // a single input has nothing to wait for one by one (32768 x 2048, kept in
    // 8 bits: 63 us, and 75 by the other way)
    if (!HAS_H || p.read == READ_SHORT) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int m = live ? n[j] : 0;
        q.x[j].load_short(p.x + base * p.xs, lx + unsigned(col[j]) * kSize, m);
        if (HAS_H) q.h[j].load_short(p.h + base * p.hs, lh, m);
        if (GATE != GATE_NONE) q.g[j].load_short(g, lg, m);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const unsigned c = chunks.from[j] * kSize;
        q.x[j].load(p.x + base * p.xs, lx + c);
        if (HAS_H) q.h[j].load(p.h + base * p.hs, lh + c);
        if (GATE != GATE_NONE) q.g[j].load(g, lg + c);
      }
    }
  };

  // The next row is on its way while this one is worked on, where the
  // registers are there for it (16384 x 4096 with a gate, kept in 8 bits: 200
  // -> 195 us; 8192 x 8192 189 -> 182).  LAYER and NV = 2 lose by it (4097 x
  // 1536 fp32 19.3 -> 22.2; 4096 x 16384 244 -> 363).
  constexpr bool kAhead = HAS_H && !LAYER && NV == 1;
  const int64_t first = int64_t(blockIdx.x) * RPB;
  const int64_t step = int64_t(gridDim.x) * RPB;
  Raw cur;
  if (kAhead) load_row(cur, first);
  for (int64_t base = first; base < p.rows; base += step) {
    Raw nxt;
    if (kAhead)
      load_row(nxt, base + step);
    else
      load_row(cur, base);
    const bool live = base + team < p.rows;
    int m_[NV];  // channels of this row: none behind the last row
    float y[NV][8], h[NV][8], g[NV][8];
    if (HAS_H && p.read == READ_RAGGED) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        cur.x[j].drop(n[j]);
        if (HAS_H) cur.h[j].drop(n[j]);
        if (GATE != GATE_NONE) cur.g[j].drop(n[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      m_[j] = live ? n[j] : 0;
      if (HAS_H) cur.x[j].blank(m_[j]);
      cur.x[j].decode(y[j]);
      if (HAS_H) {
        cur.h[j].blank(m_[j]);
        cur.h[j].decode(h[j]);
      }
      if (GATE != GATE_NONE) {
        cur.g[j].blank(m_[j]);
        cur.g[j].decode(g[j]);
      }
    }
    if (KEPT) {
      auto keep = [&](const Kept& k, const float* v, int j) {
        unsigned e;
        const uint2_t q = quantize8<DT>(v, e);
        put_codes(k.codes + base * p.C, oc + unsigned(col[j]), m_[j], q);
        if (m_[j] > 0 && (t & 3) == 0)
          *lane_at<unsigned char>(k.exps + base * p.G,
                                  oe + unsigned(col[j] >> 5)) =
              (unsigned char)e;
      };
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (next) keep(p.xk, y[j], j);
        if (HAS_H) keep(p.hk, h[j], j);
        if (GATE == GATE_FULL) keep(p.gk, g[j], j);
      }
    }
    if (HAS_H) {
      if (GATE != GATE_NONE) gate_prepare<DT, NV>(g, p.gate_act);
      float mean = 0.f, r = 1.f;
      if (p.post)
        row_stats<NV, BT, LAYER>(h, n, TPR, p.inv_c, p.eps, red, turn, mean,
                                 r);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // channels behind the last one stay zero for the sums: their
          // parameters are zero, and without LAYER hh is
          const float hh = (LAYER ? h[j][e] - mean : h[j][e]) * r;
          const float v = LAYER ? fmaf(hh, w[j][e], b[j][e]) : hh * w[j][e];
          const float sa = GATE != GATE_NONE
                               ? s[j][e] * gate_value(g[j][e], p.gate_act)
                               : s[j][e];
          y[j][e] = fmaf(!LAYER || e < m_[j] ? v : 0.f, sa, y[j][e]);
        }
#pragma unroll
      for (int j = 0; j < NV; ++j)
        put_chunk<DT>(p.y + base * p.C, (oc + unsigned(col[j])) * kSize,
                      m_[j], y[j]);
    }
    if (next) {
      float mean, r;
      row_stats<NV, BT, LAYER>(y, n, TPR, p.inv_c, p.eps, red, turn, mean,
                               r);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          u[e] = LAYER ? fmaf((y[j][e] - mean) * r, w2[j][e], b2[j][e])
                       : y[j][e] * r * w2[j][e];
        put_chunk<DT>(p.u + base * p.C, (oc + unsigned(col[j])) * kSize,
                      m_[j], u);
      }
    }
    if (kAhead) cur = nxt;
  }
}

}  // namespace

template <int DT>
void join_fwd_launch(const FwdArgs<TP<DT>>& a, const RowShape& r, bool layer,
                     bool has_h, int gate, bool kept, int grid,
                     hipStream_t s) {
#define FWD(L, H, G, K) \
  join_fwd_kernel<DT, kBT, kNV, L, H, G, K><<<grid, kBT, 0, s>>>(a)
  ROW_SWITCH(r, {
    JOIN_SWITCH(layer, has_h, gate, kept, FWD);
  });
#undef FWD
}

}  // namespace yams
