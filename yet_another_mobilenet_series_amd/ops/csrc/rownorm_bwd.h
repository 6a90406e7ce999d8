// Backward of the norms over channels and of the joins between residual
// blocks (rownorm_fwd.h has the forward):
//
//   n = w hh + b, hh = (h - mean) r;   y = x + s a(g) n;   u = w2 yh + b2
//   dY = dy + N2'(du),  N'(d) = r (d w - hh mean(d w hh) - mean(d w))
//   dx = dY;  dn = dY s a(g);  dh = N1'(dn);  dg = dY s a'(g) n
//   dscale = sum dY a(g) n;  dw = sum dn hh;  db = sum dn
//   dw2 = sum du yh;  db2 = sum du          (the mean(d w) term: LAYER only)
//
// w, b and s do not depend on the row, so three of the sums over rows are
// two: with T = sum dY a(g) hh and B = sum dY a(g),
//   dscale = w T + b B;  dw = s T;  db = s B.
//
// y is not kept: it is computed again from x, h and g, unrounded, which
// costs what reading it would.  The statistics are computed again too,
// from what the row holds here; with inputs kept in 8 bits the result is
// therefore exactly the gradient at the values the codes stand for.
//
// One pass, bound by memory.  The sums over rows stay in registers while a
// block walks its rows; a block leaves one row of partial sums for each
// parameter, and slab_reduce adds them in a fixed order: no atomics, the
// same bits every time.  A gate shared by a run of rows is summed the same
// way: a block has whole runs, or, where there are fewer runs than blocks,
// a part of one run.
//
// Measured (bf16, kept in 8 bits): rms norm of 32768 x 2048 in 78 us, 4.3
// TB/s; join of 16384 x 4096 with a gate and the next norm 226 us, 3.9 TB/s.
// What is missing to the memory's rate: the registers hold a row, the next
// one and the sums, so that a SIMD has four waves, and each row waits for
// two or three sums over its team.

#pragma once

#include <algorithm>

#include "rownorm.h"

namespace yams {

namespace {

// Per-channel parameters: read from LDS for every row where they fit (the
// registers they would take are worth a wave per SIMD), laid out so that a
// wave's 16-byte reads are contiguous.  They are zero in channels behind the
// last one, which keeps those out of every sum over a row but that of the
// squares.  Four of 16384 channels do not fit; that block reads global
// memory (L2).
template <int BT, int NV>
struct Params {
  static constexpr bool kLds = BT * NV <= 1024;
  static constexpr int kSlots = kLds && NV > 0 ? BT * NV : 1;  // chunks
  float4_t v[kSlots * 2];

  DEV_INLINE void fill(const float* p, int C, int TPR, float fallback,
                       float factor) {
    if constexpr (kLds) {
      for (int k = int(threadIdx.x); k < TPR * NV; k += BT) {
        const int n = min(8, max(0, C - k * 8));
        float q[8];
        if (p != nullptr) {
          load_chunk<DT_F32>(p + k * 8, n, q);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] = e < n ? fallback : 0.f;
        }
        v[k] = float4_t{q[0], q[1], q[2], q[3]} * factor;
        v[kSlots + k] = float4_t{q[4], q[5], q[6], q[7]} * factor;
      }
    }
  }
  DEV_INLINE void get(const float* p, int chunk, int n, float fallback,
                      float factor, float* q) const {
    if constexpr (kLds) {
      const float4_t a = v[chunk], b = v[kSlots + chunk];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        q[e] = a[e];
        q[4 + e] = b[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = e < n ? fallback : 0.f;
      if (p != nullptr) load_chunk<DT_F32>(p + chunk * 8, n, q);
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] *= factor;
    }
  }
};

// What a thread loads of a row, before any of it is decoded.
template <int DT, int NV, bool HAS_H, int GATE, bool KEPT>
struct RowRaw {
  RawChunk<DT, KEPT> h[HAS_H ? NV : 1], g[GATE == GATE_FULL ? NV : 1], x[NV];
  RawChunk<DT, false> dy[NV], du[NV];

  // f(chunk, its channels) for all of them
  template <typename Fn>
  DEV_INLINE void each(Fn f, const int (&n)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (HAS_H) f(h[j], n[j]);
      if constexpr (GATE == GATE_FULL) f(g[j], n[j]);
      f(x[j], n[j]);
      f(dy[j], n[j]);
      f(du[j], n[j]);
    }
  }
};

// Waves per SIMD to fit the registers to.  Four (128 registers) pay where
// they cost few spills: rms rows of 16 bits (16384 x 4096 with a gate, kept
// in 8 bits: 305 -> 247 us), and any row of 512 threads, of which a CU
// otherwise holds a single one (LAYER, the same rows: 610 -> 561); a norm
// alone fits anyway.  Elsewhere they lose (LAYER, 65536 x 1024: 294 -> 344 us,
// without a gate 205 -> 253; fp32, 32768 x 2048: 463 -> 724).  Three hold a
// gate shared by rows to 168 registers (98000 x 333 fp16: 297 -> 200 us, with
// what is not kept there); fp32 would spill (2000 x 800: 31 -> 40).
template <int DT, int BT, bool LAYER, bool HAS_H, int GATE>
constexpr int bwd_waves() {
  if (BT >= 512 || !HAS_H) return 4;
  if (!LAYER && DT != DT_F32 && GATE != GATE_GROUP) return 4;
  return DT == DT_F32 ? 2 : 3;
}

template <int DT, int BT, int NV, bool LAYER, bool HAS_H, int GATE, bool KEPT>
__global__ __launch_bounds__(BT, (bwd_waves<DT, BT, LAYER, HAS_H, GATE>())) void
join_bwd_kernel(
    BwdArgs<TP<DT>> p) {
  constexpr unsigned kSize = unsigned(sizeof(TP<DT>));
  constexpr unsigned kIn = KEPT ? 1u : kSize;  // bytes of h, x, g in memory
  constexpr bool SHARED = GATE == GATE_GROUP;
  __shared__ float red[6 * (BT / 64)];
  // sums over the teams of a block; a block of one team has none
  __shared__ float fold[BT <= 256 ? BT * 8 : 1];
  __shared__ Params<BT, HAS_H ? NV : 0> pw, ps, pb;
  __shared__ Params<BT, NV> pw2;
  const bool next = !HAS_H || p.next;  // without h there is nothing else
  int turn = 0;
  const int TPR = p.TPR, RPB = BT / TPR;
  const int t = int(threadIdx.x) & (TPR - 1);
  const unsigned team = threadIdx.x / unsigned(TPR);
  const Chunks<NV> chunks(p.C, t, TPR);
  const auto &n = chunks.n, &col = chunks.col;
  float a_t[NV][8] = {}, a_b[NV][8] = {};  // T and B
  float a_w2[NV][8] = {}, a_b2[NV][8] = {};
  if constexpr (HAS_H) {
    pw.fill(p.w, p.C, TPR, 1.f, 1.f);
    ps.fill(p.scale, p.C, TPR, 1.f, p.alpha);
    if (LAYER) pb.fill(p.b, p.C, TPR, 0.f, 1.f);
  }
  if (next) pw2.fill(p.w2, p.C, TPR, 1.f, 1.f);
  __syncthreads();

  // byte offsets of this lane from the first row of the block's step
  const unsigned oh = team * unsigned(p.hs) * kSize;
  const unsigned ox = team * unsigned(p.xs) * kSize;
  const unsigned og = team * unsigned(p.gs) * kSize;
  const unsigned ody = team * unsigned(p.dys) * kSize;
  const unsigned odu = team * unsigned(p.dus) * kSize;
  const unsigned oc = team * unsigned(p.C), oe = team * unsigned(p.G);

  // Whether du and w2 are read again where they are needed again, instead of
  // staying in registers over a sum: where rows of 512 threads would spill
  // (LAYER, 16384 x 4096: 508 -> 432 us).
  constexpr bool AGAIN = LAYER && BT >= 512;
  typedef RowRaw<DT, NV, HAS_H, GATE, KEPT> Raw;
  // `short_n`: 0..8 elements of a short row, or -1
  auto load = [&](RawChunk<DT, KEPT>& q, const TP<DT>* from, int64_t stride,
                  const Kept& k, int64_t row, unsigned off, unsigned team_c,
                  unsigned team_e, int j, int short_n) {
    const char* base;
    if constexpr (KEPT) {
      base = reinterpret_cast<const char*>(k.codes + row * p.C);
      off = team_c;
      q.load_exponent(k.exps + row * p.G, team_e + chunks.group[j]);
    } else {
      base = reinterpret_cast<const char*>(from + row * stride);
    }
    if (short_n < 0)
      q.load(base, off + chunks.from[j] * kIn);
    else
      q.load_short(base, off, short_n);
  };
  // Rows of a team that has none are the first team's.
  auto load_rows = [&](Raw& q, int64_t base, bool live, bool shorts) {
    const unsigned tc = live ? oc : 0u, te = live ? oe : 0u;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int nn = shorts ? (live ? n[j] : 0) : -1;
      const unsigned c = chunks.from[j] * kSize;
      if constexpr (HAS_H) {
        load(q.h[j], p.h, p.hs, p.hk, base, live ? oh : 0u, tc, te, j, nn);
        if constexpr (GATE == GATE_FULL)
          load(q.g[j], p.g, p.gs, p.gk, base, live ? og : 0u, tc, te, j, nn);
      }
      auto load_d = [&](RawChunk<DT, false>& d, const TP<DT>* from,
                        int64_t stride, unsigned off) {
        const TP<DT>* row = from + base * stride;
        off = live ? off : 0u;
        if (nn < 0)
          d.load(row, off + c);
        else
          d.load_short(row, off, nn);
      };
      if (next) {
        load(q.x[j], p.x, p.xs, p.xk, base, live ? ox : 0u, tc, te, j, nn);
        load_d(q.du[j], p.du, p.dus, odu);
      }
      if (p.dy != nullptr) load_d(q.dy[j], p.dy, p.dys, ody);
    }
  };
  auto load_row = [&](Raw& q, int64_t base, int64_t hi) {
    if (base >= hi) return;
    const bool live = base + team < hi;
    if (p.read == READ_SHORT)
      load_rows(q, base, live, true);
    else
      load_rows(q, base, live, false);
  };

  // adds a per-channel sum over the teams of the block that may have had a
  // row; the result is in the first team's registers (team by team: eight
  // values in flight, and not registers for all of them)
  const int teams = int(min(p.part_rows, int64_t(RPB)));
  auto over_teams = [&](float (&v)[NV][8]) {
    if constexpr (BT <= 256) {
      if (teams > 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          __syncthreads();
#pragma unroll
          for (int e = 0; e < 8; ++e)
            fold[e * BT + int(threadIdx.x)] = v[j][e];
          __syncthreads();
          if (team == 0) {
#pragma unroll 1
            for (int l = 1; l < teams; ++l)
#pragma unroll
              for (int e = 0; e < 8; ++e)
                v[j][e] += fold[e * BT + l * TPR + t];
          }
        }
      }
    }
  };

  // zeros behind the last channel: it has code 0 there, which is NaN in a
  // group with a non-finite value
  auto end_row = [&](float (&v)[NV][8]) {
    if (KEPT && p.read != READ_WHOLE) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = e < n[j] ? v[j][e] : 0.f;
    }
  };

  // this block's runs of rows
  int64_t run0, run1;
  int part = 0;
  if (p.parts > 1) {
    run0 = int64_t(blockIdx.x / unsigned(p.parts));
    run1 = run0 + 1;
    part = int(blockIdx.x % unsigned(p.parts));
  } else {
    run0 = p.groups * int64_t(blockIdx.x) / int64_t(gridDim.x);
    run1 = p.groups * int64_t(blockIdx.x + 1) / int64_t(gridDim.x);
  }

  for (int64_t run = run0; run < run1; ++run) {
    const int64_t lo = run * p.group_rows + part * p.part_rows;
    const int64_t hi = min(lo + p.part_rows, (run + 1) * p.group_rows);
    float a_g[SHARED ? NV : 1][8] = {};
    float gs[SHARED ? NV : 1][8];  // the run's gates
    if constexpr (SHARED) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        RawChunk<DT, KEPT> q;
        load(q, p.g, p.gs, p.gk, run, 0u, 0u, 0u, j,
             p.read == READ_SHORT ? n[j] : -1);
        if (p.read == READ_RAGGED) q.drop(n[j]);
        q.blank(n[j]);
        q.decode(gs[j]);
      }
      if constexpr (KEPT) end_row(gs);
      gate_prepare<DT, NV>(gs, p.gate_act);
    }
    Raw cur;
    load_row(cur, lo, hi);
    for (int64_t base = lo; base < hi; base += RPB) {
      // the next row is on its way while this one is worked on
      Raw nxt;
      load_row(nxt, base + RPB, hi);
      if constexpr (SHARED) {
        // what follows from the run's gates and from the parameters is not
        // to be kept in registers from row to row
        asm volatile("" ::: "memory");
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(gs[j][e]));
      }
      const bool live = base + team < hi;
      // A team without a row has zeros, and r = ry = 0: it adds nothing (its
      // shared gates are the run's, and may be infinite: they are left out).
      int m_[NV];  // channels to store
      float dY[NV][8], x[NV][8], h[NV][8], g[NV][8];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        m_[j] = live ? n[j] : 0;
        if (p.dy == nullptr) cur.dy[j].blank(0);
      }
      if (p.read == READ_RAGGED) cur.each([](auto& q, int n) { q.drop(n); }, n);
      cur.each([](auto& q, int n) { q.blank(n); }, m_);
      float r = 1.f;
      if constexpr (HAS_H) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          cur.h[j].decode(h[j]);
          if constexpr (GATE == GATE_FULL) cur.g[j].decode(g[j]);
        }
        if (KEPT && p.read != READ_WHOLE) {
          end_row(h);
          if constexpr (GATE == GATE_FULL) end_row(g);
        }
        if constexpr (GATE == GATE_FULL) gate_prepare<DT, NV>(g, p.gate_act);
        float mean = 0.f;
        if (p.post)
          row_stats<NV, BT, LAYER>(h, n, TPR, p.inv_c, p.eps, red, turn,
                                   mean, r);
        r = live ? r : 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e)  // h becomes hh
            h[j][e] = (LAYER ? h[j][e] - mean : h[j][e]) * r;
      }
      if (next) {
#pragma unroll
        for (int j = 0; j < NV; ++j) cur.x[j].decode(x[j]);
        end_row(x);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if constexpr (HAS_H) {
            float w[8], s[8], b[8] = {};
            pw.get(p.w, t + j * TPR, n[j], 1.f, 1.f, w);
            ps.get(p.scale, t + j * TPR, n[j], 1.f, p.alpha, s);
            if (LAYER) pb.get(p.b, t + j * TPR, n[j], 0.f, 1.f, b);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float v =
                  LAYER ? fmaf(h[j][e], w[e], b[e]) : h[j][e] * w[e];
              const float sa =
                  GATE == GATE_NONE
                      ? s[e]
                      : s[e] * gate_value(SHARED ? gs[SHARED ? j : 0][e]
                                                 : g[j][e],
                                          p.gate_act);
              x[j][e] = fmaf(v, sa, x[j][e]);
            }
          }
        }
        // the statistics of y and what its gradient needs of the row in one
        // reduction (after that of the mean): with c = y - mean, g = du w2
        //   mean(g yh) = ry mean(g c)
        float mean = 0.f;
        if (LAYER) {
          float q[1] = {0.f};
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) q[0] += x[j][e];
          team_sum<1, BT>(q, TPR, red, turn);
          mean = q[0] * p.inv_c;
        }
        float u[NV][8], w2[NV][8];
        float q[LAYER ? 3 : 2] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          pw2.get(p.w2, t + j * TPR, n[j], 1.f, 1.f, w2[j]);
          cur.du[j].decode(u[j]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (LAYER) x[j][e] = e < n[j] ? x[j][e] - mean : 0.f;
            const float g2 = u[j][e] * w2[j][e];
            q[0] = fmaf(x[j][e], x[j][e], q[0]);
            q[1] = fmaf(g2, x[j][e], q[1]);
            if constexpr (LAYER) q[2] += g2;
          }
        }
        team_sum<LAYER ? 3 : 2, BT>(q, TPR, red, turn);
        float ry = rsqrtf(fmaf(q[0], p.inv_c, p.eps));
        ry = live ? ry : 0.f;
        const float m0 = ry * q[1] * p.inv_c;
        const float m1 = LAYER ? q[LAYER ? 2 : 0] * p.inv_c : 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          cur.dy[j].decode(dY[j]);
          if (AGAIN) {
            auto q = cur.du[j];
            asm volatile("" : "+v"(q.w));
            q.decode(u[j]);
            pw2.get(p.w2, t + j * TPR, n[j], 1.f, 1.f, w2[j]);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float yh = x[j][e] * ry;
            a_w2[j][e] = fmaf(u[j][e], yh, a_w2[j][e]);
            if (LAYER) a_b2[j][e] += u[j][e];
            float v = fmaf(-yh, m0, u[j][e] * w2[j][e]);
            if (LAYER) v -= m1;
            dY[j][e] = fmaf(ry, v, dY[j][e]);
          }
        }
      }
      if (!next) {
#pragma unroll
        for (int j = 0; j < NV; ++j) cur.dy[j].decode(dY[j]);
      }
      if (p.dx != nullptr) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          put_chunk<DT>(p.dx + base * p.C, (oc + unsigned(col[j])) * kSize,
                        m_[j], dY[j]);
      }
      if constexpr (HAS_H) {
        // dY -> dn w, g -> dg
        float m[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float w[8], s[8], b[8] = {};
          pw.get(p.w, t + j * TPR, n[j], 1.f, 1.f, w);
          ps.get(p.scale, t + j * TPR, n[j], 1.f, p.alpha, s);
          if (LAYER) pb.get(p.b, t + j * TPR, n[j], 0.f, 1.f, b);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float a = 1.f, da = 0.f;
            if (GATE != GATE_NONE) {
              const float v = SHARED ? gs[SHARED ? j : 0][e] : g[j][e];
              a = gate_value(v, p.gate_act);
              da = gate_slope(v, p.gate_act);
            }
            const float d = dY[j][e];
            const float nn =
                LAYER ? fmaf(h[j][e], w[e], b[e]) : h[j][e] * w[e];
            if (SHARED) a = live ? a : 0.f;
            const float ga = GATE != GATE_NONE ? d * a : d;
            if (GATE != GATE_NONE) g[j][e] = d * s[e] * da * nn;
            a_t[j][e] = fmaf(ga, h[j][e], a_t[j][e]);
            if (LAYER) a_b[j][e] += ga;
            const float dw = ga * s[e] * w[e];
            dY[j][e] = dw;
            m[0] = fmaf(dw, h[j][e], m[0]);
            if (LAYER) m[1] += dw;
          }
        }
        if constexpr (SHARED) {
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) a_g[j][e] += g[j][e];
        } else if constexpr (GATE == GATE_FULL) {
          if (p.dg != nullptr) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
              put_chunk<DT>(p.dg + base * p.C,
                            (oc + unsigned(col[j])) * kSize, m_[j], g[j]);
          }
        }
        if (p.post) {
          if (LAYER) {
            team_sum<2, BT>(m, TPR, red, turn);
          } else {
            float m0[1] = {m[0]};
            team_sum<1, BT>(m0, TPR, red, turn);
            m[0] = m0[0];
          }
          m[0] *= p.inv_c;
          m[1] *= p.inv_c;
        } else {
          m[0] = m[1] = 0.f;
        }
        if (p.dh != nullptr) {
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float v = fmaf(-h[j][e], m[0], dY[j][e]);
              o[e] = r * (LAYER ? v - m[1] : v);
            }
            put_chunk<DT>(p.dh + base * p.C, (oc + unsigned(col[j])) * kSize,
                          m_[j], o);
          }
        }
      }
      cur = nxt;
    }
    if constexpr (SHARED) {
      if (p.dg != nullptr) {
        over_teams(a_g);
        if (team == 0) {
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            if (p.parts > 1)
              put_chunk<DT_F32>(
                  p.wsg + (int64_t(part) * p.groups + run) * p.C,
                  unsigned(col[j]) * 4u, n[j], a_g[j]);
            else
              put_chunk<DT>(p.dg + run * p.C, unsigned(col[j]) * kSize, n[j],
                            a_g[j]);
          }
        }
      }
    }
  }

  int k = 0;
  auto store = [&](const float (&v)[NV][8]) {
    if (team == 0) {
      float* to = p.ws + (int64_t(blockIdx.x) * __popc(p.want) + k) * p.Cp;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        put_chunk<DT_F32>(to, unsigned(col[j]) * 4u, n[j], v[j]);
    }
    ++k;
  };
  if constexpr (HAS_H) {
    if (p.want & 7u) {
      over_teams(a_t);
      if (LAYER) over_teams(a_b);
      float ds[NV][8], dw[NV][8], db[NV][8];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float w[8], s[8], b[8] = {};
        pw.get(p.w, t + j * TPR, n[j], 1.f, 1.f, w);
        ps.get(p.scale, t + j * TPR, n[j], 1.f, p.alpha, s);
        if (LAYER) pb.get(p.b, t + j * TPR, n[j], 0.f, 1.f, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // alpha is part of s, but not of what scale multiplies
          ds[j][e] = (LAYER ? fmaf(b[e], a_b[j][e], w[e] * a_t[j][e])
                            : w[e] * a_t[j][e]) * p.alpha;
          dw[j][e] = s[e] * a_t[j][e];
          db[j][e] = s[e] * a_b[j][e];
        }
      }
      if (p.want & 1u) store(ds);
      if (p.want & 2u) store(dw);
      if (p.want & 4u) store(db);
    }
  }
  if (p.want & 8u) {
    over_teams(a_w2);
    store(a_w2);
  }
  if (LAYER && (p.want & 16u)) {
    over_teams(a_b2);
    store(a_b2);
  }
}

// dg[run, c] = sum over the parts of a run, in the type of the gate
template <int DT>
__global__ __launch_bounds__(256) void gate_fold_kernel(
    const float* __restrict__ ws, TP<DT>* __restrict__ dg, int64_t elems,
    int parts) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < elems;
       i += int64_t(gridDim.x) * 256) {
    float v = 0.f;
    for (int q = 0; q < parts; ++q) v += ws[q * elems + i];
    dg[i] = Elem<DT>::put(v);
  }
}

}  // namespace

template <int DT>
void join_bwd_launch(const BwdArgs<TP<DT>>& a, const RowShape& r, bool layer,
                     bool has_h, int gate, bool kept, int grid,
                     hipStream_t s) {
#define BWD(L, H, G, K) \
  join_bwd_kernel<DT, kBT, kNV, L, H, G, K><<<grid, kBT, 0, s>>>(a)
  ROW_SWITCH(r, {
    JOIN_SWITCH(layer, has_h, gate, kept, BWD);
  });
#undef BWD
}

template <int DT>
void gate_fold_launch(const float* ws, TP<DT>* dg, int64_t elems, int parts,
                      hipStream_t s) {
  const int grid = int(std::min<int64_t>((elems + 255) / 256, 2048));
  gate_fold_kernel<DT><<<grid, 256, 0, s>>>(ws, dg, elems, parts);
}

}  // namespace yams
