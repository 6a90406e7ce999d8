// What the forward and the backward kernels of the row norms share: how a
// row is spread over threads, and sums over a row.
//
// A team of TPR threads (a power of two, 4..1024) holds a row in
// registers: thread t has the 8-channel chunks t, t + TPR, ... (NV of
// them), so a wave reads 1 KB of neighbouring bf16 at a time and a group of
// 32 channels is a quad of lanes.  Small rows share a wave, large ones
// take several, and a block of BT threads walks rows until none are left.
// The per-channel parameters are in registers in the forward pass, in LDS (or
// L2) in the backward pass.
#pragma once

#include "rows.h"
#include "rows_engine.h"

namespace yams {

struct RowShape {
  int BT, NV, TPR;
};

// One chunk a thread (NV = 1) up to 8192 channels: the fewer registers a
// row takes of a thread, the more waves hide its latency.
inline RowShape row_shape(int C) {
  RowShape r;
  const int chunks = ceil_div(C, 8);
  r.NV = chunks > 1024 ? 2 : 1;
  r.TPR = 4;
  while (r.TPR * r.NV < chunks) r.TPR *= 2;
  r.BT = r.TPR <= 256 ? 256 : r.TPR;
  return r;
}

// A lane's chunks of a row: columns, how many of them are there, and where
// they are read.
template <int NV>
struct Chunks {
  int n[NV], col[NV];
  unsigned from[NV], group[NV];  // the columns read, their exponent

  DEV_INLINE Chunks(int C, int t, int TPR) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      col[j] = (t + j * TPR) * 8;
      n[j] = min(8, max(0, C - col[j]));
      from[j] = unsigned(max(0, min(col[j], C - 8)));
      group[j] = unsigned(min(col[j], C - 1)) >> 5;
    }
  }
};

// v + the value of the lane `1 << STEP` away (in the sense of a butterfly:
// after all steps up to log2(TPR) - 1 every lane of a team has its sum).
// DPP and lane swaps: no trip through LDS.
template <int STEP>
DEV_INLINE float lane_add(float v) {
  const int i = __float_as_int(v);
  if constexpr (STEP == 0)
    return v + __int_as_float(
                   __builtin_amdgcn_mov_dpp(i, 0xB1, 0xf, 0xf, true));
  else if constexpr (STEP == 1)
    return v + __int_as_float(
                   __builtin_amdgcn_mov_dpp(i, 0x4E, 0xf, 0xf, true));
  else if constexpr (STEP == 2)  // mirror of 8: the quads are uniform
    return v + __int_as_float(
                   __builtin_amdgcn_mov_dpp(i, 0x141, 0xf, 0xf, true));
  else if constexpr (STEP == 3)  // mirror of 16
    return v + __int_as_float(
                   __builtin_amdgcn_mov_dpp(i, 0x140, 0xf, 0xf, true));
  else if constexpr (STEP == 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(unsigned(i), unsigned(i),
                                                    false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(unsigned(i), unsigned(i),
                                                    false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
}

// Sums of N values over a team, the same in all of its threads.  Every
// thread of the block calls it; `red` holds two buffers used in turn, so
// one barrier is enough: who writes a buffer again has passed the barrier
// of the other one, and so has everybody who read it.
template <int N, int BT>
DEV_INLINE void team_sum(float (&v)[N], int TPR, float* red, int& turn) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = lane_add<1>(lane_add<0>(v[k]));
  if (TPR > 4) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = lane_add<2>(v[k]);
  }
  if (TPR > 8) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = lane_add<3>(v[k]);
  }
  if (TPR > 16) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = lane_add<4>(v[k]);
  }
  if (TPR > 32) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = lane_add<5>(v[k]);
  }
  if (TPR > 64) {
    constexpr int W = BT / 64;
    float* r = red + turn * (3 * W);
    turn ^= 1;
    const int wave = int(threadIdx.x) >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) r[k * W + wave] = v[k];
    }
    __syncthreads();
    const int per = TPR >> 6, first = wave & ~(per - 1);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float t = 0.f;
      for (int i = 0; i < per; ++i) t += r[k * W + first + i];
      v[k] = t;
    }
  }
}

// The statistics of a row held as NV chunks: mean (0 without LAYER) and
// 1 / sqrt(mean square + eps).  The square sum is taken about the mean, in
// a second pass over the registers: no cancellation at large means.
template <int NV, int BT, bool LAYER>
DEV_INLINE void row_stats(const float (&v)[NV][8], const int (&n)[NV],
                          int TPR, float inv_c, float eps, float* red,
                          int& turn, float& mean, float& rstd) {
  float t[1] = {0.f};
  mean = 0.f;
  if (LAYER) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) t[0] += v[j][e];
    team_sum<1, BT>(t, TPR, red, turn);
    mean = t[0] * inv_c;
    t[0] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = LAYER ? (e < n[j] ? v[j][e] - mean : 0.f) : v[j][e];
      t[0] = fmaf(c, c, t[0]);
    }
  team_sum<1, BT>(t, TPR, red, turn);
  rstd = rsqrtf(fmaf(t[0], inv_c, eps));
}

// Gates.  prepare: what a lane keeps of a gate (sigmoid itself, since its
// exponential is the expensive part; the other activations' input).
// value: a(g);  slope: a'(g).  The activation is the same for a launch.
//
// 1 / (1 + 2^t), t = -g log2(e).  v_exp and v_rcp are good to an ulp of fp32;
// rounding t costs |t| / 2 ulps of 2^t, up to 2^-17 of it where that counts,
// which results of 16 bits do not show.  In fp32 rows 2^t is corrected by what
// the rounding of t leaves out (where it is neither 0 nor infinite).
template <int DT, int NV>
DEV_INLINE void gate_prepare(float (&g)[NV][8], int act) {
  constexpr float kLog2e = 1.44269502f;      // log2(e) to fp32,
  constexpr float kLog2eLow = 1.92596299e-8f;  // and what is left
  constexpr float kLn2 = 0.693147181f;
  if (act == GATE_SIGMOID) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float t = g[j][e] * -kLog2e;
        float p = __builtin_amdgcn_exp2f(t);
        if (DT == DT_F32) {
          const float low = fmaf(g[j][e], -kLog2eLow,
                                 fmaf(g[j][e], -kLog2e, -t));
          p = p > 0.f && p < INFINITY ? fmaf(p, low * kLn2, p) : p;
        }
        g[j][e] = __builtin_amdgcn_rcpf(1.f + p);
      }
  }
}

DEV_INLINE float gate_value(float g, int act) {
  return act == ACT_HSIGMOID ? act_fwd<ACT_HSIGMOID>(g) : g;
}

DEV_INLINE float gate_slope(float g, int act) {
  return act == GATE_SIGMOID   ? fmaf(-g, g, g)
         : act == ACT_HSIGMOID ? act_bwd<ACT_HSIGMOID>(g)
                               : 1.f;
}

// What the kernels get.  T: the rows' type.  Gates: GATE_*.
template <typename T>
struct FwdArgs {
  const T *h, *x, *g;
  int64_t hs, xs, gs;
  Kept hk, xk, gk;
  const float *w, *b, *scale, *w2, *b2;
  T *y, *u;
  int64_t rows;
  int C, G, TPR, gate_act;
  Read read;
  bool post, next;
  float eps, alpha, inv_c;
  FastDiv group;
};

template <typename T>
struct BwdArgs {
  const T *h, *x, *g, *dy, *du;
  int64_t hs, xs, gs, dys, dus;
  Kept hk, xk, gk;
  const float *w, *b, *scale, *w2;
  T *dh, *dx, *dg;
  float *ws, *wsg;  // partial sums of the parameters, of the shared gate
  int64_t rows;
  int64_t group_rows, groups, part_rows;
  int parts;
  int C, Cp, G, TPR, gate_act;
  Read read;
  bool post, next;
  unsigned want;
  float eps, alpha, inv_c;
};

// Launchers for one row type each, so that the three compile in parallel.
// has_h, gate, kept and layer choose the kernel, the shape its block.
template <int DT>
void join_fwd_launch(const FwdArgs<TP<DT>>& a, const RowShape& r, bool layer,
                     bool has_h, int gate, bool kept, int grid,
                     hipStream_t s);
template <int DT>
void join_bwd_launch(const BwdArgs<TP<DT>>& a, const RowShape& r, bool layer,
                     bool has_h, int gate, bool kept, int grid,
                     hipStream_t s);
// dg[i] = sum over the parts of a run of ws[part][i]
template <int DT>
void gate_fold_launch(const float* ws, TP<DT>* dg, int64_t elems, int parts,
                      hipStream_t s);

#define ROW_SWITCH(R, ...)                                               \
  if ((R).BT == 256 && (R).NV == 1) {                                    \
    constexpr int kBT = 256, kNV = 1;                                    \
    __VA_ARGS__;                                                         \
  } else if ((R).BT == 512 && (R).NV == 1) {                             \
    constexpr int kBT = 512, kNV = 1;                                    \
    __VA_ARGS__;                                                         \
  } else if ((R).BT == 1024 && (R).NV == 1) {                            \
    constexpr int kBT = 1024, kNV = 1;                                   \
    __VA_ARGS__;                                                         \
  } else if ((R).BT == 1024) {                                           \
    constexpr int kBT = 1024, kNV = 2;                                   \
    __VA_ARGS__;                                                         \
  } else {                                                               \
    yams_launch_fail("row shape", (R).BT, (R).NV, (R).TPR, 0);           \
  }

// K(layer, has_h, gate, kept) for the values of a launch
#define JOIN_SWITCH(LAYER, HAS_H, GATE, KEPT, K)                         \
  do {                                                                   \
    const int key = (LAYER ? 1 : 0) | (KEPT ? 2 : 0) |                   \
                    (HAS_H ? 4 + 4 * (GATE) : 0);                        \
    switch (key) {                                                       \
      case 0: K(false, false, 0, false); break;                          \
      case 1: K(true, false, 0, false); break;                           \
      case 2: K(false, false, 0, true); break;                           \
      case 3: K(true, false, 0, true); break;                            \
      case 4: K(false, true, 0, false); break;                           \
      case 5: K(true, true, 0, false); break;                            \
      case 6: K(false, true, 0, true); break;                            \
      case 7: K(true, true, 0, true); break;                             \
      case 8: K(false, true, 1, false); break;                           \
      case 9: K(true, true, 1, false); break;                            \
      case 10: K(false, true, 1, true); break;                           \
      case 11: K(true, true, 1, true); break;                            \
      case 12: K(false, true, 2, false); break;                          \
      case 13: K(true, true, 2, false); break;                           \
      case 14: K(false, true, 2, true); break;                           \
      case 15: K(true, true, 2, true); break;                            \
      default: yams_launch_fail("join", key, 0, 0, 0);                   \
    }                                                                    \
  } while (0)

}  // namespace yams
