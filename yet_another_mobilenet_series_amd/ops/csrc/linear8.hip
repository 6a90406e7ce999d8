// FC layer whose input is kept in 8 bits: y = x w^T + bias, dx = dy w,
// dw = dy^T X with X read straight from the codes.
//
// All three are C[i, j] = sum_k A(i, k) B(j, k) with operands that lie
// either along k (x and w in the forward product) or across it (w in dx,
// both in dw).  MFMA accumulates in fp32; the values of the codes are exact
// in bf16, so dw loses nothing to the 8-bit form but the form itself.
//
// One kernel.  Four waves share a tile of C and steps of 64 along k; each
// has a quarter of the tile in its accumulators, as fragments of 32 x 32.  In
// the largest tile, 256 x 256, a wave has 128 x 128 and a SIMD holds one
// wave: such waves read 128 KB of LDS for 2048 cycles of MFMA, where eight
// waves of 128 x 64 would read 192 KB and were bound by that (16384 x 4096 x
// 4096: dw 818 us).  With one wave nothing but its own order hides latency:
//   - tiles go global -> registers -> LDS.  Registers hold step t + 1 and
//     then t + 2 while LDS holds t: a load has a step to arrive, and the
//     way through registers decodes 8-bit codes and splits fp32 weights.
//   - a step is four quarters of 16 along k.  While a quarter's MFMAs run,
//     the fragments of the next one are read, and in the first three the
//     next step is stored to the other buffer.  The only barrier of a step
//     is in its last quarter, when all fragments of the buffer have been
//     read and the next step is complete.
// 32 x 32 x 16 MFMAs and not 16 x 16 x 32: a quarter's fragments take half
// the registers of a half's, and with those the compiler kept 256
// accumulators from moving between register files.
// Operands across k lie in LDS as in memory and are read with the
// transposing LDS load, which hands a lane 4 values along k.  XOR swizzles
// spread both layouts over the banks.
//
// A long reduction with few output tiles is split; the splits leave fp32
// slabs that a second kernel adds in a fixed order.
//
// fp32 weights w go to the matrix unit as two bf16 values, their upper half
// and the rounded rest, in two passes over k that add to the same
// accumulators: what is left out is at most 2^-15 of w (rounded once they
// would be off by 2^-8, which is seen in y and dx: those are rounded to bf16,
// by 2^-8 too).  fp16 weights are exact so.  It costs the second pass: 16384
// rows, 4096 x 4096 weights in fp32: y 1125 us, dx 1160 (rounded once: 535 and
// 560), 256 rows, 1280 x 1000: 14 and 17 with the join of splits (12 and 10).
//
// Measured (16384 rows, 4096 x 4096 weights, bf16, a step after another): y
// 443 us (1241 TFLOP/s), dx 461 (1193), dw 545 (1009); the library's products,
// without codes, 357, 403 and 450.  The matrix unit is busy for 53, 50 and 41 % of the cycles of
// a SIMD's wave (4096 x 4096 x 4096), which for 39 % of them waits to issue:
// MFMAs, LDS and global accesses share the one stream of instructions, and
// dw has the decoding of the codes in it besides (27 VALU instructions for
// 4 MFMAs, against 8 in y).

#include <algorithm>
#include <cmath>

#include "rows.h"
#include "rows_engine.h"

namespace yams {

namespace {

enum { OP_BF16 = 0, OP_F32 = 1, OP_CODE = 2 };

struct Operand {
  const void* p;
  int64_t stride;
  const unsigned char* exps;
  int G;
};

// fp32, or bf16 as a bf16 model has it: no launch to convert it
struct Bias {
  const void* p;
  bool bf16;
  DEV_INLINE float at(int64_t j) const {
    return bf16 ? bf2f(static_cast<const ushort_t*>(p)[j])
                : static_cast<const float*>(p)[j];
  }
};

constexpr int TK = 64;

// eight neighbours of an operand on their way from memory to LDS
template <int KIND>
struct Staged {
  static constexpr int kSize = KIND == OP_F32 ? 4 : KIND == OP_CODE ? 1 : 2;
  Words<kSize> w;
  unsigned exponent;

  // whole chunk, `off` bytes from a base that the block shares; `eoff` is
  // its exponent's place
  DEV_INLINE void load_whole(const void* base, unsigned off,
                             const unsigned char* ebase, unsigned eoff) {
    w = load_words<kSize>(base, off, 8);
    if constexpr (KIND == OP_CODE)
      exponent = *lane_at<unsigned char>(ebase, eoff);
  }
  DEV_INLINE void load(const Operand& o, int64_t row, int64_t col, int n) {
    const char* p = static_cast<const char*>(o.p) +
                    (row * o.stride + col) * kSize;
    w = load_words<kSize>(p, 0u, n);
    if constexpr (KIND == OP_CODE)
      exponent = n > 0 ? o.exps[row * o.G + (col >> 5)] : 0u;
  }
  // PART, of fp32: 0 the upper halves (truncated, so that nothing finite
  // becomes infinite), 1 what they leave; infinities leave nothing
  template <int PART>
  DEV_INLINE uint4_t bf16() const {
    uint4_t r;
    if constexpr (KIND == OP_BF16) {
      return w;
    } else if constexpr (KIND == OP_F32 && PART == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x07060302u);
      return r;
    } else {
      float v[8];
      if constexpr (KIND == OP_F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v[e] = (w[e] & 0x7fffffffu) == 0x7f800000u
                     ? 0.f
                     : __uint_as_float(w[e]) -
                           __uint_as_float(w[e] & 0xffff0000u);
      } else {
        const float unit = exp_unit(exponent);
        dequantize4(w[0], unit, v);
        dequantize4(w[1], unit, v + 4);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[e] = unsigned(f2bf(v[2 * e])) | unsigned(f2bf(v[2 * e + 1])) << 16;
      return r;
    }
  }
};

typedef __attribute__((address_space(3))) ushort_t lds_t;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// One operand's side of a tile: W rows (i or j) by TK, staged by 256 threads.
template <int W_, int KIND, bool ACROSS>
struct Side {
  static constexpr int W = W_;
  static constexpr int kElems = W * TK;
  static constexpr int N = kElems / 8 / 256;     // chunks of a thread
  // ACROSS: [TK][W], 32-byte units XORed with the bits of k that differ
  // between the lanes of one transposing read.
  static constexpr int kUnits = W / 16;
  static constexpr int kPerRow = W / 8;          // chunks of a memory row
  static constexpr int kRows = ACROSS ? 256 / kPerRow : 32;  // of a pass

  Staged<KIND> st[N];

  static DEV_INLINE int swz(int k) {
    return ((k & 3) | ((k >> 3) & 1) << 2) & (kUnits - 1);
  }

  // chunk c of the step at k, of rows i0.. below ni, k below kend
  DEV_INLINE void load(const Operand& o, int64_t i0, int64_t ni, int64_t k,
                       int64_t kend, int c) {
    const int tid = int(threadIdx.x);
    if constexpr (!ACROSS) {
      const int64_t kc = k + (tid & 7) * 8;
      const int n = int(max(int64_t(0), min(kend - kc, int64_t(8))));
      const int64_t i = i0 + (tid >> 3) + kRows * c;
      st[c].load(o, i, kc, i < ni ? n : 0);
    } else {
      const int64_t ic = i0 + (tid % kPerRow) * 8;
      const int n = int(max(int64_t(0), min(ni - ic, int64_t(8))));
      const int64_t kk = k + tid / kPerRow + kRows * c;
      st[c].load(o, kk, ic, kk < kend ? n : 0);
    }
  }

  // FAST: steps and tiles are whole.  A chunk is the block's address (it
  // moves by scalar instructions) and the lane's offset, the same for all.
  static DEV_INLINE unsigned lane_off(const Operand& o) {
    const int tid = int(threadIdx.x);
    return (ACROSS ? unsigned(tid / kPerRow) * unsigned(o.stride) +
                         unsigned(tid % kPerRow) * 8u
                   : unsigned(tid >> 3) * unsigned(o.stride) +
                         unsigned(tid & 7) * 8u) *
           unsigned(Staged<KIND>::kSize);
  }
  static DEV_INLINE unsigned lane_eoff(const Operand& o, int64_t i0) {
    const int tid = int(threadIdx.x);
    return KIND == OP_CODE
               ? unsigned(tid / kPerRow) * unsigned(o.G) +
                     ((unsigned(i0 & 31) + unsigned(tid % kPerRow) * 8u) >> 5)
               : 0u;
  }
  DEV_INLINE void load_fast(const Operand& o, int64_t i0, int64_t k, int c,
                            unsigned off, unsigned eoff) {
    const int64_t at = ACROSS ? (k + kRows * c) * o.stride + i0
                              : (i0 + kRows * c) * o.stride + k;
    st[c].load_whole(
        static_cast<const char*>(o.p) + at * Staged<KIND>::kSize, off,
        KIND == OP_CODE ? o.exps + (k + kRows * c) * o.G + (i0 >> 5)
                        : nullptr,
        eoff);
  }

  // MASK: the step's k from z on become zero
  template <int PART, bool MASK = false>
  DEV_INLINE void store(ushort_t* lds, int c, int z = 0) const {
    const int tid = int(threadIdx.x);
    uint4_t v = st[c].template bf16<PART>();
    int at;
    if constexpr (!ACROSS) {
      const int i = (tid >> 3) + kRows * c, k = (tid & 7) * 8;
      at = i * TK + (((tid & 7) ^ (i & 7)) * 8);
      if (MASK) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] &= (k + 2 * e < z ? 0xffffu : 0u) |
                  (k + 2 * e + 1 < z ? 0xffff0000u : 0u);
      }
    } else {
      const int k = tid / kPerRow + kRows * c, ic = tid % kPerRow;
      at = k * W + (((ic >> 1) ^ swz(k)) * 16) + (ic & 1) * 8;
      if (MASK) v = k < z ? v : uint4_t(0u);
    }
    *reinterpret_cast<uint4_t*>(&lds[at]) = v;
  }

  // fragment f of the wave whose rows start at w0, quarter h of the step:
  // the lane's row is w0 + 32 f + lane % 32, its k the eight from
  // 8 (lane / 32)
  static DEV_INLINE bf16x8 frag(const ushort_t* lds, int w0, int f, int h) {
    const int lane = int(threadIdx.x) & 63;
    if constexpr (!ACROSS) {
      const int i = w0 + f * 32 + (lane & 31);
      const int c = (h * 2 + (lane >> 5)) ^ (lane & 7);
      return *reinterpret_cast<const bf16x8*>(&lds[i * TK + c * 8]);
    } else {
      // sixteen lanes read 4 k by 16 rows and get 4 k of a row each
      const int k = h * 16 + (lane >> 5) * 8 + ((lane & 15) >> 2);
      const int unit = (w0 / 16 + f * 2 + ((lane >> 4) & 1)) ^ swz(k);
      const ushort_t* p = &lds[k * W + unit * 16 + (lane & 3) * 4];
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4*)(p));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4*)(p + 4 * W));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

DEV_INLINE void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Tiles in the order that shares operands through an XCD's L2: blocks go
// round the 8 XCDs, so each XCD gets a contiguous range of tiles, which
// walks groups of 8 tile rows column by column.
DEV_INLINE void tile_of(int id, int ti, int tj, int& i, int& j) {
  const int n = ti * tj;
  const int q = n >> 3, r = n & 7, x = id & 7, s = id >> 3;
  id = x * q + min(x, r) + s;
  const int band = id / (8 * tj), first = band * 8;
  const int rows = min(8, ti - first), in = id - band * 8 * tj;
  i = first + in % rows;
  j = in / rows;
}

// 2 x 2 waves of F x F fragments
template <int F_>
struct Shape {
  static constexpr int F = F_, W = 64 * F_;
};
typedef Shape<4> Large;   // 256 x 256
typedef Shape<2> Medium;  // 128 x 128
typedef Shape<1> Small;   //  64 x  64

typedef __attribute__((ext_vector_type(16))) float f32x16;

template <typename S, int KA, bool XA, int KB, bool XB, bool OUT_BF16,
          bool FAST>
__global__ __launch_bounds__(256, S::F > 2 ? 1 : 2) void product_kernel(
    Operand A, Operand B, void* __restrict__ C, Bias bias, int64_t I,
    int64_t J, int64_t K, int ti, int tj, int64_t per_split) {
  constexpr int F = S::F;
  typedef Side<S::W, KA, XA> SA;
  typedef Side<S::W, KB, XB> SB;
  constexpr int kBuf = SA::kElems + SB::kElems;
  __shared__ __attribute__((aligned(16))) ushort_t lds[2 * kBuf];
  int bi, bj;
  tile_of(int(blockIdx.x), ti, tj, bi, bj);
  // FAST: the last tiles start early enough to be whole, and do not store
  // what the ones before them store
  const int64_t i_own = int64_t(bi) * SA::W, j_own = int64_t(bj) * SB::W;
  const int64_t i0 = FAST ? min(i_own, I - SA::W) : i_own;
  // (codes start at whole chunks: up to seven columns of the last tile are
  // behind the row, in the next one or in the bytes behind the codes)
  const int64_t j_last = KB == OP_CODE ? (J - SB::W + 7) / 8 * 8 : J - SB::W;
  const int64_t j0 = FAST ? min(j_own, j_last) : j_own;
  const int64_t k0 = int64_t(blockIdx.y) * per_split;
  const int64_t k1 = min(K, k0 + per_split);
  const int wave = int(threadIdx.x) >> 6, lane = int(threadIdx.x) & 63;
  const int wi = (wave >> 1) * 32 * F, wj = (wave & 1) * 32 * F;
  const int steps = int((max(k1 - k0, int64_t(0)) + TK - 1) / TK);

  // a fragment of C: the lane has one i and, in fours, neighbouring j
  f32x16 acc[F][F];
#pragma unroll
  for (int q = 0; q < F; ++q) {
    f32x16 v = f32x16(0.f);
    if (bias.p != nullptr) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t j =
            j0 + wj + q * 32 + (e >> 2) * 8 + (lane >> 5) * 4 + (e & 3);
        if (j < J) v[e] = bias.at(j);
      }
    }
#pragma unroll
    for (int r = 0; r < F; ++r) acc[r][q] = v;
  }

  SA a;
  SB b;
  constexpr int NC = SA::N + SB::N;  // chunks of a thread: A's, then B's
  const unsigned aoff = SA::lane_off(A), boff = SB::lane_off(B);
  const unsigned aeoff = SA::lane_eoff(A, i0), beoff = SB::lane_eoff(B, j0);
  auto load = [&](int t, int c0, int c1) {
    // FAST: the first step is the short one, so that no other has anything
    // to mask; what it has of the second becomes zero on its way to LDS.
    // Behind the last step: the last one again.
    const int64_t k =
        FAST ? max(k0, min(k1 - int64_t(steps - t) * TK, k1 - TK))
             : k0 + int64_t(t) * TK;
#pragma unroll
    for (int c = c0; c < c1; ++c) {
      if (FAST) {
        if (c < SA::N)
          a.load_fast(A, i0, k, c, aoff, aeoff);
        else
          b.load_fast(B, j0, k, c - SA::N, boff, beoff);
      } else {
        if (c < SA::N)
          a.load(A, i0, I, k, k1, c);
        else
          b.load(B, j0, J, k, k1, c - SA::N);
      }
    }
  };
  auto store = [&](auto part, int t, int c0, int c1) {
    constexpr int P = decltype(part)::value;
    ushort_t* buf = lds + (t & 1) * kBuf;
#pragma unroll
    for (int c = c0; c < c1; ++c)
      if (c < SA::N)
        a.template store<P>(buf, c);
      else
        b.template store<P>(buf + SA::kElems, c - SA::N);
  };
  auto store_first = [&](auto part) {
    constexpr int P = decltype(part)::value;
    const int z = int(k1 - k0) - (steps - 1) * TK;
#pragma unroll
    for (int c = 0; c < SA::N; ++c) a.template store<P, true>(lds, c, z);
#pragma unroll
    for (int c = 0; c < SB::N; ++c)
      b.template store<P, true>(lds + SA::kElems, c, z);
  };
  bf16x8 fa[2][F], fb[2][F];
  // fragment f of quarter h: B's, which its first MFMAs all need, then A's
  auto read = [&](int t, int h, int f) {
    const ushort_t* buf = lds + (t & 1) * kBuf;
    if (f < F)
      fb[h & 1][f] = SB::frag(buf + SA::kElems, wj, f, h);
    else
      fa[h & 1][f - F] = SA::frag(buf, wi, f - F, h);
  };
  auto multiply = [&](int h, int r) {
#pragma unroll
    for (int q = 0; q < F; ++q)
      acc[r][q] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          fb[h & 1][q], fa[h & 1][r], acc[r][q], 0, 0, 0);
  };

  // one MFMA, then what else is to be issued, so that nothing piles up in
  // front of the matrix unit
  auto interleave = [&]() {
#pragma unroll
    for (int q = 0; q < F; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
      __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // LDS write
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // global load
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  auto walk = [&](auto part) {
    load(0, 0, NC);
    if (FAST)
      store_first(part);
    else
      store(part, 0, 0, NC);
    // in the order of the loop, whose waits count on it
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      load(1, c, c + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    lds_barrier();
#pragma unroll
    for (int f = 0; f < 2 * F; ++f) read(0, 0, f);
    for (int t = 0; t < steps; ++t) {
#pragma unroll
      for (int x = 0; x < 3 * F; ++x) {
        const int h = x / F, r = x % F;
        read(t, h + 1, 2 * r);
        read(t, h + 1, 2 * r + 1);
        multiply(h, r);
        store(part, t + 1, NC * x / (3 * F), NC * (x + 1) / (3 * F));
        load(t + 2, NC * x / (3 * F), NC * (x + 1) / (3 * F));
        interleave();
      }
      multiply(3, 0);
      __builtin_amdgcn_sched_barrier(0);
      lds_barrier();
      // all of the next quarter's fragments in the first rows behind it
      constexpr int R = F > 1 ? (F + 1) / 2 : 1;
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int f = 2 * F * r / R; f < 2 * F * (r + 1) / R; ++f)
          read(t + 1, 0, f);
        if (r + 1 < F) multiply(3, r + 1);
        interleave();
      }
#pragma unroll
      for (int r = R + 1; r < F; ++r) multiply(3, r);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (steps > 0) {
    walk(std::integral_constant<int, 0>{});
    if constexpr (KB == OP_F32) {
      lds_barrier();  // the buffers are still being read
      // the first pass is not to keep what this one can find again
      asm volatile("" : "+s"(A.p), "+s"(B.p));
      walk(std::integral_constant<int, 1>{});
    }
  }

  // Out: a lane's values are fours of a row, 32 rows a wave.  They go
  // through LDS, 32 rows at a time (each wave in a part of its own), so that
  // sixteen lanes store neighbouring 16 bytes of a row.
  typedef std::conditional_t<OUT_BF16, ushort_t, float> Out;
  constexpr int kV = 16 / int(sizeof(Out));          // values of a store
  constexpr int kRow = 32 * F + 16 / int(sizeof(Out));  // padded
  static_assert(4 * 32 * kRow * sizeof(Out) <= 2 * kBuf * sizeof(ushort_t),
                "the way out has to fit into the buffers");
  Out* const box = reinterpret_cast<Out*>(lds) + wave * 32 * kRow;
  Out* const out = static_cast<Out*>(C) + int64_t(blockIdx.y) * I * J;
  lds_barrier();  // the buffers are still being read
#pragma unroll
  for (int r = 0; r < F; ++r) {
#pragma unroll
    for (int q = 0; q < F; ++q)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = (lane & 31) * kRow + q * 32 + g * 8 + (lane >> 5) * 4;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[r][q][g * 4 + e];
        if constexpr (OUT_BF16)
          *reinterpret_cast<uint2_t*>(&box[at]) = uint2_t{
              unsigned(f2bf(v[0])) | unsigned(f2bf(v[1])) << 16,
              unsigned(f2bf(v[2])) | unsigned(f2bf(v[3])) << 16};
        else
          *reinterpret_cast<float4_t*>(&box[at]) =
              float4_t{v[0], v[1], v[2], v[3]};
      }
    // the wave's own stores and loads: in order, no barrier
    constexpr int kLanes = 32 * F / kV;  // of a row
    constexpr int kRows = 64 / kLanes;   // of a pass
#pragma unroll
    for (int p = 0; p < 32 / kRows; ++p) {
      const int row = p * kRows + lane / kLanes, c = lane % kLanes * kV;
      const uint4_t v = *reinterpret_cast<const uint4_t*>(&box[row * kRow + c]);
      const int64_t i = i0 + wi + r * 32 + row, j = j0 + wj + c;
      int n = int(max(int64_t(0), min(J - j, int64_t(kV))));
      const int first = FAST ? int(max(int64_t(0), j_own - j)) : 0;
      if (i >= I || (FAST && i < i_own)) n = 0;
      Out* const to = out + i * J + j;
      if (n == kV && first == 0) {
        *reinterpret_cast<uint4_u2*>(to) = v;
      } else {
#pragma unroll
        for (int e = 0; e < kV; ++e)
          if (e >= first && e < n) {
            if constexpr (OUT_BF16)
              to[e] = ushort_t(v[e / 2] >> (16 * (e & 1)));
            else
              to[e] = __uint_as_float(v[e]);
          }
      }
    }
  }
}

// out = sum over splits + bias, in the type of the output
template <bool OUT_BF16>
__global__ __launch_bounds__(256) void join_splits_kernel(
    const float* __restrict__ ws, Bias bias, void* __restrict__ out,
    int64_t elems, int64_t J, int splits) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < elems;
       i += int64_t(gridDim.x) * 256) {
    float v = 0.f;
    for (int q = 0; q < splits; ++q) v += ws[q * elems + i];
    if (bias.p != nullptr) v += bias.at(i % J);
    if (OUT_BF16)
      static_cast<ushort_t*>(out)[i] = f2bf(v);
    else
      static_cast<float*>(out)[i] = v;
  }
}

// The tile and the splits of a product: the cheapest by a model of its time
// in microseconds, fitted to runs of 256..65536 rows.  A CU holds `most`
// blocks; `one` is a step of a lone block and `full` one of `most` together,
// `base` is what a block takes besides.  Measured: 4096 x 1024 rows by 16
// steps 30 / 14 / 18 (256 / 128 / 64 wide tiles), 1024 x 1024 by 16 28 / 12
// / 8, 16384 x 4096 by 64 521 / 558.  A split writes and reads an fp32 slab
// (some 4500 bytes a us) and costs another launch.
struct Tile {
  int W, most;
  double one, full, base;
};
constexpr Tile kTiles[] = {{Large::W, 1, 1.85, 1.85, 5.0},
                           {Medium::W, 2, 0.60, 1.10, 4.5},
                           {Small::W, 4, 0.33, 0.95, 3.5}};

struct Plan {
  int W, ti, tj, splits;
  bool fast;
  int64_t per;
};

// FAST: tiles and steps are whole or can be shifted so that they are
// (`loose`: codes without readable bytes behind them cannot be).  The
// largest tile exists only so: its registers have no room for checks.
// `passes` over k: two for fp32 weights.
Plan plan_of(int64_t I, int64_t J, int64_t K, int passes, bool loose) {
  Plan best{};
  double least = 0.0;
  for (const Tile& tile : kTiles) {
    for (int splits = 1; splits <= 64; splits *= 2) {
      if (splits > 1 && K / splits < 256) break;
      Plan p;
      p.W = tile.W;
      p.ti = ceil_div(I, p.W);
      p.tj = ceil_div(J, p.W);
      p.per = (K + splits - 1) / splits;
      p.per = std::max<int64_t>(TK, (p.per + TK - 1) / TK * TK);
      p.splits = int(std::max<int64_t>(1, (K + p.per - 1) / p.per));
      const int64_t last = K - (p.splits - 1) * p.per;
      p.fast = last >= TK && I >= p.W && J >= p.W && !loose;
      if (p.W == Large::W && !p.fast) continue;
      const double blocks = double(p.ti) * p.tj * p.splits;
      const double each = std::ceil(blocks / 256);  // of a CU
      const double rounds = std::ceil(blocks / (256.0 * tile.most));
      const double held = std::min<double>(each, tile.most);
      const double step =
          tile.most == 1 ? tile.one
                         : tile.one + (tile.full - tile.one) * (held - 1) /
                                          (tile.most - 1);
      double t = rounds * (tile.base + step * double(p.per / TK * passes) *
                                           (p.fast ? 1.0 : 1.5));
      if (p.splits > 1) t += 4.0 + 8.0 * I * J * p.splits / 4.5e6;
      if (best.W == 0 || t < least) {
        best = p;
        least = t;
      }
    }
  }
  return best;
}

template <typename S, bool FAST, int KA, bool XA, int KB, bool XB>
void launch(const Plan& p, Operand A, Operand B, bool bf16, void* C,
            Bias bias, int64_t I, int64_t J, int64_t K, hipStream_t s) {
  const dim3 grid(p.ti * p.tj, p.splits);
  if (bf16)
    product_kernel<S, KA, XA, KB, XB, true, FAST>
        <<<grid, 256, 0, s>>>(A, B, C, bias, I, J, K, p.ti, p.tj, p.per);
  else
    product_kernel<S, KA, XA, KB, XB, false, FAST>
        <<<grid, 256, 0, s>>>(A, B, C, bias, I, J, K, p.ti, p.tj, p.per);
}

template <int KA, bool XA, int KB, bool XB>
void product(Operand A, Operand B, int odt, void* C, Bias bias, float* ws,
             int64_t I, int64_t J, int64_t K, bool loose, hipStream_t s) {
  const Plan p = plan_of(I, J, K, KB == OP_F32 ? 2 : 1, loose);
  const bool split = p.splits > 1, bf16 = odt == DT_BF16 && !split;
  void* to = split ? ws : C;
  const Bias add = split ? Bias{} : bias;
#define LAUNCH(S, FAST) \
  launch<S, FAST, KA, XA, KB, XB>(p, A, B, bf16, to, add, I, J, K, s)
  if (p.W == Large::W)
    LAUNCH(Large, true);
  else if (p.W == Medium::W && p.fast)
    LAUNCH(Medium, true);
  else if (p.W == Medium::W)
    LAUNCH(Medium, false);
  else if (p.fast)
    LAUNCH(Small, true);
  else
    LAUNCH(Small, false);
#undef LAUNCH
  if (!split) return;
  const int64_t elems = I * J;
  const int blocks = int(std::min<int64_t>((elems + 255) / 256, 8192));
  if (odt == DT_BF16)
    join_splits_kernel<true>
        <<<blocks, 256, 0, s>>>(ws, bias, C, elems, J, p.splits);
  else
    join_splits_kernel<false>
        <<<blocks, 256, 0, s>>>(ws, bias, C, elems, J, p.splits);
}

// db: a thread sums one chunk of channels over the block's rows.  16384 x
// 4096 bf16 in 20 us, 6.6 TB/s.
template <int DT, int ODT, bool RAGGED>
__global__ __launch_bounds__(256) void row_sum_kernel(
    const TP<DT>* __restrict__ dy, int64_t stride, TP<ODT>* __restrict__ out,
    int64_t rows, int C, int TX, int64_t per, int out_stride) {
  __shared__ float red[256 * 8];
  const int tx = int(threadIdx.x) % TX, ty = int(threadIdx.x) / TX;
  const int TY = 256 / TX;
  const int c = (int(blockIdx.x) * TX + tx) * 8;
  const int n = min(8, max(0, C - c));
  const int64_t lo = int64_t(blockIdx.y) * per, hi = min(lo + per, rows);
  float s[8] = {};
  if (n > 0)
    for (int64_t r = lo + ty; r < hi; r += TY) {
      float v[8];
      take_chunk<DT, RAGGED>(dy + r * stride, c, n, C, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += v[e];
    }
#pragma unroll
  for (int e = 0; e < 8; ++e) red[e * 256 + int(threadIdx.x)] = s[e];
  __syncthreads();
  for (int k = int(threadIdx.x); k < 8 * TX; k += 256) {
    const int x = k >> 3, e = k & 7;
    float t = 0.f;
    for (int l = 0; l < TY; ++l) t += red[e * 256 + l * TX + x];
    const int col = (int(blockIdx.x) * TX + x) * 8 + e;
    if (col < C)
      out[int64_t(blockIdx.y) * out_stride + col] = Elem<ODT>::put(t);
  }
}

__global__ __launch_bounds__(256) void narrow_kernel(
    const float* __restrict__ v, ushort_t* __restrict__ out, int C) {
  const int i = int(blockIdx.x) * 256 + int(threadIdx.x);
  if (i < C) out[i] = f2bf(v[i]);
}

struct SumShape {
  int TX, gx, gy;
  int64_t per;
};

// few rows: narrow blocks that have all of them, and no second launch (256 x
// 1280: 4.2 us against 4.3 + 4.1)
SumShape sum_shape(int64_t rows, int C) {
  SumShape b;
  const int chunks = ceil_div(C, 8);
  b.TX = 4;
  if (rows <= 16 * 256 / b.TX && chunks / b.TX < kMaxBlocks) {
    b.gx = ceil_div(chunks, b.TX);
    b.gy = 1;
    b.per = rows;
    return b;
  }
  while (b.TX < 64 && b.TX < chunks) b.TX *= 2;
  b.gx = ceil_div(chunks, b.TX);
  const int TY = 256 / b.TX;
  const int64_t want = std::max<int64_t>(1, 1024 / b.gx);
  const int64_t most = std::max<int64_t>(1, rows / (8 * TY));
  b.gy = int(std::min(want, most));
  b.per = (rows + b.gy - 1) / b.gy;
  b.gy = int((rows + b.per - 1) / b.per);
  return b;
}

Operand operand(RowsDesc r) { return {r.p, r.stride, nullptr, 0}; }

}  // namespace

int64_t linear8_ws(int64_t rows, int64_t cols, int64_t depth, int wdt,
                   bool loose) {
  if (rows == 0 || cols == 0 || depth == 0) return 0;
  const int splits =
      plan_of(rows, cols, depth, wdt == DT_F32 ? 2 : 1, loose).splits;
  return splits > 1 ? splits * rows * cols : 0;
}

// codes of a width that is no multiple of 8 are read up to seven behind a row
bool linear8_loose(int64_t K, bool padded) { return K % 8 != 0 && !padded; }

void linear8_fwd(RowsDesc x, int wdt, RowsDesc w, int bdt, const void* b,
                 void* y, float* ws, int64_t M, int N, int K, hipStream_t s) {
  if (M == 0 || N == 0) return;
  const Bias bias{b, bdt == DT_BF16};
  if (wdt == DT_F32)
    product<OP_BF16, false, OP_F32, false>(operand(x), operand(w), DT_BF16, y,
                                           bias, ws, M, N, K, false, s);
  else
    product<OP_BF16, false, OP_BF16, false>(operand(x), operand(w), DT_BF16,
                                            y, bias, ws, M, N, K, false, s);
}

void linear8_dgrad(RowsDesc dy, int wdt, RowsDesc w, void* dx, float* ws,
                   int64_t M, int N, int K, hipStream_t s) {
  if (M == 0 || K == 0) return;
  if (wdt == DT_F32)
    product<OP_BF16, false, OP_F32, true>(operand(dy), operand(w), DT_BF16,
                                          dx, Bias{}, ws, M, K, N, false, s);
  else
    product<OP_BF16, false, OP_BF16, true>(operand(dy), operand(w), DT_BF16,
                                           dx, Bias{}, ws, M, K, N, false, s);
}

void linear8_wgrad(RowsDesc dy, Kept x, bool padded, int odt, void* dw,
                   float* ws, int64_t M, int N, int K, hipStream_t s) {
  if (N == 0 || K == 0) return;
  Operand b{x.codes, K, x.exps, ceil_div(K, kGroup)};
  product<OP_BF16, true, OP_CODE, true>(operand(dy), b, odt, dw, Bias{}, ws,
                                        N, K, M, linear8_loose(K, padded), s);
}

int64_t row_sum_ws(int64_t rows, int C) {
  if (rows == 0) return 0;
  const SumShape b = sum_shape(rows, C);
  // (and the sums themselves, before they are narrowed)
  return b.gy == 1 ? 0 : int64_t(b.gy + 1) * ((C + 3) / 4 * 4);
}

void row_sum(int dt, RowsDesc dy, int odt, void* db, float* ws, int64_t rows,
             int C, hipStream_t s) {
  if (rows == 0 || C == 0) return;
  const SumShape b = sum_shape(rows, C);
  const int stride = (C + 3) / 4 * 4;
  const bool bf16 = odt == DT_BF16;
  float* const sums = static_cast<float*>(db);
  const dim3 grid(b.gx, b.gy);
  DT_SWITCH(dt, RAGGED_SWITCH(C, {
    auto* p = static_cast<const TP<kDT>*>(dy.p);
    if (b.gy == 1 && bf16)
      row_sum_kernel<kDT, DT_BF16, kRagged><<<grid, 256, 0, s>>>(
          p, dy.stride, static_cast<ushort_t*>(db), rows, C, b.TX, b.per, 0);
    else
      row_sum_kernel<kDT, DT_F32, kRagged><<<grid, 256, 0, s>>>(
          p, dy.stride, b.gy == 1 ? sums : ws, rows, C, b.TX, b.per, stride);
  }));
  if (b.gy == 1) return;
  float* const to = bf16 ? ws + int64_t(b.gy) * stride : sums;
  slab_reduce(ws, to, stride, b.gy, s);
  if (bf16)
    narrow_kernel<<<ceil_div(C, 256), 256, 0, s>>>(
        to, static_cast<ushort_t*>(db), C);
}

}  // namespace yams
