// Device helpers of the row operators: rows of channels in bf16, fp16 or
// fp32 with any row stride and alignment, and the 8-bit form that keeps
// them for a backward pass.
//
// 8-bit form.  A row is cut into groups of 32 neighbouring channels (the
// last one may be short).  A group holds integers q, |q| <= 127, and one
// exponent byte E that stands for the unit 2^(E-127): the smallest power
// of two with max|x| <= 127 units.  value = q * unit.  A power of two
// costs up to one bit against a free scale, and buys that every value is
// exact in bf16 (q has 7 bits, bf16 8) and in fp16 (units stop at its
// smallest step 2^-24): matrix instructions and fp32 code see the same
// operand.  In the top binade of the type |q| stops at 63, so nothing
// finite comes back infinite.  E = 255 marks a group with a non-finite
// value: 255 << 23 is fp32 infinity, so codes +-1 give the infinities
// back and code 0 (NaN, and whatever was finite) gives NaN.
#pragma once

#include <type_traits>

#include "common.h"

// Products and sums are fused where this code says so and nowhere else: a
// gradient from codes has the bits of the gradient from their values, which
// the compiler's own choices (code * unit + b) would not keep.
#pragma clang fp contract(off)

namespace yams {

constexpr int kGroup = 32;  // channels that share an exponent byte

constexpr int DT_BF16 = 0, DT_F16 = 1, DT_F32 = 2;

// Unaligned 8-element chunks: gfx950 loads and stores global memory at
// any element address, so odd row strides and views cost no other path.
typedef short8_t short8_u __attribute__((aligned(2)));
typedef float4_t float4_u __attribute__((aligned(4)));
typedef __attribute__((ext_vector_type(2))) unsigned uint2_t;
typedef uint2_t uint2_u __attribute__((aligned(1)));
typedef __attribute__((ext_vector_type(4))) unsigned uint4_t;
typedef uint4_t uint4_u2 __attribute__((aligned(2)));
typedef uint4_t uint4_u4 __attribute__((aligned(4)));

template <int DT>
struct Elem;

template <>
struct Elem<DT_BF16> {
  typedef ushort_t T;
  static constexpr unsigned kFloor = 1, kTop = 249;
  static DEV_INLINE float get(T v) { return bf2f(v); }
  static DEV_INLINE T put(float v) { return f2bf(v); }
  static DEV_INLINE void load8(const T* p, float* v) {
    const short8_t r = *reinterpret_cast<const short8_u*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = bf2f(ushort_t(r[e]));
  }
  static DEV_INLINE void store8(T* p, const float* v) {
    short8_t r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = short(f2bf(v[e]));
    *reinterpret_cast<short8_u*>(p) = r;
  }
};

template <>
struct Elem<DT_F16> {
  typedef _Float16 T;
  static constexpr unsigned kFloor = 103, kTop = 137;
  typedef __attribute__((ext_vector_type(8))) _Float16 half8_t;
  typedef half8_t half8_u __attribute__((aligned(2)));
  static DEV_INLINE float get(T v) { return float(v); }
  static DEV_INLINE T put(float v) { return T(v); }
  static DEV_INLINE void load8(const T* p, float* v) {
    const half8_t r = *reinterpret_cast<const half8_u*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = float(r[e]);
  }
  static DEV_INLINE void store8(T* p, const float* v) {
    half8_t r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = T(v[e]);
    *reinterpret_cast<half8_u*>(p) = r;
  }
};

template <>
struct Elem<DT_F32> {
  typedef float T;
  static constexpr unsigned kFloor = 1, kTop = 249;
  static DEV_INLINE float get(T v) { return v; }
  static DEV_INLINE T put(float v) { return v; }
  static DEV_INLINE void load8(const T* p, float* v) {
    const float4_t a = *reinterpret_cast<const float4_u*>(p);
    const float4_t b = *reinterpret_cast<const float4_u*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
  }
  static DEV_INLINE void store8(T* p, const float* v) {
    *reinterpret_cast<float4_u*>(p) = float4_t{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<float4_u*>(p + 4) = float4_t{v[4], v[5], v[6], v[7]};
  }
};

template <int DT>
using TP = typename Elem<DT>::T;

#define DT_SWITCH(DTV, ...)                                            \
  switch (DTV) {                                                       \
    case DT_BF16: { constexpr int kDT = DT_BF16; __VA_ARGS__; break; } \
    case DT_F16:  { constexpr int kDT = DT_F16;  __VA_ARGS__; break; } \
    case DT_F32:  { constexpr int kDT = DT_F32;  __VA_ARGS__; break; } \
    default: yams_launch_fail("rows dtype", (DTV), 0, 0, 0);           \
  }

// `n` (0..8) valid elements at p; the others read as zero
template <int DT>
DEV_INLINE void load_chunk(const typename Elem<DT>::T* p, int n, float* v) {
  if (n == 8) {
    Elem<DT>::load8(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (n > 0) {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < n) v[e] = Elem<DT>::get(p[e]);
    }
  }
}

template <int DT>
DEV_INLINE void store_chunk(typename Elem<DT>::T* p, int n, const float* v) {
  if (n == 8) {
    Elem<DT>::store8(p, v);
  } else if (n > 0) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = Elem<DT>::put(v[e]);
  }
}

DEV_INLINE unsigned f_bits(float v) { return __float_as_uint(v); }
DEV_INLINE float exp_unit(unsigned e) { return __uint_as_float(e << 23); }

// max over the four lanes of a quad (a group of 32 channels is four
// chunks of 8, held by one quad); every lane of the quad must be active
DEV_INLINE unsigned quad_max(unsigned v) {
  const unsigned a = unsigned(
      __builtin_amdgcn_mov_dpp(int(v), 0xB1, 0xf, 0xf, true));  // 1 0 3 2
  v = a > v ? a : v;
  const unsigned b = unsigned(
      __builtin_amdgcn_mov_dpp(int(v), 0x4E, 0xf, 0xf, true));  // 2 3 0 1
  return b > v ? b : v;
}

// Eight values of a lane -> eight codes (two dwords) and the exponent
// byte of the quad's group.  Lanes without values pass zeros.
template <int DT>
DEV_INLINE uint2_t quantize8(const float* v, unsigned& exponent) {
  unsigned m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const unsigned b = f_bits(v[e]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  m = quad_max(m);
  uint2_t out;
  if (m >= 0x7f800000u) {  // rare, and the same for the whole quad
    exponent = 255;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      unsigned w = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned b = f_bits(v[d * 4 + e]);
        const unsigned q = b == 0x7f800000u ? 1u : b == 0xff800000u ? 255u : 0u;
        w |= q << (8 * e);
      }
      out[d] = w;
    }
    return out;
  }
  // 127 = 1.984375 * 2^6: one unit more where the mantissa passes that
  const int raw = int((m + 0x1ffffu) >> 23) - 6;
  const unsigned E = raw < int(Elem<DT>::kFloor) ? Elem<DT>::kFloor
                                                 : unsigned(raw);
  const float inv = __uint_as_float((254u - E) << 23);
  exponent = E;
  // x * inv + 1.5 * 2^23 rounds to a whole number (half to even: the
  // product is exact), whose low byte is the code in two's complement
  constexpr float kRound = 12582912.f;
  unsigned q[8];
  if (E < Elem<DT>::kTop) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = f_bits(fmaf(v[e], inv, kRound));
  } else {  // the top binade, rare: stop at 63
#pragma unroll
    for (int e = 0; e < 8; ++e)
      q[e] = f_bits(fminf(fmaxf(v[e] * inv, -63.f), 63.f) + kRound);
  }
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    // the low bytes of four registers (v_perm: bytes 0..3 are the second
    // operand's, 4..7 the first's)
    const unsigned lo = __builtin_amdgcn_perm(q[4 * d + 1], q[4 * d], 0x0400u);
    const unsigned hi =
        __builtin_amdgcn_perm(q[4 * d + 3], q[4 * d + 2], 0x0400u);
    out[d] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  return out;
}

DEV_INLINE void dequantize4(unsigned w, float unit, float* v) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    v[e] = float(int((signed char)(w >> (8 * e)))) * unit;
}

// `n` (0..8) codes at p -> values
DEV_INLINE void load_codes(const signed char* p, int n, unsigned exponent,
                           float* v) {
  const float unit = exp_unit(exponent);
  if (n == 8) {
    const uint2_t w = *reinterpret_cast<const uint2_u*>(p);
    dequantize4(w[0], unit, v);
    dequantize4(w[1], unit, v + 4);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (n > 0) {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < n) v[e] = float(int(p[e])) * unit;
    }
  }
}

DEV_INLINE void store_codes(signed char* p, int n, uint2_t w) {
  if (n == 8) {
    *reinterpret_cast<uint2_u*>(p) = w;
  } else if (n > 0) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = (signed char)(w[e >> 2] >> (8 * (e & 3)));
  }
}

// Loads and stores address memory as a base that is the same for the whole
// wave plus a 32-bit byte offset of the lane: one register per address, and
// the base moves by scalar instructions.
template <typename T>
DEV_INLINE const T* lane_at(const void* base, unsigned off) {
  return reinterpret_cast<const T*>(static_cast<const char*>(base) + off);
}
template <typename T>
DEV_INLINE T* lane_at(void* base, unsigned off) {
  return reinterpret_cast<T*>(static_cast<char*>(base) + off);
}

typedef unsigned u32_u1 __attribute__((aligned(1)));
typedef uint2_t uint2_u1 __attribute__((aligned(1)));
typedef unsigned short u16_u1 __attribute__((aligned(1)));

// SIZE * 2 words: eight elements of SIZE bytes.  A vector and not an array,
// so that no choice between words becomes an address.
template <int SIZE>
struct WordsOf {
  typedef __attribute__((ext_vector_type(SIZE * 2))) unsigned T;
};
template <int SIZE>
using Words = typename WordsOf<SIZE>::T;

// The first n (0..8) of eight elements of SIZE bytes; the rest reads as
// zero.  A short chunk is four, two and one of them, so it takes three
// accesses, which waves without one skip.
template <int SIZE>
DEV_INLINE Words<SIZE> load_words(const void* base, unsigned off, int n) {
  Words<SIZE> w;
  if (n == 8) {
    if constexpr (SIZE == 1) {
      w = *lane_at<uint2_u1>(base, off);
    } else if constexpr (SIZE == 2) {
      w = *lane_at<uint4_u2>(base, off);
    } else {
      const uint4_t a = *lane_at<uint4_u4>(base, off);
      const uint4_t b = *lane_at<uint4_u4>(base, off + 16);
      w = Words<SIZE>{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
    return w;
  }
  w = Words<SIZE>(0u);
  if (n == 0) return w;
  const bool four = (n & 4) != 0;
  const unsigned tail = off + SIZE * (n & 4), last = off + SIZE * (n & 6);
  if constexpr (SIZE == 4) {
    uint4_t a = uint4_t(0u);
    unsigned b = 0u, c = 0u, d = 0u;
    if (four) a = *lane_at<uint4_u4>(base, off);
    if ((n & 3) > 0) b = *lane_at<unsigned>(base, tail);
    if ((n & 3) > 1) c = *lane_at<unsigned>(base, tail + 4);
    if ((n & 3) > 2) d = *lane_at<unsigned>(base, tail + 8);
    w[0] = four ? a[0] : b;
    w[1] = four ? a[1] : c;
    w[2] = four ? a[2] : d;
    w[3] = a[3];
    w[4] = four ? b : 0u;
    w[5] = four ? c : 0u;
    w[6] = four ? d : 0u;
  } else if constexpr (SIZE == 2) {
    uint2_t a = uint2_t(0u);
    unsigned b = 0u, c = 0u;
    if (four) a = *lane_at<uint2_u1>(base, off);
    if (n & 2) b = *lane_at<u32_u1>(base, tail);
    if (n & 1) c = *lane_at<unsigned short>(base, last);
    // after `four` come b, if there are two, and c
    const unsigned p = n & 2 ? b : c, q = n & 2 ? c : 0u;
    w[0] = four ? a[0] : p;
    w[1] = four ? a[1] : q;
    w[2] = four ? p : 0u;
    w[3] = four ? q : 0u;
  } else {
    unsigned a = 0u, b = 0u;
    if (four) a = *lane_at<u32_u1>(base, off);
    if (n & 2) b = *lane_at<u16_u1>(base, tail);
    if (n & 1)
      b |= unsigned(*lane_at<unsigned char>(base, last)) << (8 * (n & 2));
    w[0] = four ? a : b;
    w[1] = four ? b : 0u;
  }
  return w;
}

template <int SIZE>
DEV_INLINE void store_words(void* base, unsigned off, int n, Words<SIZE> w) {
  if (n == 8) {
    if constexpr (SIZE == 1) {
      *lane_at<uint2_u1>(base, off) = w;
    } else if constexpr (SIZE == 2) {
      *lane_at<uint4_u2>(base, off) = w;
    } else {
      *lane_at<uint4_u4>(base, off) = uint4_t{w[0], w[1], w[2], w[3]};
      *lane_at<uint4_u4>(base, off + 16) = uint4_t{w[4], w[5], w[6], w[7]};
    }
    return;
  }
  if (n == 0) return;
  const bool four = (n & 4) != 0;
  const unsigned tail = off + SIZE * (n & 4), last = off + SIZE * (n & 6);
  if constexpr (SIZE == 4) {
    const unsigned b = four ? w[4] : w[0], c = four ? w[5] : w[1];
    const unsigned d = four ? w[6] : w[2];
    if (four) *lane_at<uint4_u4>(base, off) = uint4_t{w[0], w[1], w[2], w[3]};
    if ((n & 3) > 0) *lane_at<unsigned>(base, tail) = b;
    if ((n & 3) > 1) *lane_at<unsigned>(base, tail + 4) = c;
    if ((n & 3) > 2) *lane_at<unsigned>(base, tail + 8) = d;
  } else if constexpr (SIZE == 2) {
    const unsigned p = four ? w[2] : w[0], q = four ? w[3] : w[1];
    if (four) *lane_at<uint2_u1>(base, off) = uint2_t{w[0], w[1]};
    if (n & 2) *lane_at<u32_u1>(base, tail) = p;
    if (n & 1)
      *lane_at<unsigned short>(base, last) =
          (unsigned short)(n & 2 ? q : p);
  } else {
    const unsigned b = four ? w[1] : w[0];
    if (four) *lane_at<u32_u1>(base, off) = w[0];
    if (n & 2) *lane_at<u16_u1>(base, tail) = (unsigned short)b;
    if (n & 1)
      *lane_at<unsigned char>(base, last) =
          (unsigned char)(b >> (8 * (n & 2)));
  }
}

// the elements from s (0..7) on, and zeros behind them
template <int SIZE>
DEV_INLINE Words<SIZE> drop_words(Words<SIZE> w, int s) {
  constexpr int N = SIZE * 2;
  const int bytes = s * SIZE;
#pragma unroll
  for (int d = N / 2; d > 0; d /= 2) {
    const bool by = (bytes / 4 & d) != 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned from = i + d < N ? w[i + d < N ? i + d : 0] : 0u;
      w[i] = by ? from : w[i];
    }
  }
  if constexpr (SIZE < 4) {
    const unsigned bits = unsigned(bytes & 3) * 8u;
#pragma unroll
    for (int i = 0; i < N; ++i)
      w[i] = __builtin_amdgcn_alignbit(i + 1 < N ? w[i + 1 < N ? i + 1 : 0]
                                                 : 0u,
                                       w[i], bits);
  }
  return w;
}

// How the chunks of a row are read.  The choice between short loads
// (READ_SHORT, for rows of less than eight) waits for each of them, and so for
// the memory once for every input of a row.  Longer rows are read without
// any choice: the last chunk, if it is short, as the last eight elements, of
// which the first are dropped later (READ_RAGGED); chunks behind the row
// likewise, and blanked.  Backward pass of 98000 x 333 fp16: 499 -> 298 us,
// of 200704 x 120 bf16 142 -> 115.
enum Read { READ_WHOLE, READ_RAGGED, READ_SHORT };

inline Read read_of(int C) {
  return C < 8 ? READ_SHORT : C % 8 == 0 ? READ_WHOLE : READ_RAGGED;
}

#define RAGGED_SWITCH(C, ...)            \
  if (read_of(C) == READ_RAGGED) {       \
    constexpr bool kRagged = true;       \
    __VA_ARGS__;                         \
  } else {                               \
    constexpr bool kRagged = false;      \
    __VA_ARGS__;                         \
  }

// A chunk as it lies in memory, loaded early and decoded late: eight
// elements, or (KEPT) eight codes and the exponent of their group.
template <int DT, bool KEPT>
struct RawChunk {
  static constexpr int kSize = KEPT ? 1 : int(sizeof(typename Elem<DT>::T));
  Words<kSize> w;
  unsigned exponent;

  // `off` counts bytes of the elements or codes
  DEV_INLINE void load(const void* base, unsigned off) {
    w = load_words<kSize>(base, off, 8);
  }
  DEV_INLINE void load_short(const void* base, unsigned off, int n) {
    w = load_words<kSize>(base, off, n);
  }
  // what load() has read of a chunk of n (0..8)
  DEV_INLINE void drop(int n) { w = drop_words<kSize>(w, n > 0 ? 8 - n : 0); }
  // (its group too: code 0 of a group with a non-finite value is NaN)
  DEV_INLINE void blank(int n) {
    w = n > 0 ? w : Words<kSize>(0u);
    if constexpr (KEPT) exponent = n > 0 ? exponent : 0u;
  }
  DEV_INLINE void load_exponent(const unsigned char* base, unsigned off) {
    exponent = *lane_at<unsigned char>(base, off);
  }
  DEV_INLINE void decode(float* v) const {
    if constexpr (KEPT) {
      const float unit = exp_unit(exponent);
      dequantize4(w[0], unit, v);
      dequantize4(w[1], unit, v + 4);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (DT == DT_F32) {
          v[e] = __uint_as_float(w[e]);
        } else if constexpr (DT == DT_BF16) {
          v[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u
                                       : w[e >> 1] << 16);
        } else {
          union { ushort_t u; _Float16 t; } c;
          c.u = ushort_t(w[e >> 1] >> (16 * (e & 1)));
          v[e] = float(c.t);
        }
      }
    }
  }
};

// eight values -> the type's words, and the store of the first n
template <int DT>
DEV_INLINE void put_chunk(void* base, unsigned off, int n, const float* v) {
  constexpr int kSize = int(sizeof(typename Elem<DT>::T));
  Words<kSize> w;
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = f_bits(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      union { typename Elem<DT>::T t; ushort_t u; } a, b;
      a.t = Elem<DT>::put(v[2 * e]);
      b.t = Elem<DT>::put(v[2 * e + 1]);
      w[e] = unsigned(a.u) | unsigned(b.u) << 16;
    }
  }
  store_words<kSize>(base, off, n, w);
}

DEV_INLINE void put_codes(void* base, unsigned off, int n, uint2_t q) {
  store_words<1>(base, off, n, q);
}

// Chunk of the row at `row` from column c on: n (0..8) of its C elements.
// RAGGED: rows with a short last chunk (READ_RAGGED).  Both sides measured,
// backward of bias + activation, kept in 8 bits: 98000 x 333 104 us without
// RAGGED and 44 with it; 16384 x 8192 133, and 146 read RAGGED's way.
template <int DT, bool RAGGED>
DEV_INLINE void take_chunk(const TP<DT>* row, int c, int n, int C, float* v) {
  if constexpr (RAGGED) {
    RawChunk<DT, false> q;
    q.load(row, unsigned(min(c, C - 8)) * unsigned(sizeof(TP<DT>)));
    q.drop(n);
    q.blank(n);
    q.decode(v);
  } else {
    load_chunk<DT>(row + c, n, v);
  }
}
template <bool RAGGED>
DEV_INLINE void take_codes(const signed char* row, int c, int n, int C,
                           unsigned exponent, float* v) {
  if constexpr (RAGGED) {
    RawChunk<DT_F32, true> q;
    q.load(row, unsigned(min(c, C - 8)));
    q.drop(n);
    q.blank(n);
    q.exponent = exponent;
    q.decode(v);
  } else {
    load_codes(row + c, n, exponent, v);
  }
}
template <int DT, bool RAGGED>
DEV_INLINE void give_chunk(TP<DT>* row, int c, int n, const float* v) {
  if constexpr (RAGGED)
    put_chunk<DT>(row, unsigned(c) * unsigned(sizeof(TP<DT>)), n, v);
  else
    store_chunk<DT>(row + c, n, v);
}
template <bool RAGGED>
DEV_INLINE void give_codes(signed char* row, int c, int n, uint2_t q) {
  if constexpr (RAGGED)
    put_codes(row, unsigned(c), n, q);
  else
    store_codes(row + c, n, q);
}

// n / d for n < 2^31 by one multiplication (d is fixed for a launch; the
// hardware has no integer division): Granlund and Montgomery, "Division by
// invariant integers using multiplication", 1994
struct FastDiv {
  unsigned d, mul, shift;
  DEV_INLINE unsigned div(unsigned n) const {
    return (__umulhi(n, mul) + n) >> shift;
  }
};

inline FastDiv fast_div(unsigned d) {
  FastDiv f;
  f.d = d;
  f.shift = 0;
  while ((1ull << f.shift) < d) ++f.shift;
  f.mul = unsigned(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
  return f;
}

}  // namespace yams
