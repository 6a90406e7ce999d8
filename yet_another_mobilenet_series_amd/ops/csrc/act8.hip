// Activations kept in 8 bits for the backward pass (rows.h defines the
// form): the codec, and bias + activation on an input that is kept so.
//
// All of it is bound by memory: a chunk of 8 channels is one 16-byte load
// (bf16) against ~40 VALU operations.  One lane holds one chunk, so a
// group of 32 channels is one quad of lanes and its maximum costs two DPP
// moves.  Chunks are numbered row by row, each row padded to whole groups,
// so that a quad never straddles two rows.
//
// Measured (reads and writes together, one call after another): pack 16384 x
// 4096 bf16 or fp16 in 38 us, 5.4 TB/s, fp32 79 (4.3), unpack 31 and 75;
// 200704 x 120 bf16 13 (5.7) and 12, fp32 18 and 20; bias and hard-swish kept
// in 8 bits, 16384 x 8192 bf16, forward 122 us, 5.5 TB/s, backward 134, 5.0.
// A large copy reaches 4.9 to 6.7, the less the larger it is.

#include <algorithm>

#include "rows.h"
#include "rows_engine.h"

namespace yams {

namespace {

struct ChunkMap {
  FastDiv per_row;  // chunks of a row, padded to whole groups
  unsigned total;
  int C;
};

ChunkMap chunk_map(int64_t rows, int C) {
  const unsigned per_row = unsigned(ceil_div(C, kGroup)) * 4;
  return {fast_div(per_row), unsigned(rows * per_row), C};
}

constexpr int kThreads = 256;

int chunk_grid(const ChunkMap& m) {
  return int(std::min<int64_t>((int64_t(m.total) + kThreads - 1) / kThreads,
                               16384));
}

template <int DT, bool RAGGED>
__global__ __launch_bounds__(kThreads) void pack_kernel(
    const typename Elem<DT>::T* __restrict__ x, int64_t stride,
    signed char* __restrict__ codes, unsigned char* __restrict__ exps,
    ChunkMap m) {
  const unsigned step = gridDim.x * kThreads;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < m.total;
       i += step) {
    const unsigned row = m.per_row.div(i);
    const unsigned chunk = i - row * m.per_row.d;
    const int c = int(chunk) * 8, n = min(8, max(0, m.C - c));
    float v[8];
    take_chunk<DT, RAGGED>(x + int64_t(row) * stride, c, n, m.C, v);
    unsigned e;
    const uint2_t q = quantize8<DT>(v, e);
    give_codes<RAGGED>(codes + int64_t(row) * m.C, c, n, q);
    if ((chunk & 3) == 0) exps[i >> 2] = (unsigned char)e;
  }
}

template <int DT, bool RAGGED>
__global__ __launch_bounds__(kThreads) void unpack_kernel(
    const signed char* __restrict__ codes,
    const unsigned char* __restrict__ exps,
    typename Elem<DT>::T* __restrict__ y, ChunkMap m) {
  const unsigned step = gridDim.x * kThreads;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < m.total;
       i += step) {
    const unsigned row = m.per_row.div(i);
    const unsigned chunk = i - row * m.per_row.d;
    const int c = int(chunk) * 8, n = min(8, max(0, m.C - c));
    const int64_t at = int64_t(row) * m.C;
    float v[8];
    take_codes<RAGGED>(codes + at, c, n, m.C, exps[i >> 2], v);
    give_chunk<DT, RAGGED>(y + at, c, n, v);
  }
}

template <int DT, int ACT, bool KEEP, bool RAGGED>
__global__ __launch_bounds__(kThreads) void act_fwd_kernel(
    const typename Elem<DT>::T* __restrict__ z, int64_t stride,
    const float* __restrict__ bias, typename Elem<DT>::T* __restrict__ y,
    signed char* __restrict__ codes, unsigned char* __restrict__ exps,
    ChunkMap m) {
  const unsigned step = gridDim.x * kThreads;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < m.total;
       i += step) {
    const unsigned row = m.per_row.div(i);
    const unsigned chunk = i - row * m.per_row.d;
    const int c = int(chunk) * 8, n = min(8, max(0, m.C - c));
    const int64_t at = int64_t(row) * m.C;
    float v[8], b[8] = {}, o[8];
    take_chunk<DT, RAGGED>(z + int64_t(row) * stride, c, n, m.C, v);
    if (bias != nullptr) take_chunk<DT_F32, RAGGED>(bias, c, n, m.C, b);
    if (KEEP) {
      unsigned e;
      const uint2_t q = quantize8<DT>(v, e);
      give_codes<RAGGED>(codes + at, c, n, q);
      if ((chunk & 3) == 0) exps[i >> 2] = (unsigned char)e;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = act_fwd<ACT>(v[e] + b[e]);
    give_chunk<DT, RAGGED>(y + at, c, n, o);
  }
}

// Backward.  A thread keeps its 8 channels for all its rows, so that the
// bias gradient is a sum in registers: a block is TX chunks by 256 / TX
// rows, walks `per` rows, and leaves one row of partial sums.
template <int DT, int ACT, bool KEPT, bool RAGGED>
__global__ __launch_bounds__(kThreads) void act_bwd_kernel(
    const typename Elem<DT>::T* __restrict__ dy, int64_t dy_stride,
    const typename Elem<DT>::T* __restrict__ z, int64_t z_stride,
    const signed char* __restrict__ codes,
    const unsigned char* __restrict__ exps, const float* __restrict__ bias,
    typename Elem<DT>::T* __restrict__ dz, float* __restrict__ ws,
    int64_t rows, int C, int G, int TX, int64_t per, int ws_stride) {
  __shared__ float red[kThreads * 8];
  const int tx = int(threadIdx.x) % TX, ty = int(threadIdx.x) / TX;
  const int TY = kThreads / TX;
  const int c = (int(blockIdx.x) * TX + tx) * 8;
  const int n = min(8, max(0, C - c));
  const int64_t lo = int64_t(blockIdx.y) * per;
  const int64_t hi = min(lo + per, rows);
  float b[8] = {}, s[8] = {};
  if (bias != nullptr) load_chunk<DT_F32>(bias + c, n, b);
  if (n > 0) {
    for (int64_t r = lo + ty; r < hi; r += TY) {
      float g[8], v[8], o[8];
      take_chunk<DT, RAGGED>(dy + r * dy_stride, c, n, C, g);
      if (KEPT)
        take_codes<RAGGED>(codes + r * C, c, n, C, exps[r * G + (c >> 5)], v);
      else
        take_chunk<DT, RAGGED>(z + r * z_stride, c, n, C, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o[e] = g[e] * act_bwd<ACT>(v[e] + b[e]);
        s[e] += o[e];
      }
      give_chunk<DT, RAGGED>(dz + r * C, c, n, o);
    }
  }
  if (ws == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[e * kThreads + int(threadIdx.x)] = s[e];
  __syncthreads();
  // 8 * TX sums of TY partial ones each
  for (int k = int(threadIdx.x); k < 8 * TX; k += kThreads) {
    const int x = k >> 3, e = k & 7;
    float t = 0.f;
    for (int l = 0; l < TY; ++l) t += red[e * kThreads + l * TX + x];
    const int col = (int(blockIdx.x) * TX + x) * 8 + e;
    if (col < C) ws[int64_t(blockIdx.y) * ws_stride + col] = t;
  }
}

struct BwdShape {
  int TX, gx, gy;
  int64_t per;
};

// Enough blocks to fill the chip (16384 x 8192: 133 us with 2048, 172 with
// 1024), but at least four rows a thread, which keeps the partial sums below
// 1/16 of the rows' bytes, and at most 1024 rows of them, which the second
// launch walks (200704 x 120: 31.6 us in all, 34.7 with 2048).  Few rows take
// narrow blocks that have all of them: no second launch (256 x 1280: 6.2
// us against 5.9 + 4.0).
BwdShape bwd_shape(int64_t rows, int C) {
  BwdShape b;
  const int chunks = ceil_div(C, 8);
  b.TX = 4;
  if (rows <= 4 * kThreads / b.TX && chunks / b.TX < kMaxBlocks) {
    b.gx = ceil_div(chunks, b.TX);
    b.gy = 1;
    b.per = rows;
    return b;
  }
  while (b.TX < 64 && b.TX < chunks) b.TX *= 2;
  b.gx = ceil_div(chunks, b.TX);
  const int TY = kThreads / b.TX;
  const int64_t want = std::max(1, std::min(1024, 2048 / b.gx));
  const int64_t most = std::max<int64_t>(1, rows / (4 * TY));
  b.gy = int(std::min(want, most));
  b.per = (rows + b.gy - 1) / b.gy;
  b.gy = int((rows + b.per - 1) / b.per);
  return b;
}

}  // namespace

void pack_rows(int dt, RowsDesc x, Kept out, int64_t rows, int C,
               hipStream_t s) {
  if (rows == 0 || C == 0) return;
  const ChunkMap m = chunk_map(rows, C);
  const int grid = chunk_grid(m);
  DT_SWITCH(dt, RAGGED_SWITCH(C, {
    pack_kernel<kDT, kRagged><<<grid, kThreads, 0, s>>>(
        static_cast<const TP<kDT>*>(x.p), x.stride, out.codes, out.exps, m);
  }));
}

void unpack_rows(int dt, Kept in, void* y, int64_t rows, int C,
                 hipStream_t s) {
  if (rows == 0 || C == 0) return;
  const ChunkMap m = chunk_map(rows, C);
  const int grid = chunk_grid(m);
  DT_SWITCH(dt, RAGGED_SWITCH(C, {
    unpack_kernel<kDT, kRagged><<<grid, kThreads, 0, s>>>(
        in.codes, in.exps, static_cast<TP<kDT>*>(y), m);
  }));
}

void act_rows_fwd(int dt, RowsDesc z, const float* bias, int act, void* y,
                  Kept kept, int64_t rows, int C, hipStream_t s) {
  if (rows == 0 || C == 0) return;
  const ChunkMap m = chunk_map(rows, C);
  const int grid = chunk_grid(m);
  DT_SWITCH(dt, ACT_SWITCH(act, RAGGED_SWITCH(C, {
    auto* zp = static_cast<const TP<kDT>*>(z.p);
    auto* yp = static_cast<TP<kDT>*>(y);
    if (kept.codes != nullptr)
      act_fwd_kernel<kDT, kAct, true, kRagged><<<grid, kThreads, 0, s>>>(
          zp, z.stride, bias, yp, kept.codes, kept.exps, m);
    else
      act_fwd_kernel<kDT, kAct, false, kRagged><<<grid, kThreads, 0, s>>>(
          zp, z.stride, bias, yp, nullptr, nullptr, m);
  })));
}

int64_t act_rows_ws(int64_t rows, int C) {
  if (rows == 0) return 0;
  return int64_t(bwd_shape(rows, C).gy) * ((C + 3) / 4 * 4);
}

void act_rows_bwd(int dt, RowsDesc dy, RowsDesc z, Kept kept,
                  const float* bias, int act, void* dz, float* dbias,
                  float* ws, int64_t rows, int C, hipStream_t s) {
  if (rows == 0 || C == 0) return;
  const BwdShape b = bwd_shape(rows, C);
  const int G = ceil_div(C, kGroup);
  const bool one = b.gy == 1;  // a single row of partial sums is the sum
  float* part = dbias == nullptr ? nullptr : (one ? dbias : ws);
  const int ws_stride = (C + 3) / 4 * 4;
  DT_SWITCH(dt, ACT_SWITCH(act, RAGGED_SWITCH(C, {
    auto* gp = static_cast<const TP<kDT>*>(dy.p);
    auto* zp = static_cast<const TP<kDT>*>(z.p);
    auto* op = static_cast<TP<kDT>*>(dz);
    const dim3 grid(b.gx, b.gy);
    if (zp == nullptr)
      act_bwd_kernel<kDT, kAct, true, kRagged><<<grid, kThreads, 0, s>>>(
          gp, dy.stride, nullptr, 0, kept.codes, kept.exps, bias, op, part,
          rows, C, G, b.TX, b.per, ws_stride);
    else
      act_bwd_kernel<kDT, kAct, false, kRagged><<<grid, kThreads, 0, s>>>(
          gp, dy.stride, zp, z.stride, nullptr, nullptr, bias, op, part,
          rows, C, G, b.TX, b.per, ws_stride);
  })));
  if (dbias != nullptr && !one) slab_reduce(ws, dbias, ws_stride, b.gy, s);
}

}  // namespace yams
