// Launchers of the row operators (activations kept in 8 bits, norms over
// channels, the FC layer on an 8-bit input): the interface between
// bindings_rows.cpp and act8.hip, rownorm.hip and linear8.hip.
//
// Rows: `p` points at element [0, 0] of [rows, C] with unit stride along
// C and `stride` elements between rows; any element alignment.  `dt` is
// one of DT_BF16 / DT_F16 / DT_F32 (rows.h).  Codes are [rows, C] bytes
// without gaps, exponents [rows, ceil(C / 32)] bytes.  Launches are
// asynchronous on `s`; rows == 0 launches nothing.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace yams {

struct Kept {  // a kept activation; null pointers where there is none
  signed char* codes = nullptr;
  unsigned char* exps = nullptr;
};

// elements between rows where a kernel addresses up to 64 of them with 32
// bits of bytes (norms and products)
constexpr int64_t kMaxStride = int64_t(1) << 22;

// blocks of a launch along one axis, at 256 threads: it has fewer than 2^32
// threads
constexpr int kMaxBlocks = (1 << 24) - 1;

struct RowsDesc {
  const void* p = nullptr;
  int64_t stride = 0;
};

// --- codec (act8.hip) ----------------------------------------------------
void pack_rows(int dt, RowsDesc x, Kept out, int64_t rows, int C,
               hipStream_t s);
void unpack_rows(int dt, Kept in, void* y, int64_t rows, int C,
                 hipStream_t s);
// chunk indices are 32-bit: rows * 4 * ceil(C / 32) has to stay below this
constexpr int64_t kMaxChunks = int64_t(1) << 31;

// --- bias + activation on a kept input (act8.hip) ------------------------
// y = act(z + bias); `kept` (optional) receives z's 8-bit form
void act_rows_fwd(int dt, RowsDesc z, const float* bias, int act, void* y,
                  Kept kept, int64_t rows, int C, hipStream_t s);
// dz = dy * act'(z + bias) with z from `z` or, where that is null, from
// `kept`; dbias fp32 [C] (optional) with ws of act_rows_ws floats
void act_rows_bwd(int dt, RowsDesc dy, RowsDesc z, Kept kept,
                  const float* bias, int act, void* dz, float* dbias,
                  float* ws, int64_t rows, int C, hipStream_t s);
// (the last four-column step of dbias is written whole: allocate C rounded
// up to 4)
int64_t act_rows_ws(int64_t rows, int C);
// out[i] = sum over `splits` slabs of ws[split][i], in a fixed order
void slab_reduce(const float* ws, float* out, int64_t elems, int splits,
                 hipStream_t s);

// --- norms over channels (rownorm.hip) -----------------------------------
// n = N1(h) (post; n = h without it);  t = scale * alpha * a(g) * n
// y = x + t (no h: y = x);             u = N2(y) (next)
// Gates: one value for each element, or for each channel of every run of
// `group_rows` rows.
constexpr int GATE_NONE = 0, GATE_FULL = 1, GATE_GROUP = 2;
// gate activations: an activation code of common.h, or
constexpr int GATE_SIGMOID = 5;
constexpr int kMaxNormC = 16384;

struct JoinDesc {
  int64_t rows = 0;
  int C = 0;
  bool layer = false, post = true, next = true;
  int gate = GATE_NONE, gate_act = 0;
  int64_t group_rows = 1;
  float eps = 0.f, alpha = 1.f;
  RowsDesc h, x, g;           // inputs (h null: a norm alone, y = x)
  Kept hk, xk, gk;            // forward: written; backward: read if set
  const float *w = nullptr, *b = nullptr, *scale = nullptr;
  const float *w2 = nullptr, *b2 = nullptr;
  void *y = nullptr, *u = nullptr;   // forward (y null: not wanted)
  RowsDesc dy, du;            // backward: either may be null
  void *dh = nullptr, *dx = nullptr, *dg = nullptr;  // null: not wanted
  // parameter sums wanted: bits 0..4 are scale, w, b, w2, b2.  `sums`
  // receives them one after another, each C rounded up to 4 floats long
  unsigned want = 0;
  float *sums = nullptr, *ws = nullptr;
};
void join_fwd(int dt, const JoinDesc& d, hipStream_t s);
void join_bwd(int dt, const JoinDesc& d, hipStream_t s);
int64_t join_bwd_ws(int dt, const JoinDesc& d);  // floats of `ws`

// --- FC layer on a kept input (linear8.hip) -------------------------------
// Row-major operands with any row stride.  `wdt`: DT_BF16 or DT_F32 (which
// goes in as two bf16 parts); out types DT_BF16 or DT_F32.
// y[M, N] = x[M, K] w[N, K]^T + bias; `bdt`: the bias, DT_BF16 or DT_F32
void linear8_fwd(RowsDesc x, int wdt, RowsDesc w, int bdt, const void* bias,
                 void* y, float* ws, int64_t M, int N, int K, hipStream_t s);
// dx[M, K] = dy[M, N] w[N, K]
void linear8_dgrad(RowsDesc dy, int wdt, RowsDesc w, void* dx, float* ws,
                   int64_t M, int N, int K, hipStream_t s);
// dw[N, K] = dy[M, N]^T X, X the values of the codes; `padded`: seven bytes
// behind the codes may be read
void linear8_wgrad(RowsDesc dy, Kept x, bool padded, int odt, void* dw,
                   float* ws, int64_t M, int N, int K, hipStream_t s);
// floats of `ws` for [rows, cols] outputs over a reduction of `depth`; `wdt`
// of the weights (the weight gradient has codes in their place: DT_BF16, and
// says whether they are `loose`)
int64_t linear8_ws(int64_t rows, int64_t cols, int64_t depth, int wdt,
                   bool loose = false);
bool linear8_loose(int64_t K, bool padded);
// db = sum over rows of dy; ws of row_sum_ws floats; db as dbias above
// (`odt` DT_F32) or bf16 [C] (DT_BF16)
void row_sum(int dt, RowsDesc dy, int odt, void* db, float* ws, int64_t rows,
             int C, hipStream_t s);
int64_t row_sum_ws(int64_t rows, int C);

}  // namespace yams
