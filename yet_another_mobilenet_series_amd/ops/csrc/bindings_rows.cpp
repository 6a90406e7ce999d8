// Torch bindings of the row operators: activations kept in 8 bits, norms
// over channels and the joins between blocks, the FC layer on a kept input.
//
// Tensor contract: "rows" are 2D [rows, C] with unit stride along C and any
// stride between rows; outputs, codes (int8) and exponents (uint8) are
// contiguous; per-channel parameters and sums are fp32 contiguous.  Every
// launch goes to the current stream of the tensors' own device.

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "bindings_rows.h"

namespace {

using torch::Tensor;
typedef c10::optional<Tensor> Opt;

constexpr int kBf16 = 0, kF16 = 1, kF32 = 2;  // DT_* of rows.h
using yams::kMaxStride;

int dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kBFloat16: return kBf16;
    case torch::kFloat16: return kF16;
    case torch::kFloat32: return kF32;
    default:
      TORCH_CHECK(false, name, " must be bf16, fp16 or fp32, got ",
                  t.scalar_type());
  }
}

hipStream_t stream_of(const Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

float* ws_ptr(const Tensor& ws) {
  return ws.defined() ? ws.data_ptr<float>() : nullptr;
}

// How far apart a kernel takes rows: norms and products address the rows of a
// block from a common base with 32 bits, the others every row with 64.
enum Apart { NEAR, ANY };

// the tensors of one call: one device, one row type, one shape
struct Call {
  const Tensor& ref;
  Apart apart;
  int dt;
  int64_t rows;
  int C;

  Call(const Tensor& t, const char* name, Apart a = NEAR) : ref(t), apart(a) {
    TORCH_CHECK(t.is_cuda() && t.dim() == 2, name,
                " must be [rows, C] on a GPU");
    dt = dtype_of(t, name);
    rows = t.size(0);
    TORCH_CHECK(t.size(1) >= 1 && t.size(1) < (int64_t(1) << 30), name,
                ": bad number of channels");
    C = int(t.size(1));
  }

  // other channels of the same rows
  Call(const Call& o, int channels)
      : ref(o.ref), apart(o.apart), dt(o.dt), rows(o.rows), C(channels) {}

  int64_t groups() const { return (int64_t(C) + 31) / 32; }

  void check_chunks(int64_t r = -1) const {
    const int64_t n = r < 0 ? rows : r;
    TORCH_CHECK(n * groups() * 4 < yams::kMaxChunks,
                "too many rows for one call: ", n, " x ", C);
  }

  yams::RowsDesc in(const Tensor& t, const char* name, int64_t r = -1) const {
    const int64_t want = r < 0 ? rows : r;
    TORCH_CHECK(t.device() == ref.device(), name, " is on another device");
    TORCH_CHECK(t.scalar_type() == ref.scalar_type(), name,
                " has another dtype than the rows");
    TORCH_CHECK(t.dim() == 2 && t.size(0) == want && t.size(1) == C, name,
                " has the wrong shape");
    TORCH_CHECK(C == 1 || t.stride(1) == 1, name,
                " needs unit stride along the channels");
    TORCH_CHECK(apart == ANY || want <= 1 || t.stride(0) <= kMaxStride, name,
                ": rows are too far apart");
    return {t.data_ptr(), t.stride(0)};
  }
  yams::RowsDesc in(const Opt& t, const char* name, int64_t r = -1) const {
    return t.has_value() ? in(*t, name, r) : yams::RowsDesc{};
  }
  // outputs are contiguous, in any number of axes
  void* out(const Tensor& t, const char* name, int64_t r = -1) const {
    TORCH_CHECK(t.device() == ref.device(), name, " is on another device");
    TORCH_CHECK(t.scalar_type() == ref.scalar_type(), name,
                " has another dtype than the rows");
    TORCH_CHECK(t.dim() >= 1 && t.size(-1) == C &&
                    t.numel() == (r < 0 ? rows : r) * C,
                name, " has the wrong shape");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    return t.data_ptr();
  }
  void* out(const Opt& t, const char* name, int64_t r = -1) const {
    return t.has_value() ? out(*t, name, r) : nullptr;
  }
  const float* param(const Opt& t, const char* name) const {
    return static_cast<const float*>(param(t, name, false));
  }
  // `narrow`: bf16
  const void* param(const Opt& t, const char* name, bool narrow) const {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == ref.device() &&
                    t->scalar_type() ==
                        (narrow ? torch::kBFloat16 : torch::kFloat32) &&
                    t->is_contiguous() && t->numel() == C,
                name, " must be fp32 [C] on the rows' device");
    return t->data_ptr();
  }
  yams::Kept kept(const Opt& codes, const Opt& exps, const char* name,
                  int64_t r = -1) const {
    TORCH_CHECK(codes.has_value() == exps.has_value(), name,
                ": codes and exponents go together");
    if (!codes.has_value()) return {};
    const int64_t want = r < 0 ? rows : r;
    TORCH_CHECK(codes->device() == ref.device() &&
                    exps->device() == ref.device(),
                name, ": codes are on another device");
    TORCH_CHECK(codes->scalar_type() == torch::kInt8 &&
                    codes->is_contiguous() && codes->numel() == want * C,
                name, ": codes must be int8 [rows, C]");
    TORCH_CHECK(exps->scalar_type() == torch::kUInt8 &&
                    exps->is_contiguous() &&
                    exps->numel() == want * groups(),
                name, ": exponents must be uint8 [rows, ceil(C / 32)]");
    return {reinterpret_cast<signed char*>(codes->data_ptr<int8_t>()),
            exps->data_ptr<uint8_t>()};
  }
  // fp32 sums, each C rounded up to four floats
  float* sums(const Opt& t, int count, const char* name) const {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == ref.device() &&
                    t->scalar_type() == torch::kFloat32 &&
                    t->is_contiguous() &&
                    t->numel() == int64_t(count) * ((C + 3) / 4 * 4),
                name, " must be fp32 with C rounded up to 4 per sum");
    return t->data_ptr<float>();
  }
  Tensor ws(int64_t floats) const {
    return floats == 0 ? Tensor()
                       : torch::empty({floats}, ref.options().dtype(
                                                    torch::kFloat32));
  }
};

}  // namespace

void pack_rows(const Tensor& x, const Tensor& codes, const Tensor& exps) {
  const Call c(x, "x", ANY);
  c10::cuda::CUDAGuard guard(x.device());
  c.check_chunks();
  yams::pack_rows(c.dt, c.in(x, "x"), c.kept(codes, exps, "x"), c.rows, c.C,
                  stream_of(x));
}

void unpack_rows(const Tensor& codes, const Tensor& exps, const Tensor& y) {
  const Call c(y, "y", ANY);
  c10::cuda::CUDAGuard guard(y.device());
  c.check_chunks();
  yams::unpack_rows(c.dt, c.kept(codes, exps, "y"), c.out(y, "y"), c.rows,
                    c.C, stream_of(y));
}

void act_rows_fwd(const Tensor& z, const Opt& bias, int64_t act,
                  const Tensor& y, const Opt& codes, const Opt& exps) {
  const Call c(z, "z", ANY);
  c10::cuda::CUDAGuard guard(z.device());
  c.check_chunks();
  yams::act_rows_fwd(c.dt, c.in(z, "z"), c.param(bias, "bias"), int(act),
                     c.out(y, "y"), c.kept(codes, exps, "z"), c.rows, c.C,
                     stream_of(z));
}

void act_rows_bwd(const Tensor& dy, const Opt& z, const Opt& codes,
                  const Opt& exps, const Opt& bias, int64_t act,
                  const Tensor& dz, const Opt& dbias) {
  const Call c(dy, "dy", ANY);
  c10::cuda::CUDAGuard guard(dy.device());
  TORCH_CHECK(z.has_value() != codes.has_value(),
              "act_rows_bwd takes z or its codes");
  Tensor ws;
  if (dbias.has_value()) ws = c.ws(yams::act_rows_ws(c.rows, c.C));
  yams::act_rows_bwd(c.dt, c.in(dy, "dy"), c.in(z, "z"),
                     c.kept(codes, exps, "z"), c.param(bias, "bias"),
                     int(act), c.out(dz, "dz"), c.sums(dbias, 1, "dbias"),
                     ws_ptr(ws), c.rows,
                     c.C, stream_of(dy));
}

// what join_fwd and join_bwd share; `gate_rows` is the gate's first size
static yams::JoinDesc join_desc(const Call& c, bool layer, bool post, bool next,
                         int64_t gate, int64_t gate_act, int64_t gate_rows,
                         double eps, double alpha, const Opt& w, const Opt& b,
                         const Opt& scale, const Opt& w2, const Opt& b2) {
  TORCH_CHECK(c.C <= yams::kMaxNormC, "norms take at most ",
              yams::kMaxNormC, " channels, got ", c.C);
  TORCH_CHECK(c.rows < (int64_t(1) << 31), "norms take fewer than 2^31 rows");
  TORCH_CHECK(gate >= 0 && gate <= 2, "bad gate mode");
  yams::JoinDesc d;
  d.rows = c.rows;
  d.C = c.C;
  d.layer = layer;
  d.post = post;
  d.next = next;
  d.gate = int(gate);
  d.gate_act = int(gate_act);
  d.eps = float(eps);
  d.alpha = float(alpha);
  if (gate == yams::GATE_GROUP) {
    TORCH_CHECK(gate_rows > 0 && c.rows % gate_rows == 0,
                "the gate's rows have to divide the rows");
    d.group_rows = std::max<int64_t>(1, c.rows / gate_rows);
  }
  d.w = c.param(w, "weight");
  d.b = c.param(b, "bias");
  d.scale = c.param(scale, "scale");
  d.w2 = c.param(w2, "next_weight");
  d.b2 = c.param(b2, "next_bias");
  return d;
}

void join_fwd(const Opt& h, const Tensor& x, const Opt& g, bool layer,
              bool post, bool next, int64_t gate, int64_t gate_act,
              double eps, double alpha, const Opt& w, const Opt& b,
              const Opt& scale, const Opt& w2, const Opt& b2, const Opt& y,
              const Opt& u, const Opt& hc, const Opt& he, const Opt& xc,
              const Opt& xe, const Opt& gc, const Opt& ge) {
  const Call c(x, "x");
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t gate_rows = g.has_value() ? g->size(0) : c.rows;
  TORCH_CHECK(g.has_value() == (gate != yams::GATE_NONE),
              "gate mode without a gate");
  TORCH_CHECK(!g.has_value() || h.has_value(), "a gate needs h");
  TORCH_CHECK(next == u.has_value() && h.has_value() == y.has_value(),
              "u goes with the next norm, y with h");
  TORCH_CHECK(next || h.has_value(), "neither h nor a next norm");
  yams::JoinDesc d = join_desc(c, layer, post, next, gate, gate_act,
                               gate_rows, eps, alpha, w, b, scale, w2, b2);
  // gates of runs are packed by themselves
  if (gate == yams::GATE_GROUP && gc.has_value()) c.check_chunks(gate_rows);
  TORCH_CHECK(xc.has_value() == (next && (hc.has_value() || !h.has_value()) &&
                                 (xc.has_value() || hc.has_value())) &&
                  hc.has_value() == (h.has_value() &&
                                     (xc.has_value() || hc.has_value())) &&
                  gc.has_value() == (g.has_value() && hc.has_value()),
              "all inputs that a gradient needs are kept in 8 bits or none");
  d.h = c.in(h, "h");
  d.x = c.in(x, "x");
  d.g = c.in(g, "gate", gate == yams::GATE_GROUP ? gate_rows : c.rows);
  d.hk = c.kept(hc, he, "h");
  d.xk = c.kept(xc, xe, "x");
  d.gk = c.kept(gc, ge, "gate", gate_rows);
  d.y = c.out(y, "y");
  d.u = c.out(u, "u");
  if (c.rows == 0) return;
  yams::join_fwd(c.dt, d, stream_of(x));
  if (gate == yams::GATE_GROUP && d.gk.codes != nullptr)
    yams::pack_rows(c.dt, d.g, d.gk, gate_rows, c.C, stream_of(x));
}

// `like`: a [rows, C] tensor with the rows' type (dy or du)
void join_bwd(const Tensor& like, const Opt& dy, const Opt& du, const Opt& h,
              const Opt& x, const Opt& g, const Opt& hc, const Opt& he,
              const Opt& xc, const Opt& xe, const Opt& gc, const Opt& ge,
              int64_t gate_rows, bool layer, bool post, bool next,
              int64_t gate, int64_t gate_act, double eps, double alpha,
              const Opt& w, const Opt& b, const Opt& scale, const Opt& w2,
              const Opt& b2, const Opt& dh, const Opt& dx, const Opt& dg,
              int64_t want, const Opt& sums) {
  const Call c(like, "dy");
  c10::cuda::CUDAGuard guard(like.device());
  const bool has_h = h.has_value() || hc.has_value();
  const bool has_g = g.has_value() || gc.has_value();
  TORCH_CHECK(has_g == (gate != yams::GATE_NONE) && (has_h || !has_g),
              "gate mode without a gate");
  TORCH_CHECK(next == du.has_value() &&
                  next == (x.has_value() || xc.has_value()),
              "the next norm's gradient needs x and du");
  TORCH_CHECK(next || has_h, "neither h nor a next norm");
  const bool kept = hc.has_value() || xc.has_value();
  TORCH_CHECK(!kept || (!h.has_value() && !x.has_value() && !g.has_value()),
              "inputs are all kept in 8 bits or none is");
  TORCH_CHECK(want >= 0 && want < 32 && (has_h || (want & 7) == 0) &&
                  (layer || (want & 20) == 0) && (next || (want & 24) == 0),
              "sums wanted of parameters that are not there");
  TORCH_CHECK((want != 0) == sums.has_value(), "want goes with sums");
  TORCH_CHECK(has_h || (!dh.has_value() && !dg.has_value()),
              "dh without h");
  yams::JoinDesc d = join_desc(c, layer, post, next, gate, gate_act,
                               gate_rows, eps, alpha, w, b, scale, w2, b2);
  const int64_t grows = gate == yams::GATE_GROUP ? gate_rows : c.rows;
  d.h = c.in(h, "h");
  d.x = c.in(x, "x");
  d.g = c.in(g, "gate", grows);
  d.hk = c.kept(hc, he, "h");
  d.xk = c.kept(xc, xe, "x");
  d.gk = c.kept(gc, ge, "gate", grows);
  d.dy = c.in(dy, "dy");
  d.du = c.in(du, "du");
  d.dh = c.out(dh, "dh");
  d.dx = c.out(dx, "dx");
  d.dg = c.out(dg, "dgate", grows);
  d.want = unsigned(want);
  d.sums = c.sums(sums, __builtin_popcount(d.want), "sums");
  if (c.rows == 0) return;
  Tensor ws = c.ws(yams::join_bwd_ws(c.dt, d));
  d.ws = ws_ptr(ws);
  yams::join_bwd(c.dt, d, stream_of(like));
}

namespace {

struct Weight {
  int dt;
  yams::RowsDesc rows;
  int N, K;
};

Weight weight_of(const Tensor& w, const Tensor& ref) {
  TORCH_CHECK(w.device() == ref.device(), "weight is on another device");
  const int dt = dtype_of(w, "weight");
  TORCH_CHECK(dt != kF16, "weight must be bf16 or fp32");
  TORCH_CHECK(w.dim() == 2 && (w.size(1) == 1 || w.stride(1) == 1),
              "weight must be [out, in] with unit stride along in");
  TORCH_CHECK(w.size(0) <= 1 || w.stride(0) <= kMaxStride,
              "weight: rows are too far apart");
  TORCH_CHECK(w.size(0) < (int64_t(1) << 30) &&
                  w.size(1) < (int64_t(1) << 30),
              "weight is too large");
  return {dt, {w.data_ptr(), w.stride(0)}, int(w.size(0)), int(w.size(1))};
}

// a launch has fewer than 2^32 threads: 256 for each tile of 64 x 64
void check_tiles(int64_t rows, int64_t cols) {
  TORCH_CHECK((rows + 63) / 64 * ((cols + 63) / 64) < (int64_t(1) << 24),
              "linear8: ", rows, " x ", cols, " is too large for one call");
}

void need_bf16(const Call& c, const char* name) {
  TORCH_CHECK(c.dt == kBf16, name, " must be bf16");
}

}  // namespace

void linear8_fwd(const Tensor& x, const Tensor& w, const Opt& bias,
                 const Tensor& y) {
  const Call cx(x, "x");
  c10::cuda::CUDAGuard guard(x.device());
  need_bf16(cx, "x");
  const Weight W = weight_of(w, x);
  TORCH_CHECK(W.K == cx.C, "linear8 shape mismatch");
  check_tiles(cx.rows, W.N);
  const Call cy(cx, W.N);
  Tensor ws = cx.ws(yams::linear8_ws(cx.rows, W.N, W.K, W.dt));
  const bool narrow =
      bias.has_value() && bias->scalar_type() == torch::kBFloat16;
  yams::linear8_fwd(cx.in(x, "x"), W.dt, W.rows, narrow ? kBf16 : kF32,
                    cy.param(bias, "bias", narrow), cy.out(y, "y"),
                    ws_ptr(ws), cx.rows, W.N, W.K, stream_of(x));
}

void linear8_dgrad(const Tensor& dy, const Tensor& w, const Tensor& dx) {
  const Call cy(dy, "dy");
  c10::cuda::CUDAGuard guard(dy.device());
  need_bf16(cy, "dy");
  const Weight W = weight_of(w, dy);
  TORCH_CHECK(W.N == cy.C, "linear8 shape mismatch");
  check_tiles(cy.rows, W.K);
  const Call cx(cy, W.K);
  Tensor ws = cx.ws(yams::linear8_ws(cx.rows, W.K, W.N, W.dt));
  yams::linear8_dgrad(cy.in(dy, "dy"), W.dt, W.rows, cx.out(dx, "dx"),
                      ws_ptr(ws), cx.rows, W.N, W.K, stream_of(dy));
}

void linear8_wgrad(const Tensor& dy, const Tensor& codes, const Tensor& exps,
                   const Tensor& dw) {
  const Call cy(dy, "dy");
  c10::cuda::CUDAGuard guard(dy.device());
  need_bf16(cy, "dy");
  TORCH_CHECK(dw.dim() == 2 && dw.is_contiguous() && dw.size(0) == cy.C &&
                  dw.device() == dy.device(),
              "dw must be [out, in], contiguous, on dy's device");
  const int odt = dtype_of(dw, "dw");
  TORCH_CHECK(odt != kF16, "dw must be bf16 or fp32");
  const int64_t K = dw.size(1), M = cy.rows;
  check_tiles(cy.C, K);
  TORCH_CHECK(codes.device() == dy.device() && exps.device() == dy.device() &&
                  codes.scalar_type() == torch::kInt8 &&
                  exps.scalar_type() == torch::kUInt8 &&
                  codes.is_contiguous() && exps.is_contiguous() &&
                  codes.numel() == M * K &&
                  exps.numel() == M * ((K + 31) / 32),
              "codes must be int8 [rows, in] with their exponents");
  const yams::Kept x{reinterpret_cast<signed char*>(codes.data_ptr<int8_t>()),
                     exps.data_ptr<uint8_t>()};
  const bool padded =
      int64_t(codes.storage().nbytes()) - codes.storage_offset() >= M * K + 7;
  Tensor ws = cy.ws(yams::linear8_ws(cy.C, K, M, kBf16,
                                     yams::linear8_loose(K, padded)));
  yams::linear8_wgrad(cy.in(dy, "dy"), x, padded, odt, dw.data_ptr(),
                      ws_ptr(ws), M, cy.C, int(K), stream_of(dy));
}

void row_sum(const Tensor& dy, const Tensor& db) {
  const Call c(dy, "dy", ANY);
  c10::cuda::CUDAGuard guard(dy.device());
  Tensor ws = c.ws(yams::row_sum_ws(c.rows, c.C));
  const bool narrow = db.scalar_type() == torch::kBFloat16;
  if (narrow)
    TORCH_CHECK(db.device() == dy.device() && db.is_contiguous() &&
                    db.numel() == c.C,
                "db must be [C] on dy's device");
  yams::row_sum(c.dt, c.in(dy, "dy"), narrow ? kBf16 : kF32,
                narrow ? db.data_ptr() : c.sums(db, 1, "db"), ws_ptr(ws),
                c.rows, c.C, stream_of(dy));
}

void register_rows(pybind11::module_& m) {
  m.def("pack_rows", &pack_rows);
  m.def("unpack_rows", &unpack_rows);
  m.def("act_rows_fwd", &act_rows_fwd);
  m.def("act_rows_bwd", &act_rows_bwd);
  m.def("join_fwd", &join_fwd);
  m.def("join_bwd", &join_bwd);
  m.def("linear8_fwd", &linear8_fwd);
  m.def("linear8_dgrad", &linear8_dgrad);
  m.def("linear8_wgrad", &linear8_wgrad);
  m.def("row_sum", &row_sum);
  register_rows_autograd(m);
}
