// Autograd of the row operators.  In C++ because their calls are short: a
// forward and a backward pass of a small row operator take 10..20 us of GPU
// time, and the same nodes written in Python took 70 us and more of the host
// (a bias + activation of 256 x 1280: 108 us a training step).
//
// The callers (ops/rows.py) have checked shapes, types and devices, and say
// whether inputs are kept in 8 bits.  Tensors arrive in any layout.

#include <torch/extension.h>

#include "bindings_rows.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> Opt;

Tensor plain(const Opt& t) { return t.has_value() ? *t : Tensor(); }
Opt maybe(const Tensor& t) { return t.defined() ? Opt(t) : Opt(); }

// [rows, C] with unit stride along C: a view where there is one
Tensor any_rows(const Tensor& x) {
  const int64_t c = x.size(-1);
  Tensor r = x.dim() == 2 ? x : x.reshape({x.numel() / c, c});
  if (c == 1 || r.stride(1) == 1) return r;
  // (contiguous() leaves an empty tensor as it is)
  return r.numel() == 0 ? torch::empty(r.sizes(), r.options())
                        : r.contiguous();
}

// ... and rows that norms and products reach (longer ones they refuse)
Tensor rows_view(const Tensor& x) {
  Tensor r = any_rows(x);
  return r.size(0) <= 1 || r.stride(0) <= yams::kMaxStride ? r
                                                           : r.contiguous();
}

Opt rows_opt(const Tensor& x) {
  return x.defined() ? Opt(rows_view(x)) : Opt();
}

// for the kernels only, so without a graph (the callers are in no-grad mode
// or want no gradient)
Opt param32(const Tensor& p) {
  if (!p.defined()) return {};
  if (p.scalar_type() == torch::kFloat32 && p.is_contiguous()) return p;
  return p.detach().to(torch::kFloat32).contiguous();
}

Tensor as_type(const Tensor& t, c10::ScalarType type) {
  return t.scalar_type() == type ? t : t.to(type);
}

// sum number k of a buffer of sums_of(), in a parameter's type
Tensor sum_at(const Tensor& sums, int64_t k, int64_t c,
              c10::ScalarType type) {
  return as_type(sums.size(0) == c ? sums
                                   : sums.narrow(0, (c + 3) / 4 * 4 * k, c),
                 type);
}

struct Codes {
  Tensor codes, exps;
};

// Eight bytes behind the codes: the weight gradient of an odd width reads
// whole chunks of eight (and does without where they are not there).
Codes empty_codes(const Tensor& rows) {
  const int64_t m = rows.size(0), c = rows.size(1);
  const auto o = rows.options().requires_grad(false);
  return {torch::empty({m * c + 8}, o.dtype(torch::kInt8))
              .as_strided({m, c}, {c, 1}),
          torch::empty({m, (c + 31) / 32}, o.dtype(torch::kUInt8))};
}

Tensor sums_of(const Tensor& like, int64_t count, int64_t rows) {
  const int64_t cp = (like.size(-1) + 3) / 4 * 4;
  const auto o = like.options().dtype(torch::kFloat32);
  return rows > 0 ? torch::empty({count * cp}, o)
                  : torch::zeros({count * cp}, o);
}

Tensor like(const Tensor& t) {  // contiguous, of its shape and type
  return torch::empty(t.sizes(), t.options());
}

// A tangent is refused here: the kernels would drop it, and an output without
// one counts as a constant.
bool wants_grad(std::initializer_list<Tensor> ts) {
  for (const Tensor& t : ts)
    TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(),
                "the row operators have no forward-mode derivative");
  if (!torch::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// The gradients are kernels and carry no graph: without this, a gradient of
// a gradient would silently lack them.
void once() {
  TORCH_CHECK(!torch::GradMode::is_enabled(),
              "the row operators can be differentiated once: run their "
              "backward pass without create_graph");
}

// --- bias + activation ---------------------------------------------------

Tensor bias_act_run(const Tensor& rows, const Tensor& z, const Tensor& bias,
                    int64_t act, const Codes& k) {
  Tensor y = like(z);
  if (rows.size(0) > 0)
    act_rows_fwd(rows, param32(bias), act, y,
                 maybe(k.codes), maybe(k.exps));
  return y;
}

struct BiasActFn : Function<BiasActFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z,
                        const Opt& bias_opt, int64_t act, bool keep) {
    const Tensor rows = any_rows(z), bias = plain(bias_opt);
    Codes k;
    if (keep) k = empty_codes(rows);
    Tensor y = bias_act_run(rows, z, bias, act, k);
    ctx->save_for_backward({keep ? Tensor() : z, k.codes, k.exps, bias});
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    once();
    const variable_list s = ctx->get_saved_variables();
    const Tensor &z = s[0], &bias = s[3];
    const Tensor rows = any_rows(dys[0]);
    const int64_t m = rows.size(0), c = rows.size(1);
    Tensor dz = like(dys[0]), sums, db;
    if (bias.defined() && ctx->needs_input_grad(1))
      sums = sums_of(rows, 1, m);
    if (m > 0)
      act_rows_bwd(rows, z.defined() ? Opt(any_rows(z)) : Opt(), maybe(s[1]), maybe(s[2]),
                   param32(bias), ctx->saved_data["act"].toInt(),
                   dz, maybe(sums));
    if (sums.defined()) db = sum_at(sums, 0, c, bias.scalar_type());
    return {dz, db, Tensor(), Tensor()};
  }
};

Tensor bias_act(const Tensor& z, const Opt& bias, int64_t act, bool save8) {
  const Tensor b = plain(bias);
  if (!wants_grad({z, b}))
    return bias_act_run(any_rows(z), z, b, act, Codes());
  return BiasActFn::apply(z, bias, act, save8);
}

// --- FC layer on a kept input ----------------------------------------------

// bf16 or fp32 (which holds what other types have beyond bf16)
Tensor weight_view(const Tensor& w) {
  const auto t = w.scalar_type();
  return rows_view(t == torch::kBFloat16 || t == torch::kFloat32
                       ? w
                       : w.detach().to(torch::kFloat32));
}

std::vector<int64_t> with_last(const Tensor& t, int64_t n) {
  std::vector<int64_t> s = t.sizes().vec();
  s.back() = n;
  return s;
}

// fp32 or bf16
Opt linear_bias(const Tensor& b) {
  return b.defined() && b.scalar_type() == torch::kBFloat16 &&
                 b.is_contiguous()
             ? Opt(b)
             : param32(b);
}

Tensor linear8_run(const Tensor& rows, const Tensor& x, const Tensor& w,
                   const Tensor& bias) {
  const int64_t n = w.size(0), m = rows.size(0);
  Tensor y = torch::empty(with_last(x, n), rows.options());
  if (m > 0)
    linear8_fwd(rows, weight_view(w), linear_bias(bias), y);
  return y;
}

struct Linear8Fn : Function<Linear8Fn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const Tensor& weight, const Opt& bias_opt,
                        bool want_dw) {
    const Tensor bias = plain(bias_opt);
    const Tensor rows = rows_view(as_type(x, torch::kBFloat16));
    Tensor y = linear8_run(rows, x, weight, bias);
    Codes k;
    if (want_dw) {
      k = empty_codes(rows);
      if (rows.size(0) > 0) pack_rows(rows, k.codes, k.exps);
    }
    ctx->save_for_backward({k.codes, k.exps, weight, bias});
    ctx->saved_data["dtype"] = int64_t(x.scalar_type());
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    once();
    const variable_list s = ctx->get_saved_variables();
    const Tensor &weight = s[2], &bias = s[3];
    const Tensor rows = rows_view(as_type(dys[0], torch::kBFloat16));
    const int64_t m = rows.size(0), n = rows.size(1), k = weight.size(1);
    Tensor dx, dw, db;
    if (ctx->needs_input_grad(0)) {
      dx = torch::empty(with_last(dys[0], k), rows.options());
      if (m > 0) linear8_dgrad(rows, weight_view(weight), dx);
      dx = as_type(dx, c10::ScalarType(ctx->saved_data["dtype"].toInt()));
    }
    if (ctx->needs_input_grad(1)) {
      const auto t = weight.scalar_type();
      const auto o = rows.options().dtype(
          t == torch::kBFloat16 ? torch::kBFloat16 : torch::kFloat32);
      dw = m > 0 ? torch::empty({n, k}, o) : torch::zeros({n, k}, o);
      if (m > 0) linear8_wgrad(rows, s[0], s[1], dw);
      dw = as_type(dw, t);
    }
    if (bias.defined() && ctx->needs_input_grad(2)) {
      const auto t = bias.scalar_type();
      Tensor sums = t == torch::kBFloat16 && m > 0
                        ? torch::empty({n}, rows.options())
                        : sums_of(rows, 1, m);
      if (m > 0) row_sum(rows, sums);
      db = sum_at(sums, 0, n, t);
    }
    return {dx, dw, db, Tensor()};
  }
};

Tensor linear8(const Tensor& x, const Tensor& weight, const Opt& bias) {
  const Tensor b = plain(bias);
  if (!wants_grad({x, weight, b}))
    return linear8_run(rows_view(x.detach().to(torch::kBFloat16)), x, weight,
                       b);
  return Linear8Fn::apply(x, weight, bias, weight.requires_grad());
}

// --- norms -----------------------------------------------------------------

struct JoinConfig {
  bool layer, post, next;
  int64_t gate, gate_act;
  double eps, alpha;
};

struct JoinOut {
  Tensor y, u;
  Codes h, x, g;
};

JoinOut join_run(const Tensor& h, const Tensor& x, const Tensor& gate,
                 const Tensor& w, const Tensor& b, const Tensor& scale,
                 const Tensor& w2, const Tensor& b2, const JoinConfig& c,
                 bool keep) {
  const Tensor xr = rows_view(x);
  const Opt hr = rows_opt(h), gr = rows_opt(gate);
  JoinOut o;
  if (h.defined()) o.y = like(x);
  if (c.next) o.u = like(x);
  if (keep) {
    if (c.next) o.x = empty_codes(xr);
    if (hr.has_value()) o.h = empty_codes(*hr);
    if (gr.has_value()) o.g = empty_codes(*gr);
  }
  if (xr.size(0) > 0)
    join_fwd(hr, xr, gr, c.layer, c.post, c.next, c.gate, c.gate_act, c.eps,
             c.alpha, param32(w), param32(b), param32(scale), param32(w2),
             param32(b2), maybe(o.y), maybe(o.u),
             maybe(o.h.codes), maybe(o.h.exps), maybe(o.x.codes),
             maybe(o.x.exps), maybe(o.g.codes), maybe(o.g.exps));
  return o;
}

// h undefined: a norm alone, u = N2(x)
struct JoinFn : Function<JoinFn> {
  static variable_list forward(AutogradContext* ctx, const Opt& h_opt,
                               const Tensor& x, const Opt& gate_opt,
                               const Opt& w_opt, const Opt& b_opt,
                               const Opt& scale_opt, const Opt& w2_opt,
                               const Opt& b2_opt, bool layer, bool post,
                               bool next, int64_t gmode, int64_t gact,
                               double eps, double alpha, bool keep) {
    const Tensor h = plain(h_opt), gate = plain(gate_opt), w = plain(w_opt),
                 b = plain(b_opt), scale = plain(scale_opt),
                 w2 = plain(w2_opt), b2 = plain(b2_opt);
    // which of the tensors are there: needs_input_grad counts those
    const Tensor all[] = {h, x, gate, w, b, scale, w2, b2};
    int64_t there = 0;
    for (int i = 0; i < 8; ++i) there |= int64_t(all[i].defined()) << i;
    const JoinConfig c{layer, post, next, gmode, gact, eps, alpha};
    JoinOut o = join_run(h, x, gate, w, b, scale, w2, b2, c, keep);
    ctx->save_for_backward({keep ? Tensor() : h,
                            keep || !next ? Tensor() : x,
                            keep ? Tensor() : gate, o.h.codes, o.h.exps,
                            o.x.codes, o.x.exps, o.g.codes, o.g.exps, w, b,
                            scale, w2, b2});
    ctx->saved_data["flags"] =
        int64_t(layer) | int64_t(post) << 1 | int64_t(next) << 2 |
        int64_t(h.defined()) << 3 | gmode << 4 | gact << 8 | there << 16;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["alpha"] = alpha;
    if (gate.defined()) ctx->saved_data["gate"] = gate.sizes().vec();
    ctx->set_materialize_grads(false);
    if (!h.defined()) return {o.u};
    if (!next) return {o.y};
    return {o.y, o.u};
  }

  static variable_list backward(AutogradContext* ctx, variable_list douts) {
    once();
    const variable_list s = ctx->get_saved_variables();
    const int64_t f = ctx->saved_data["flags"].toInt();
    const bool layer = f & 1, post = f & 2, has_h = f & 8;
    bool next = f & 4;
    const int64_t gmode = f >> 4 & 15, gact = f >> 8 & 255, there = f >> 16;
    auto needed = [&](int i) {
      return (there >> i & 1) != 0 &&
             ctx->needs_input_grad(size_t(
                 __builtin_popcountll(there & ((int64_t(1) << i) - 1))));
    };
    variable_list out(16);
    Tensor dy, du;
    if (has_h) dy = douts[0];
    if (next) du = douts[has_h ? 1 : 0];
    const Tensor& ref = dy.defined() ? dy : du;
    if (!ref.defined()) return out;
    if (!du.defined()) next = false;  // no part in this gradient
    const Tensor &w = s[9], &b = s[10], &scale = s[11], &w2 = s[12],
                 &b2 = s[13];
    const Tensor refr = rows_view(ref);
    const int64_t m = refr.size(0), c = refr.size(1);
    Tensor dh, dx, dg;
    if (needed(0)) dh = like(ref);
    if (needed(1)) dx = like(ref);
    int64_t grows = m;
    if (gmode != yams::GATE_NONE) {
      const auto gs = ctx->saved_data["gate"].toIntVector();
      if (gmode == yams::GATE_GROUP) grows = gs[0];
      if (needed(2))
        dg = m > 0 ? torch::empty(gs, ref.options())
                   : torch::zeros(gs, ref.options());
    }
    const Tensor* params[] = {&scale, &w, &b, &w2, &b2};
    const int at[] = {5, 3, 4, 6, 7};  // among the forward's tensors
    int64_t want = 0, count = 0;
    for (int i = 0; i < 5; ++i)
      if (needed(at[i]) && (next || i < 3)) {
        want |= int64_t(1) << i;
        ++count;
      }
    Tensor sums;
    if (count > 0) sums = sums_of(refr, count, m);
    if (m > 0)
      join_bwd(refr, dy.defined() ? Opt(rows_view(dy)) : Opt(),
               next ? Opt(rows_view(du)) : Opt(), rows_opt(s[0]),
               next ? rows_opt(s[1]) : Opt(), rows_opt(s[2]), maybe(s[3]),
               maybe(s[4]), next ? maybe(s[5]) : Opt(),
               next ? maybe(s[6]) : Opt(), maybe(s[7]), maybe(s[8]), grows,
               layer, post, next, gmode, gact,
               ctx->saved_data["eps"].toDouble(),
               ctx->saved_data["alpha"].toDouble(), param32(w), param32(b),
               param32(scale), next ? param32(w2) : Opt(),
               next ? param32(b2) : Opt(), maybe(dh), maybe(dx), maybe(dg),
               want, maybe(sums));
    out[0] = dh;
    out[1] = dx;
    out[2] = dg;
    for (int i = 0, k = 0; i < 5; ++i)
      if (want >> i & 1)
        out[at[i]] = sum_at(sums, k++, c, params[i]->scalar_type());
    return out;
  }
};

std::vector<Tensor> join(const Opt& h, const Tensor& x, const Opt& gate,
                         const Opt& w, const Opt& b, const Opt& scale,
                         const Opt& w2, const Opt& b2, bool layer, bool post,
                         bool next, int64_t gmode, int64_t gact, double eps,
                         double alpha, bool save8) {
  const Tensor H = plain(h), G = plain(gate), W = plain(w), B = plain(b),
               S = plain(scale), W2 = plain(w2), B2 = plain(b2);
  if (!wants_grad({H, x, G, W, B, S, W2, B2})) {
    const JoinConfig c{layer, post, next, gmode, gact, eps, alpha};
    JoinOut o = join_run(H, x, G, W, B, S, W2, B2, c, false);
    std::vector<Tensor> r;
    if (H.defined()) r.push_back(o.y);
    if (next) r.push_back(o.u);
    return r;
  }
  return JoinFn::apply(h, x, gate, w, b, scale, w2, b2, layer, post, next,
                       gmode, gact, eps, alpha, save8);
}

// --- codec -----------------------------------------------------------------

std::pair<Tensor, Tensor> pack(const Tensor& x) {
  const Tensor rows = any_rows(x.requires_grad() ? x.detach() : x);
  Codes k = empty_codes(rows);
  if (rows.size(0) > 0) pack_rows(rows, k.codes, k.exps);
  return {k.codes, k.exps};
}

// the values that codes [rows, C] stand for, as a tensor of `shape`
Tensor unpack(const Tensor& codes, const Tensor& exps, c10::ScalarType type,
              c10::IntArrayRef shape) {
  Tensor y = torch::empty(codes.sizes(), codes.options().dtype(type));
  if (y.numel() > 0) unpack_rows(codes, exps, y);
  return y.sizes() == shape ? y : y.view(shape);
}

}  // namespace

void register_rows_autograd(pybind11::module_& m) {
  m.def("pack", &pack);
  m.def("unpack", &unpack);
  m.def("bias_act", &bias_act);
  m.def("linear8", &linear8);
  m.def("join", &join);
}
