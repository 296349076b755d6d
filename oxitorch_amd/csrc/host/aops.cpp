// Differentiable ops: restates crates/oxi-autograd/src/ops.rs over device
// tensors, plus the fused hot-path nodes (one graph node and one kernel per
// direction for rms_norm, layer_norm, gelu, silu, softmax/log_softmax,
// cross_entropy and the embedding gather).
//
// Gradients produced inside VJPs keep the common dense layout of their
// operands (result_strides): a gradient flowing through a permuted view stays
// permuted, so the permute VJP hands the next node a contiguous tensor.
#include <algorithm>
#include <atomic>
#include <cstdlib>
#include <cstring>

#include "host.h"

namespace oxt {
namespace aops {

namespace {

using Grads = std::vector<std::optional<Tensor>>;

Tensor un(int op, const Tensor& a) { return t_unary(op, a, true); }
Tensor bin(int op, const Tensor& a, const Tensor& b) { return t_binary(op, a, b, true); }
Tensor ones_of(const Tensor& t) { return t_scalar_full(t.shape, 1.0f, t.dev()); }

}  // namespace

// ---- binary (ops.rs:37-114) -------------------------------------------------------

Var add(const Var& a, const Var& b) {
  Tensor out = t_binary(OXI_BINARY_ADD, a.value(), b.value());
  return Var::op(out, "add", {a, b}, [](const Tensor& g, const std::vector<bool>& need) -> Grads {
    return {need[0] ? std::optional<Tensor>(g) : std::nullopt, need[1] ? std::optional<Tensor>(g) : std::nullopt};
  });
}

Var sub(const Var& a, const Var& b) {
  Tensor out = t_binary(OXI_BINARY_SUB, a.value(), b.value());
  return Var::op(out, "sub", {a, b}, [](const Tensor& g, const std::vector<bool>& need) -> Grads {
    Grads r(2);
    if (need[0]) r[0] = g;
    if (need[1]) r[1] = un(OXI_UNARY_NEG, g);
    return r;
  });
}

Var mul(const Var& a, const Var& b) {
  Tensor out = t_binary(OXI_BINARY_MUL, a.value(), b.value());
  Tensor av = a.value(), bv = b.value();
  return Var::op(out, "mul", {a, b}, [av, bv](const Tensor& g, const std::vector<bool>& need) -> Grads {
    Grads r(2);
    if (need[0]) r[0] = bin(OXI_BINARY_MUL, g, bv);
    if (need[1]) r[1] = bin(OXI_BINARY_MUL, g, av);
    return r;
  });
}

Var div(const Var& a, const Var& b) {
  Tensor out = t_binary(OXI_BINARY_DIV, a.value(), b.value());
  Tensor av = a.value(), bv = b.value();
  return Var::op(out, "div", {a, b}, [av, bv](const Tensor& g, const std::vector<bool>& need) -> Grads {
    Grads r(2);
    if (need[0]) r[0] = bin(OXI_BINARY_DIV, g, bv);
    if (need[1]) {
      Tensor b2 = bin(OXI_BINARY_MUL, bv, bv);
      r[1] = un(OXI_UNARY_NEG, bin(OXI_BINARY_DIV, bin(OXI_BINARY_MUL, g, av), b2));
    }
    return r;
  });
}

Var pow(const Var& a, const Var& b) {
  Tensor out = t_binary(OXI_BINARY_POW, a.value(), b.value());
  Tensor av = a.value(), bv = b.value();
  return Var::op(out, "pow", {a, b}, [av, bv](const Tensor& g, const std::vector<bool>& need) -> Grads {
    Grads r(2);
    if (need[0]) {
      Tensor bm1 = bin(OXI_BINARY_ADD, bv, t_scalar_full({}, -1.0f, bv.dev()));
      Tensor apow = bin(OXI_BINARY_POW, av, bm1);
      r[0] = bin(OXI_BINARY_MUL, bin(OXI_BINARY_MUL, g, bv), apow);
    }
    if (need[1]) {
      Tensor o = bin(OXI_BINARY_POW, av, bv);
      r[1] = bin(OXI_BINARY_MUL, bin(OXI_BINARY_MUL, g, o), un(OXI_UNARY_LOG, av));
    }
    return r;
  });
}

// ---- unary (ops.rs:126-268) --------------------------------------------------------

namespace {
// unary_generic: gx = g * dfdx(x), dfdx recomputed from the saved input
Var unary_generic(const Var& x, int fwd_op, const char* name, std::function<Tensor(const Tensor&)> dfdx) {
  Tensor out = t_unary(fwd_op, x.value());
  Tensor xv = x.value();
  return Var::op(out, name, {x}, [xv, dfdx](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    return {bin(OXI_BINARY_MUL, g, dfdx(xv))};
  });
}
}  // namespace

Var neg(const Var& x) {
  Tensor out = t_unary(OXI_UNARY_NEG, x.value());
  return Var::op(out, "neg", {x}, [](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    return {un(OXI_UNARY_NEG, g)};
  });
}

Var abs(const Var& x) {
  return unary_generic(x, OXI_UNARY_ABS, "abs", [](const Tensor& t) { return un(OXI_UNARY_SIGN, t); });
}

Var exp(const Var& x) {
  return unary_generic(x, OXI_UNARY_EXP, "exp", [](const Tensor& t) { return un(OXI_UNARY_EXP, t); });
}

Var log(const Var& x) {
  return unary_generic(x, OXI_UNARY_LOG, "log",
                       [](const Tensor& t) { return bin(OXI_BINARY_DIV, ones_of(t), t); });
}

Var sqrt(const Var& x) {
  return unary_generic(x, OXI_UNARY_SQRT, "sqrt", [](const Tensor& t) {
    Tensor denom = bin(OXI_BINARY_MUL, un(OXI_UNARY_SQRT, t), t_scalar_full(t.shape, 2.0f, t.dev()));
    return bin(OXI_BINARY_DIV, ones_of(t), denom);
  });
}

Var tanh(const Var& x) {
  return unary_generic(x, OXI_UNARY_TANH, "tanh", [](const Tensor& t) {
    Tensor th = un(OXI_UNARY_TANH, t);
    return bin(OXI_BINARY_SUB, ones_of(t), bin(OXI_BINARY_MUL, th, th));
  });
}

Var sigmoid(const Var& x) {
  return unary_generic(x, OXI_UNARY_SIGMOID, "sigmoid", [](const Tensor& t) {
    Tensor s = un(OXI_UNARY_SIGMOID, t);
    return bin(OXI_BINARY_MUL, s, bin(OXI_BINARY_SUB, ones_of(t), s));
  });
}

Var relu(const Var& x) {  // ops.rs:254-268: grad mask x > 0
  Tensor out = t_unary(OXI_UNARY_RELU, x.value());
  Tensor mask = t_binary(OXI_CMP_GT, x.value(), t_scalar_full(x.value().shape, 0.0f, x.value().dev()));
  return Var::op(out, "relu", {x}, [mask](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    return {bin(OXI_BINARY_MUL, g, mask)};
  });
}

// ---- reductions (ops.rs:327-388, 679-737) ---------------------------------------------

namespace {
// normalize_reduce_grad + expand_to: the upstream grad as a view of x's shape.
Tensor expand_grad(const Tensor& g, const Shape& x_shape, int dim) {
  if (g.shape == x_shape) return g;
  std::vector<int64_t> padded(g.shape.begin(), g.shape.end());
  if (g.shape.size() + 1 == x_shape.size()) padded.insert(padded.begin() + std::min<size_t>(dim, padded.size()), 1);
  Tensor r = t_reshape(g, padded);
  std::vector<int64_t> full(x_shape.size(), 1);
  const size_t tail = x_shape.size() - r.shape.size();
  for (size_t i = tail; i < x_shape.size(); ++i) full[i] = r.shape[i - tail];
  return t_broadcast_to(t_reshape(r, full), x_shape);
}
}  // namespace

Var reduce(const Var& x, Reduce kind, int64_t dim, bool keepdim) {
  Tensor out = t_reduce(kind, x.value(), dim, keepdim);
  const int d = normalize_dim(dim, x.value().ndim());
  const Shape xs = x.value().shape;
  Tensor xv = x.value();
  switch (kind) {
    case Reduce::Sum:
      return Var::op(out, "sum", {x}, [xs, d](const Tensor& g, const std::vector<bool>& need) -> Grads {
        if (!need[0]) return {std::nullopt};
        return {expand_grad(g, xs, d)};
      });
    case Reduce::Mean: {
      const float n = (float)xs[d];
      return Var::op(out, "mean", {x}, [xs, d, n](const Tensor& g, const std::vector<bool>& need) -> Grads {
        if (!need[0]) return {std::nullopt};
        Tensor up = expand_grad(g, xs, d);
        return {t_binary(OXI_BINARY_MUL, up, t_scalar_full(xs, 1.0f / n, up.dev()))};
      });
    }
    case Reduce::Max:
    case Reduce::Min: {
      // winners captured at forward; the grad goes to the single first winner
      Tensor arg = t_reduce(kind == Reduce::Max ? Reduce::ArgMax : Reduce::ArgMin, xv, d, true);
      return Var::op(out, "maxmin", {x}, [xs, d, arg](const Tensor& g, const std::vector<bool>& need) -> Grads {
        if (!need[0]) return {std::nullopt};
        Tensor up = expand_grad(g, xs, d);
        std::vector<float> pos((size_t)xs[d]);
        for (int64_t k = 0; k < xs[d]; ++k) pos[(size_t)k] = (float)k;
        Shape ps(xs.size(), 1);
        ps[d] = xs[d];
        Tensor positions = t_from_host(pos.data(), ps, Dev::Hip);
        Tensor mask = t_binary(OXI_CMP_EQ, t_broadcast_to(positions, xs), t_broadcast_to(arg, xs));
        return {t_binary(OXI_BINARY_MUL, mask, up)};
      });
    }
    case Reduce::Norm:
      return Var::op(out, "norm", {x}, [xs, d, xv](const Tensor& g, const std::vector<bool>& need) -> Grads {
        if (!need[0]) return {std::nullopt};
        Tensor up = expand_grad(g, xs, d);
        Tensor n = t_reduce(Reduce::Norm, xv, d, true);
        Tensor safe = t_binary(OXI_BINARY_ADD, n, t_scalar_full(n.shape, 1e-12f, n.dev()));
        Tensor ratio = t_binary(OXI_BINARY_DIV, xv, safe);
        return {t_binary(OXI_BINARY_MUL, up, ratio)};
      });
    default:
      err_notimpl("argmax/argmin are integer outputs and have no gradient");
  }
}

// ---- views (ops.rs:396-488) -------------------------------------------------------

Var reshape(const Var& x, const std::vector<int64_t>& shape) {
  Tensor out = t_reshape(x.value(), shape);
  const Shape orig = x.value().shape;
  return Var::op(out, "reshape", {x}, [orig](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    return {t_reshape(g, orig)};
  });
}

Var permute(const Var& x, const std::vector<int64_t>& order) {
  Tensor out = t_permute(x.value(), order);
  std::vector<int64_t> inv(order.size());
  for (size_t i = 0; i < order.size(); ++i) inv[(size_t)normalize_dim(order[i], (int)order.size())] = (int64_t)i;
  Var v = Var::op(out, "permute", {x}, [inv](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    return {t_permute(g, inv)};
  });
  if (v.node->op)
    for (int64_t o : order) v.node->perm.push_back((int64_t)normalize_dim(o, (int)order.size()));
  return v;
}

Var transpose(const Var& x) {
  Tensor out = t_transpose(x.value());
  Var v = Var::op(out, "transpose", {x}, [](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    return {t_transpose(g)};
  });
  if (v.node->op) v.node->perm = {1, 0};
  return v;
}

Var broadcast_to(const Var& x, const Shape& shape) {
  Tensor out = t_broadcast_to(x.value(), shape);
  const Shape xs = x.value().shape;
  return Var::op(out, "broadcast_to", {x}, [xs](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    return {unbroadcast(g, xs)};
  });
}

// The reference's narrow_dim0 (ops.rs:428-442) pads the gradient with zero
// rows; here the window of a zero tensor is written through a strided view.
Var narrow(const Var& x, int64_t dim, int64_t lo, int64_t hi, int64_t by) {
  Tensor out = t_narrow(x.value(), dim, lo, hi, by);
  const Shape xs = x.value().shape;
  return Var::op(out, "narrow", {x}, [xs, dim, lo, hi, by](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    Tensor z = t_zeros(xs, g.dev());
    t_copy_into(t_narrow(z, dim, lo, hi, by), g);
    return {z};
  });
}

// ---- index_select (ops.rs:498-517, 741-769) -----------------------------------------

// The VJP's id sort is queued at forward time (oxi_index_select_bwd_plan):
// up to 32768 ids in order, more on the library's second stream, where the sort
// overlaps the forward; the backward only waits for it and runs the segment sums.
Var index_select(const Var& x, int64_t dim, const std::vector<int64_t>& indices) {
  if (!is_grad_enabled() || !x.requires_grad()) return Var::leaf(t_index_select(x.value(), dim, indices), false);
  if (x.value().ndim() == 0) err_invalid("dim " + std::to_string(dim) + " out of range for 0-D tensor");
  const int d = normalize_dim(dim, x.value().ndim());
  const Shape xs = x.value().shape;
  auto ids = device_i64(resolve_indices(indices, xs[d], d));
  const int64_t n = (int64_t)indices.size();
  // queued before the gather: a sort on the second stream overlaps it too
  void* raw = nullptr;
  hip_check(oxi_index_select_bwd_plan(static_cast<const int64_t*>(ids->ptr), n, xs[d], &raw));
  std::shared_ptr<void> plan(raw, [ids](void* p) { (void)oxi_index_select_bwd_plan_free(p); });
  Tensor out = t_index_select_dev(x.value(), d, ids, n);
  return Var::op(out, "index_select", {x}, [xs, d, plan](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    Tensor gc = t_contiguous(g);
    int64_t outer = 1, inner = 1;
    for (int i = 0; i < d; ++i) outer *= xs[i];
    for (size_t i = d + 1; i < xs.size(); ++i) inner *= xs[i];
    Tensor grad = Tensor::empty(xs, Dev::Hip);
    hip_check(oxi_index_select_bwd_apply(plan.get(), gc.data(), outer, inner, grad.data()));
    return {grad};
  });
}

// aops::scatter_dim0 (crates/oxi-autograd/src/ops.rs:531-600): the written
// rows of base get no gradient, the last writer of each row gets that row's.
Var scatter_dim0(const Var& base, const std::vector<int64_t>& indices, const Var& values) {
  Tensor out = t_scatter_dim0(base.value(), indices, values.value());
  const Shape bs = base.value().shape;
  const Shape vs = values.value().shape;
  const int64_t rows = bs[0];
  int64_t inner = 1;
  for (size_t d = 1; d < bs.size(); ++d) inner *= bs[d];
  auto ids = device_i64(resolve_indices(indices, rows, 0));
  const int64_t n = (int64_t)indices.size();
  return Var::op(out, "scatter_dim0", {base, values},
                 [bs, vs, rows, inner, ids, n](const Tensor& g, const std::vector<bool>& need) -> Grads {
                   std::optional<Tensor> gb, gv;
                   if (need[0]) gb = Tensor::empty(bs, Dev::Hip);
                   if (need[1]) gv = Tensor::empty(vs, Dev::Hip);
                   if (gb || gv) {
                     Tensor gc = t_contiguous(g);
                     hip_check(oxi_scatter_rows_bwd(gc.data(), rows, inner, static_cast<const int64_t*>(ids->ptr), n,
                                                    gb ? gb->data() : nullptr, gv ? gv->data() : nullptr));
                   }
                   return {gb, gv};
                 });
}

// aops::masked_select (crates/oxi-autograd/src/ops.rs:609-667): each pick's
// gradient goes back to its x element, accumulating over broadcast points.
// The VJP keeps the forward's selection record (one bit per grid point)
// instead of x and the mask.
Var masked_select(const Var& x, const Var& mask) {
  const bool record = is_grad_enabled() && x.requires_grad();
  std::shared_ptr<Storage> rec;
  Tensor out = t_masked_select(x.value(), mask.value(), record ? &rec : nullptr);
  const Shape xshape = x.value().shape;
  const Shape grid = broadcast_shapes(xshape, mask.value().shape);
  const int64_t count = out.numel();
  return Var::op(out, "masked_select", {x},
                 [rec, xshape, grid, count](const Tensor& g, const std::vector<bool>& need) -> Grads {
                   if (!need[0]) return {std::nullopt};
                   if (!rec) err_other("masked_select: the forward kept no selection record");
                   // row-major strides of x's own shape on the grid, 0 where x
                   // broadcasts (a missing or size-1 dim): x_flat_str, ops.rs:628-634
                   const Shape rm = row_major_strides(xshape);
                   const size_t lead = grid.size() - xshape.size();
                   Shape gxs(grid.size(), 0);
                   for (size_t d = lead; d < grid.size(); ++d)
                     if (xshape[d - lead] != 1) gxs[d] = rm[d - lead];
                   Tensor gc = t_contiguous(g);
                   Tensor gx = Tensor::empty(xshape, Dev::Hip);
                   hip_check(oxi_masked_select_bwd(rec->ptr, grid.data(), (int)grid.size(), gc.data(), count,
                                                   gx.data(), gxs.data(), gx.numel()));
                   return {gx};
                 });
}

Var embedding(const std::vector<int64_t>& indices, const Var& weight) {
  return index_select(weight, 0, indices);
}

// ---- fused norms (functional.py:227-240) ----------------------------------------------

NormVjp norm_vjp_mode() {
  const char* e = std::getenv("OXI_NORM_VJP");
  if (!e || !*e || std::strcmp(e, "ref") == 0) return NormVjp::Ref;
  if (std::strcmp(e, "exact") == 0) return NormVjp::Exact;
  err_invalid(std::string("OXI_NORM_VJP must be \"ref\" or \"exact\", got \"") + e + "\"");
}

namespace {
int64_t last_dim(const Tensor& x, const char* what) {
  if (x.ndim() == 0) err_invalid(std::string(what) + " needs at least one dim");
  return x.shape.back();
}
void check_param(const Tensor& p, int64_t H, const char* what) {
  if (p.ndim() != 1 || p.shape[0] != H) err_shape(fmt_shape(p.shape), fmt_shape({H}));
  (void)what;
}
}  // namespace

Var rms_norm(const Var& x, const Var& w, float eps, NormVjp mode) {
  const int64_t H = last_dim(x.value(), "rms_norm");
  check_param(w.value(), H, "weight");
  Tensor xc = t_contiguous(x.value());
  Tensor wc = t_contiguous(w.value());
  const int64_t rows = H ? xc.numel() / H : 0;
  Tensor y = Tensor::empty(xc.shape, Dev::Hip);
  Tensor rstd = Tensor::empty({rows}, Dev::Hip);
  hip_check(oxi_rms_norm_fwd(xc.data(), wc.data(), y.data(), rstd.data(), rows, H, eps));
  auto saved = std::make_shared<NormSaved>();
  saved->x = xc;
  saved->w = wc;
  saved->has_w = true;
  saved->rstd = rstd;
  saved->rows = rows;
  saved->H = H;
  saved->mode = (int)mode;
  saved->wi = 1;
  Var v = Var::op(y, "rms_norm", {x, w}, [xc, wc, rstd, rows, H, mode](const Tensor& g, const std::vector<bool>& need) {
    Grads r(2);
    Tensor gc = t_contiguous(g);
    Tensor dx, dw;
    if (need[0]) dx = Tensor::empty(xc.shape, Dev::Hip);
    if (need[1]) dw = Tensor::empty({H}, Dev::Hip);
    if (!need[0] && !need[1]) return r;
    hip_check(oxi_rms_norm_bwd(xc.data(), wc.data(), rstd.data(), gc.data(), need[0] ? dx.data() : nullptr,
                               need[1] ? dw.data() : nullptr, rows, H, (int)mode));
    if (need[0]) r[0] = dx;
    if (need[1]) r[1] = dw;
    return r;
  });
  if (v.node->op) v.node->norm = std::move(saved);
  return v;
}

std::pair<Var, Var> add_rms_norm(const Var& x, const Var& r, const Var& w, float eps, NormVjp mode) {
  const int64_t H = last_dim(x.value(), "add_rms_norm");
  if (r.value().shape != x.value().shape) err_shape(fmt_shape(x.value().shape), fmt_shape(r.value().shape));
  check_param(w.value(), H, "weight");
  for (const Var* v : {&x, &r, &w}) require_hip(v->value(), "add_rms_norm");
  Tensor xc = t_contiguous(x.value());
  Tensor rc = t_contiguous(r.value());
  Tensor wc = t_contiguous(w.value());
  const int64_t rows = H ? xc.numel() / H : 0;
  Tensor h = Tensor::empty(xc.shape, Dev::Hip);
  Tensor y = Tensor::empty(xc.shape, Dev::Hip);
  Tensor rstd = Tensor::empty({rows}, Dev::Hip);
  hip_check(oxi_add_rms_norm_fwd(xc.data(), rc.data(), wc.data(), h.data(), y.data(), rstd.data(), rows, H, eps));
  Var hv = Var::op(h, "add", {x, r}, [](const Tensor& g, const std::vector<bool>& need) {
    Grads d(2);
    if (need[0]) d[0] = g;
    if (need[1]) d[1] = g;
    return d;
  });
  auto saved = std::make_shared<NormSaved>();
  saved->x = h;
  saved->w = wc;
  saved->has_w = true;
  saved->rstd = rstd;
  saved->rows = rows;
  saved->H = H;
  saved->mode = (int)mode;
  saved->residual = true;
  saved->wi = 1;
  Var yv = Var::op(y, "rms_norm", {hv, w}, [h, wc, rstd, rows, H, mode](const Tensor& g, const std::vector<bool>& need) {
    Grads d(2);
    if (!need[0] && !need[1]) return d;
    Tensor gc = t_contiguous(g);
    Tensor dx = need[0] ? Tensor::empty(h.shape, Dev::Hip) : Tensor();
    Tensor dw = need[1] ? Tensor::empty({H}, Dev::Hip) : Tensor();
    hip_check(oxi_add_rms_norm_bwd(h.data(), wc.data(), rstd.data(), gc.data(), nullptr, need[0] ? dx.data() : nullptr,
                                   need[1] ? dw.data() : nullptr, nullptr, rows, H, (int)mode));
    if (need[0]) d[0] = dx;
    if (need[1]) d[1] = dw;
    return d;
  });
  if (yv.node->op) yv.node->norm = std::move(saved);
  return {yv, hv};
}

void add_rms_norm_vjp(const NormSaved& s, const Tensor& g, const Tensor& gh, bool need_dw, Tensor* total,
                      Grads& grads) {
  grads.assign(2, std::nullopt);
  const Tensor gc = t_contiguous(g), hc = t_contiguous(gh);
  Tensor dx = Tensor::empty(s.x.shape, Dev::Hip);
  Tensor dw = need_dw ? Tensor::empty({s.H}, Dev::Hip) : Tensor();
  hip_check(oxi_add_rms_norm_bwd(s.x.data(), s.w.data(), s.rstd.data(), gc.data(), hc.data(), dx.data(),
                                 need_dw ? dw.data() : nullptr, nullptr, s.rows, s.H, s.mode));
  *total = dx;
  if (need_dw) grads[1] = dw;
}

Var layer_norm(const Var& x, const std::optional<Var>& w, const std::optional<Var>& b, float eps, NormVjp mode) {
  const int64_t H = last_dim(x.value(), "layer_norm");
  if (w) check_param(w->value(), H, "weight");
  if (b) check_param(b->value(), H, "bias");
  Tensor xc = t_contiguous(x.value());
  Tensor wc = w ? t_contiguous(w->value()) : Tensor();
  Tensor bc = b ? t_contiguous(b->value()) : Tensor();
  const int64_t rows = H ? xc.numel() / H : 0;
  Tensor y = Tensor::empty(xc.shape, Dev::Hip);
  Tensor mean = Tensor::empty({rows}, Dev::Hip);
  Tensor rstd = Tensor::empty({rows}, Dev::Hip);
  hip_check(oxi_layer_norm_fwd(xc.data(), w ? wc.data() : nullptr, b ? bc.data() : nullptr, y.data(), mean.data(),
                               rstd.data(), rows, H, eps));
  std::vector<Var> inputs{x};
  const int wi = w ? (int)inputs.size() : -1;
  if (w) inputs.push_back(*w);
  const int bi = b ? (int)inputs.size() : -1;
  if (b) inputs.push_back(*b);
  const bool has_w = (bool)w;
  auto saved = std::make_shared<NormSaved>();
  saved->ln = true;
  saved->x = xc;
  saved->w = wc;
  saved->b = bc;
  saved->has_w = has_w;
  saved->has_b = (bool)b;
  saved->mean = mean;
  saved->rstd = rstd;
  saved->rows = rows;
  saved->H = H;
  saved->mode = (int)mode;
  saved->wi = wi;
  saved->bi = bi;
  Var v = Var::op(y, "layer_norm", inputs,
                 [xc, wc, mean, rstd, rows, H, mode, wi, bi, has_w](const Tensor& g, const std::vector<bool>& need) {
                   Grads r(need.size());
                   const bool ndx = need[0], ndw = wi >= 0 && need[wi], ndb = bi >= 0 && need[bi];
                   if (!ndx && !ndw && !ndb) return r;
                   Tensor gc = t_contiguous(g);
                   Tensor dx = ndx ? Tensor::empty(xc.shape, Dev::Hip) : Tensor();
                   Tensor dw = ndw ? Tensor::empty({H}, Dev::Hip) : Tensor();
                   Tensor db = ndb ? Tensor::empty({H}, Dev::Hip) : Tensor();
                   hip_check(oxi_layer_norm_bwd(xc.data(), has_w ? wc.data() : nullptr, mean.data(), rstd.data(),
                                                gc.data(), ndx ? dx.data() : nullptr, ndw ? dw.data() : nullptr,
                                                ndb ? db.data() : nullptr, rows, H, (int)mode));
                   if (ndx) r[0] = dx;
                   if (ndw) r[wi] = dw;
                   if (ndb) r[bi] = db;
                   return r;
                 });
  if (v.node->op) v.node->norm = std::move(saved);
  return v;
}

bool norm_vjp_fused(const NormSaved& s, int act, const Tensor& g, const std::vector<bool>& need, Tensor* dy,
                    Grads& grads, int64_t lead, Tensor* lsum) {
  grads.assign(need.size(), std::nullopt);
  const bool ndx = need[0] || lsum, ndw = s.wi >= 0 && need[s.wi], ndb = s.bi >= 0 && need[s.bi];
  Tensor gc = t_contiguous(g.shape == s.x.shape ? g : t_broadcast_to(g, s.x.shape));
  const bool ndy = act >= 0 && dy;  // the activation's input gradient, when the caller keeps it
  Tensor d = ndy ? Tensor::empty(s.x.shape, Dev::Hip) : Tensor();
  Tensor dx = ndx ? Tensor::empty(s.x.shape, Dev::Hip) : Tensor();
  Tensor dw = ndw ? Tensor::empty({s.H}, Dev::Hip) : Tensor();
  Tensor db = ndb ? Tensor::empty({s.H}, Dev::Hip) : Tensor();
  Tensor ls = lsum ? Tensor::empty({s.rows / lead, s.H}, Dev::Hip) : Tensor();
  const float* w = s.has_w ? s.w.data() : nullptr;
  const float* b = s.has_b ? s.b.data() : nullptr;
  float* dp = ndy ? d.data() : nullptr;
  float* dxp = ndx ? dx.data() : nullptr;
  float* dwp = ndw ? dw.data() : nullptr;
  float* dbp = ndb ? db.data() : nullptr;
  int rc;
  if (lsum)
    rc = s.ln ? oxi_layer_norm_bwd_lead_sum(s.x.data(), w, b, s.mean.data(), s.rstd.data(), gc.data(), act, dp, dxp,
                                            dwp, dbp, ls.data(), lead, s.rows, s.H, s.mode)
              : oxi_rms_norm_bwd_lead_sum(s.x.data(), w, s.rstd.data(), gc.data(), act, dp, dxp, dwp, ls.data(),
                                          lead, s.rows, s.H, s.mode);
  else if (act >= 0)
    rc = s.ln ? oxi_layer_norm_act_bwd(s.x.data(), w, b, s.mean.data(), s.rstd.data(), gc.data(), act, dp, dxp, dwp,
                                       dbp, s.rows, s.H, s.mode)
              : oxi_rms_norm_act_bwd(s.x.data(), w, s.rstd.data(), gc.data(), act, dp, dxp, dwp, s.rows, s.H,
                                     s.mode);
  else
    return false;
  if (rc == OXI_NOT_IMPLEMENTED) return false;
  hip_check(rc);
  if (ndy) *dy = d;
  if (lsum) *lsum = ls;
  if (need[0]) grads[0] = dx;
  if (ndw) grads[s.wi] = dw;
  if (ndb) grads[s.bi] = db;
  return true;
}

// ---- fused activations (functional.py:194-204) ----------------------------------------

Var gelu(const Var& x, int approximate) {
  const Tensor& xv = x.value();
  require_hip(xv, "gelu");
  Tensor y = Tensor::empty(xv.shape, Dev::Hip);
  hip_check(oxi_gelu_fwd(xv.data(), xv.strides.data(), y.data(), y.strides.data(), xv.shape.data(), xv.ndim(),
                         approximate));
  Tensor xs = xv;
  Var v = Var::op(y, "gelu", {x}, [xs, approximate](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    Tensor gb = g.shape == xs.shape ? g : t_broadcast_to(g, xs.shape);
    Tensor dx = Tensor::empty(xs.shape, Dev::Hip);
    dx.strides = result_strides(xs.shape, {&xs, &gb});
    hip_check(oxi_gelu_bwd(xs.data(), xs.strides.data(), gb.data(), gb.strides.data(), dx.data(), dx.strides.data(),
                           xs.shape.data(), xs.ndim(), approximate));
    return {dx};
  });
  if (v.node->op) v.node->act = approximate == OXI_GELU_ERF ? OXI_ACT_GELU_ERF : OXI_ACT_GELU_TANH;
  return v;
}

Var silu(const Var& x) {
  const Tensor& xv = x.value();
  require_hip(xv, "silu");
  Tensor y = Tensor::empty(xv.shape, Dev::Hip);
  hip_check(oxi_silu_fwd(xv.data(), xv.strides.data(), y.data(), y.strides.data(), xv.shape.data(), xv.ndim()));
  Tensor xs = xv;
  Var v = Var::op(y, "silu", {x}, [xs](const Tensor& g, const std::vector<bool>& need) -> Grads {
    if (!need[0]) return {std::nullopt};
    Tensor gb = g.shape == xs.shape ? g : t_broadcast_to(g, xs.shape);
    Tensor dx = Tensor::empty(xs.shape, Dev::Hip);
    dx.strides = result_strides(xs.shape, {&xs, &gb});
    hip_check(oxi_silu_bwd(xs.data(), xs.strides.data(), gb.data(), gb.strides.data(), dx.data(), dx.strides.data(),
                           xs.shape.data(), xs.ndim()));
    return {dx};
  });
  if (v.node->op) v.node->act = OXI_ACT_SILU;
  return v;
}

// ---- softmax family (functional.py:211-222) ---------------------------------------------

Var softmax(const Var& x, int64_t dim, bool log) {
  const Tensor& xv = x.value();
  if (xv.ndim() == 0) err_invalid("dim " + std::to_string(dim) + " out of range for 0-D tensor");
  const int d = normalize_dim(dim, xv.ndim());
  if (xv.shape[d] == 0) err_invalid("cannot compute max/min over a zero-length dim");
  Tensor xc = t_contiguous(xv);
  int64_t outer = 1, inner = 1;
  for (int i = 0; i < d; ++i) outer *= xv.shape[i];
  for (int i = d + 1; i < xv.ndim(); ++i) inner *= xv.shape[i];
  const int64_t len = xv.shape[d];
  Tensor y = Tensor::empty(xv.shape, Dev::Hip);
  hip_check(log ? oxi_log_softmax_fwd(xc.data(), y.data(), outer, len, inner)
                : oxi_softmax_fwd(xc.data(), y.data(), outer, len, inner));
  Var v = Var::op(y, log ? "log_softmax" : "softmax", {x},
                  [y, outer, len, inner, log](const Tensor& g, const std::vector<bool>& need) -> Grads {
                    if (!need[0]) return {std::nullopt};
                    Tensor gc = t_contiguous(g.shape == y.shape ? g : t_broadcast_to(g, y.shape));
                    Tensor dx = Tensor::empty(y.shape, Dev::Hip);
                    hip_check(log ? oxi_log_softmax_bwd(y.data(), gc.data(), dx.data(), outer, len, inner)
                                  : oxi_softmax_bwd(y.data(), gc.data(), dx.data(), outer, len, inner));
                    return {dx};
                  });
  // over the last dim a norm VJP can absorb it
  if (v.node->op && inner == 1) v.node->act = log ? OXI_ACT_LOG_SOFTMAX : OXI_ACT_SOFTMAX;
  return v;
}

// ---- cross entropy (functional.py:277-293), targets already resolved ------------------------

Var cross_entropy(const Var& logits, const std::vector<int64_t>& targets) {
  const Tensor& lv = logits.value();
  if (lv.ndim() != 2) err_invalid("cross_entropy expects (batch, classes) logits, got " + fmt_shape(lv.shape));
  const int64_t n = lv.shape[0], c = lv.shape[1];
  if ((int64_t)targets.size() != n)
    err_invalid(std::to_string(targets.size()) + " targets for batch of " + std::to_string(n));
  for (int64_t t : targets)
    if (t < 0 || t >= c)
      err_oob("index " + std::to_string(t) + " is out of bounds for axis 1 with size " + std::to_string(c));
  require_hip(lv, "cross_entropy");
  Tensor lc = t_contiguous(lv);
  auto tg = device_i64(targets);
  const int64_t* tp = static_cast<const int64_t*>(tg->ptr);
  Tensor loss = Tensor::empty({}, Dev::Hip);
  Tensor lse = Tensor::empty({n}, Dev::Hip);
  // With a gradient to come, the forward pass also forms the gradient for an
  // upstream 1 (loss.backward()'s seed) from the logits it holds: the first
  // backward seeded so takes it as is; any other upstream, or a second
  // backward, runs the backward kernel. That gradient is an n x c tensor held
  // until the backward: a loop that scales the loss first, or never calls
  // backward, pays its write and memory for nothing, and turns it off with
  // OXI_CE_ONE_PASS=0 (or set_ce_one_pass(False)).
  std::optional<Tensor> unit;
  if (logits.requires_grad() && is_grad_enabled() && ce_one_pass()) {
    Tensor d = Tensor::empty({n, c}, Dev::Hip);
    const int rc = oxi_cross_entropy_fwd_grad(lc.data(), tp, loss.data(), lse.data(), d.data(), n, c);
    if (rc == OXI_OK) unit = d;
    else if (rc != OXI_NOT_IMPLEMENTED) hip_check(rc);
  }
  if (!unit) hip_check(oxi_cross_entropy_fwd(lc.data(), tp, loss.data(), lse.data(), n, c));
  auto fresh = std::make_shared<std::atomic<bool>>(unit.has_value());
  return Var::op(loss, "cross_entropy", {logits},
                 [lc, tg, lse, n, c, unit, fresh](const Tensor& g, const std::vector<bool>& need) -> Grads {
                   if (!need[0]) return {std::nullopt};
                   if (is_implicit_seed(g) && fresh->exchange(false)) return {*unit};
                   Tensor gs = t_contiguous(g);
                   Tensor d = Tensor::empty({n, c}, Dev::Hip);
                   hip_check(oxi_cross_entropy_bwd(lc.data(), static_cast<const int64_t*>(tg->ptr), lse.data(),
                                                   gs.data(), d.data(), n, c));
                   return {d};
                 });
}

// ---- rotary positions ---------------------------------------------------------------

Var rotary(const Var& x, const RotaryFrequencies& f, const std::optional<std::vector<int64_t>>& positions,
           int64_t offset, int layout) {
  const Tensor& xv = x.value();
  require_hip(xv, "rotary_embedding");
  if (xv.ndim() != 3 && xv.ndim() != 4)
    err_invalid("rotary_embedding expects (batch, tokens, heads, dim) or (tokens, heads, dim), got " +
                fmt_shape(xv.shape));
  if (2 * f.pairs > xv.shape.back())
    err_invalid("rotary_embedding: " + std::to_string(f.pairs) + " pairs do not fit in heads of " +
                std::to_string(xv.shape.back()));
  const bool batched = xv.ndim() == 4;
  const int64_t B = batched ? xv.shape[0] : 1, T = xv.shape[batched ? 1 : 0];
  std::shared_ptr<Storage> pos;
  Shape ps{0, 0};
  if (positions) {
    const int64_t n = (int64_t)positions->size();
    if (n != T && n != B * T)
      err_invalid("rotary_embedding: " + std::to_string(n) + " positions for " + std::to_string(B) + " x " +
                  std::to_string(T) + " tokens");
    pos = device_i64(*positions);
    ps = n == B * T ? Shape{T, 1} : Shape{0, 1};
  }
  auto freq = f.values;
  const int64_t rot = 2 * f.pairs;
  const float scale = f.scale;
  auto turn = [pos, ps, freq, rot, scale, layout, offset, batched](const Tensor& in, bool inverse) {
    Tensor out = Tensor::empty(in.shape, Dev::Hip);
    out.strides = result_strides(in.shape, {&in});
    auto four = [batched](const Shape& v, int64_t first) {
      Shape s = v;
      if (!batched) s.insert(s.begin(), first);
      return s;
    };
    const Shape shape = four(in.shape, 1), xs = four(in.strides, 0), ys = four(out.strides, 0);
    hip_check(oxi_rotary(in.data(), xs.data(), out.data(), ys.data(), shape.data(),
                         pos ? static_cast<const int64_t*>(pos->ptr) : nullptr, ps.data(), offset,
                         rot ? static_cast<const double*>(freq->ptr) : nullptr, rot, layout, inverse ? 1 : 0, scale));
    return out;
  };
  const Shape xshape = xv.shape;
  return Var::op(turn(xv, false), "rotary_embedding", {x},
                 [turn, xshape](const Tensor& g, const std::vector<bool>& need) -> Grads {
                   if (!need[0]) return {std::nullopt};
                   return {turn(g.shape == xshape ? g : t_broadcast_to(g, xshape), true)};
                 });
}

// ---- distillation ---------------------------------------------------------------------

Var distillation_loss(const Var& logits, const std::vector<int64_t>& ids, const Tensor& top,
                      const std::optional<Tensor>& top_lse, float temperature) {
  const Tensor& lv = logits.value();
  if (lv.ndim() != 2) err_invalid("distillation_loss expects (batch, classes) logits, got " + fmt_shape(lv.shape));
  const int64_t n = lv.shape[0], c = lv.shape[1];
  if (top.ndim() != 2 || top.shape[0] != n) err_shape(fmt_shape(lv.shape), fmt_shape(top.shape));
  const int64_t k = top.shape[1];
  if ((int64_t)ids.size() != n * k)
    err_invalid(std::to_string(ids.size()) + " teacher ids for logits of shape " + fmt_shape(top.shape));
  if (top_lse && top_lse->shape != Shape{n}) err_shape(fmt_shape({n}), fmt_shape(top_lse->shape));
  for (int64_t i : ids)
    if (i >= c)
      err_oob("index " + std::to_string(i) + " is out of bounds for axis 1 with size " + std::to_string(c));
  require_hip(lv, "distillation_loss");
  require_hip(top, "distillation_loss");
  if (top_lse) require_hip(*top_lse, "distillation_loss");
  Tensor lc = t_contiguous(lv), tc = t_contiguous(top);
  std::optional<Tensor> ec;
  if (top_lse) ec = t_contiguous(*top_lse);
  auto id = device_i64(ids);
  Tensor loss = Tensor::empty({}, Dev::Hip), row = Tensor::empty({n}, Dev::Hip), lse = Tensor::empty({n}, Dev::Hip),
         rest = Tensor::empty({n}, Dev::Hip), count = Tensor::empty({}, Dev::Hip);
  // With a gradient to come, the forward pass also forms the gradient for
  // loss.backward()'s seed, as cross_entropy does (and the same switch turns off).
  std::optional<Tensor> unit;
  if (logits.requires_grad() && is_grad_enabled() && ce_one_pass()) unit = Tensor::empty({n, c}, Dev::Hip);
  const int64_t* ip = static_cast<const int64_t*>(id->ptr);
  hip_check(oxi_distill_fwd_counted(lc.data(), ip, tc.data(), ec ? ec->data() : nullptr, loss.data(), row.data(),
                                    lse.data(), rest.data(), unit ? unit->data() : nullptr, count.data(), n, c, k,
                                    temperature));
  auto fresh = std::make_shared<std::atomic<bool>>(unit.has_value());
  return Var::op(loss, "distillation_loss", {logits},
                 [lc, tc, ec, id, lse, rest, count, n, c, k, temperature, unit, fresh](
                     const Tensor& g, const std::vector<bool>& need) -> Grads {
                   if (!need[0]) return {std::nullopt};
                   if (is_implicit_seed(g) && fresh->exchange(false)) return {*unit};
                   Tensor gs = t_contiguous(g);
                   Tensor d = Tensor::empty({n, c}, Dev::Hip);
                   hip_check(oxi_distill_bwd_counted(lc.data(), static_cast<const int64_t*>(id->ptr), tc.data(),
                                                     ec ? ec->data() : nullptr, lse.data(), rest.data(), gs.data(),
                                                     d.data(), count.data(), n, c, k, temperature));
                   return {d};
                 });
}

// ---- post-training losses ------------------------------------------------------------

namespace {

// (batch, classes) logits and one id a row; ids below 0 are padding.
void check_tokens(const Tensor& lv, const std::vector<int64_t>& ids, const char* what) {
  if (lv.ndim() != 2) err_invalid(std::string(what) + " expects (batch, classes) logits, got " + fmt_shape(lv.shape));
  if ((int64_t)ids.size() != lv.shape[0])
    err_invalid(std::to_string(ids.size()) + " tokens for batch of " + std::to_string(lv.shape[0]));
  for (int64_t i : ids)
    if (i >= lv.shape[1])
      err_oob("index " + std::to_string(i) + " is out of bounds for axis 1 with size " + std::to_string(lv.shape[1]));
  require_hip(lv, what);
}

// A row's number each, contiguous on the device; unset stays unset.
std::optional<Tensor> per_row(const std::optional<Tensor>& t, int64_t n, const char* what) {
  if (!t) return std::nullopt;
  if (t->shape != Shape{n}) err_shape(fmt_shape({n}), fmt_shape(t->shape));
  require_hip(*t, what);
  return t_contiguous(*t);
}

float* ptr(const std::optional<Tensor>& t) { return t ? t->data() : nullptr; }

// The node of a loss whose gradient goes by each row's logp and, with `gh`, its entropy:
// `unit`, what the forward wrote for backward()'s seed, or a pass from coef and saved.
Var token_loss(const Tensor& loss, const char* op, const Var& logits, const Tensor& lc,
               const std::shared_ptr<Storage>& id, const Tensor& saved, const Tensor& coef, bool gh, float temperature,
               const std::optional<Tensor>& unit) {
  const int64_t n = lc.shape[0], c = lc.shape[1];
  auto fresh = std::make_shared<std::atomic<bool>>(unit.has_value());
  return Var::op(loss, op, {logits},
                 [lc, id, saved, coef, gh, temperature, n, c, unit, fresh](const Tensor& g,
                                                                          const std::vector<bool>& need) -> Grads {
                   if (!need[0]) return {std::nullopt};
                   if (is_implicit_seed(g) && fresh->exchange(false)) return {*unit};
                   Tensor gs = t_contiguous(g);
                   Tensor d = Tensor::empty({n, c}, Dev::Hip);
                   hip_check(oxi_token_logp_bwd(lc.data(), static_cast<const int64_t*>(id->ptr), saved.data(),
                                                coef.data(), gh ? coef.data() + n : nullptr, gs.data(), d.data(), n, c,
                                                temperature));
                   return {d};
                 });
}

bool wants_gradient(const Var& logits) { return logits.requires_grad() && is_grad_enabled(); }

}  // namespace

Var token_log_probs(const Var& logits, const std::vector<int64_t>& ids, float temperature, bool entropy) {
  const Tensor& lv = logits.value();
  check_tokens(lv, ids, "token_log_probs");
  const int64_t n = lv.shape[0], c = lv.shape[1];
  Tensor lc = t_contiguous(lv);
  auto id = device_i64(ids);
  Tensor out = Tensor::empty(entropy ? Shape{2, n} : Shape{n}, Dev::Hip);
  std::optional<Tensor> saved;
  if (wants_gradient(logits)) saved = Tensor::empty({n, 4}, Dev::Hip);
  hip_check(oxi_token_logp_fwd(lc.data(), static_cast<const int64_t*>(id->ptr), out.data(),
                               entropy ? out.data() + n : nullptr, saved ? saved->data() : nullptr, nullptr, n, c,
                               temperature));
  return Var::op(out, "token_log_probs", {logits},
                 [lc, id, saved, entropy, n, c, temperature](const Tensor& g, const std::vector<bool>& need) -> Grads {
                   if (!need[0]) return {std::nullopt};
                   Tensor gs = t_contiguous(g);
                   Tensor d = Tensor::empty({n, c}, Dev::Hip);
                   hip_check(oxi_token_logp_bwd(lc.data(), static_cast<const int64_t*>(id->ptr), saved->data(),
                                                gs.data(), entropy ? gs.data() + n : nullptr, nullptr, d.data(), n, c,
                                                temperature));
                   return {d};
                 });
}

std::pair<Var, Tensor> policy_loss(const Var& logits, const std::vector<int64_t>& ids, const Tensor& advantages,
                                   const std::optional<Tensor>& old_logp, const std::optional<Tensor>& ref_logp,
                                   const std::optional<Tensor>& weights, const PolicyOptions& o) {
  const Tensor& lv = logits.value();
  check_tokens(lv, ids, "policy_loss");
  const int64_t n = lv.shape[0], c = lv.shape[1];
  const auto adv = per_row(advantages, n, "policy_loss"), old = per_row(old_logp, n, "policy_loss"),
             ref = per_row(ref_logp, n, "policy_loss"), w = per_row(weights, n, "policy_loss");
  Tensor lc = t_contiguous(lv);
  auto id = device_i64(ids);
  Tensor out = Tensor::empty({4}, Dev::Hip), rows = Tensor::empty({4, n}, Dev::Hip), coef = Tensor::empty({2, n}, Dev::Hip),
         saved = Tensor::empty({n, 4}, Dev::Hip);
  // With a gradient to come, the forward pass also forms the gradient for
  // loss.backward()'s seed, as cross_entropy does (and the same switch turns off).
  std::optional<Tensor> unit;
  if (wants_gradient(logits) && ce_one_pass()) unit = Tensor::empty({n, c}, Dev::Hip);
  hip_check(oxi_policy_loss_fwd(lc.data(), static_cast<const int64_t*>(id->ptr), ptr(adv), ptr(old), ptr(ref), ptr(w),
                                out.data(), rows.data(), nullptr, coef.data(), saved.data(), ptr(unit), nullptr, n, c,
                                o.temperature, o.clip_low, o.clip_high, o.clip_max, o.kl, o.entropy, o.divisor));
  const Tensor loss = t_select(out, 0, 0);
  return {token_loss(loss, "policy_loss", logits, lc, id, saved, coef, o.entropy != 0.0f, o.temperature, unit),
          t_narrow(out, 0, 1, 4, 1)};
}

std::pair<Var, std::pair<Tensor, Tensor>> preference_loss(const Var& logits, const std::vector<int64_t>& ids,
                                                          const std::vector<int64_t>& lengths,
                                                          const std::optional<Tensor>& ref_logp,
                                                          const PreferenceOptions& o) {
  const Tensor& lv = logits.value();
  check_tokens(lv, ids, "preference_loss");
  const int64_t n = lv.shape[0], c = lv.shape[1], pairs = (int64_t)lengths.size() / 2;
  if (lengths.size() % 2) err_invalid("preference_loss: an odd number of sequences: " + std::to_string(lengths.size()));
  std::vector<int64_t> starts{0};
  for (int64_t l : lengths) {
    if (l < 0 || l > n - starts.back())
      err_invalid("preference_loss: a sequence of " + std::to_string(l) + " rows after " +
                  std::to_string(starts.back()) + " of " + std::to_string(n));
    starts.push_back(starts.back() + l);
  }
  const auto ref = per_row(ref_logp, n, "preference_loss");
  Tensor lc = t_contiguous(lv);
  auto id = device_i64(ids), at = device_i64(starts);
  Tensor loss = Tensor::empty({}, Dev::Hip), pair = Tensor::empty({pairs}, Dev::Hip),
         seq = Tensor::empty({pairs, 2}, Dev::Hip), coef = Tensor::empty({n}, Dev::Hip),
         saved = Tensor::empty({n, 4}, Dev::Hip);
  std::optional<Tensor> unit;
  if (wants_gradient(logits) && ce_one_pass()) unit = Tensor::empty({n, c}, Dev::Hip);
  hip_check(oxi_preference_loss_fwd(lc.data(), static_cast<const int64_t*>(id->ptr),
                                    static_cast<const int64_t*>(at->ptr), ptr(ref), loss.data(), pair.data(), seq.data(),
                                    coef.data(), saved.data(), ptr(unit), nullptr, n, c, pairs, o.kind, o.average ? 1 : 0,
                                    o.beta, o.margin, o.smoothing));
  return {token_loss(loss, "preference_loss", logits, lc, id, saved, coef, false, 1.0f, unit), {pair, seq}};
}

}  // namespace aops

RotaryFrequencies::RotaryFrequencies(const std::vector<double>& inv_freq, float s)
    : pairs((int64_t)inv_freq.size()), scale(s) {
  if (inv_freq.empty()) return;
  values = std::make_shared<Storage>(Dev::Hip, sizeof(double) * inv_freq.size());
  hip_check(oxi_hip_upload(values->ptr, inv_freq.data(), sizeof(double) * inv_freq.size()));
}

// ---- serving ------------------------------------------------------------------------------

E4m3Rows t_add_rms_norm_e4m3(const Tensor& x, const std::optional<Tensor>& r, const Tensor& w, float eps,
                             int64_t group, Tensor* h) {
  if (x.ndim() == 0) err_invalid("add_rms_norm_e4m3 needs at least one dim");
  const int64_t H = x.shape.back();
  if (r && r->shape != x.shape) err_shape(fmt_shape(x.shape), fmt_shape(r->shape));
  if (w.ndim() != 1 || w.shape[0] != H) err_shape(fmt_shape(w.shape), fmt_shape({H}));
  if (group < 1) err_invalid("add_rms_norm_e4m3: groups of " + std::to_string(group) + " columns");
  require_hip(x, "add_rms_norm_e4m3");
  if (r) require_hip(*r, "add_rms_norm_e4m3");
  require_hip(w, "add_rms_norm_e4m3");
  const Tensor xc = t_contiguous(x), wc = t_contiguous(w);
  Tensor rc;
  if (r) {
    rc = t_contiguous(*r);
    *h = Tensor::empty(x.shape, Dev::Hip);
  }
  E4m3Rows q;
  q.shape = x.shape;
  q.group = group;
  const int64_t rows = H ? xc.numel() / H : 0;
  Shape ss = x.shape;
  ss.back() = (H + group - 1) / group;
  q.scale = Tensor::empty(ss, Dev::Hip);
  q.codes = std::make_shared<Storage>(Dev::Hip, (size_t)xc.numel());
  hip_check(oxi_add_rms_norm_e4m3_fwd(xc.data(), r ? rc.data() : nullptr, wc.data(), r ? h->data() : nullptr,
                                      static_cast<uint8_t*>(q.codes->ptr), q.scale.data(), rows, H, group, eps));
  return q;
}

Tensor t_dequantize(const E4m3Rows& q) {
  Tensor y = Tensor::empty(q.shape, Dev::Hip);
  const int64_t H = q.shape.back();
  hip_check(oxi_e4m3_dequantize(static_cast<const uint8_t*>(q.codes->ptr), q.scale.data(), y.data(),
                                H ? y.numel() / H : 0, H, q.group));
  return y;
}

std::pair<std::vector<int64_t>, std::vector<int64_t>> t_verify_drafts(
    const Tensor& target, const std::optional<Tensor>& draft, const std::vector<int64_t>& tokens,
    const std::optional<std::vector<int64_t>>& lengths, const Tensor& uniforms) {
  if (target.ndim() != 3)
    err_invalid("verify_drafts expects (batch, drafts + 1, classes) probabilities, got " + fmt_shape(target.shape));
  const int64_t b = target.shape[0], rows = target.shape[1], v = target.shape[2];
  if (rows < 1) err_invalid("verify_drafts: no row of target probabilities");
  const int64_t k = rows - 1;
  if (draft && draft->shape != Shape{b, k, v}) err_shape(fmt_shape(draft->shape), fmt_shape({b, k, v}));
  if (uniforms.shape != Shape{b, rows}) err_shape(fmt_shape(uniforms.shape), fmt_shape({b, rows}));
  if ((int64_t)tokens.size() != b * k)
    err_invalid(std::to_string(tokens.size()) + " drafted tokens for " + std::to_string(b) + " x " +
                std::to_string(k) + " drafts");
  if (lengths && (int64_t)lengths->size() != b)
    err_invalid(std::to_string(lengths->size()) + " lengths for batch of " + std::to_string(b));
  if (lengths)
    for (int64_t n : *lengths)
      if (n < 0 || n > k)
        err_invalid("verify_drafts: a length of " + std::to_string(n) + " of " + std::to_string(k) + " drafts");
  for (int64_t s = 0; s < b; ++s)
    for (int64_t i = 0; i < (lengths ? (*lengths)[(size_t)s] : k); ++i) {
      const int64_t x = tokens[(size_t)(s * k + i)];
      if (x < 0 || x >= v)
        err_oob("index " + std::to_string(x) + " is out of bounds for axis 2 with size " + std::to_string(v));
    }
  require_hip(target, "verify_drafts");
  if (draft) require_hip(*draft, "verify_drafts");
  require_hip(uniforms, "verify_drafts");
  const Tensor tc = t_contiguous(target), uc = t_contiguous(uniforms);
  Tensor dc;
  if (draft) dc = t_contiguous(*draft);
  std::vector<int64_t> accepted((size_t)b), out((size_t)(b * rows));
  if (b == 0) return {accepted, out};
  auto td = device_i64(tokens);
  std::shared_ptr<Storage> ld;
  if (lengths) ld = device_i64(*lengths);
  // one buffer, and one copy to the host
  Storage res(Dev::Hip, sizeof(int64_t) * (size_t)(b + b * rows));
  int64_t* rp = static_cast<int64_t*>(res.ptr);
  hip_check(oxi_verify_drafts(tc.data(), draft ? dc.data() : nullptr, static_cast<const int64_t*>(td->ptr),
                              ld ? static_cast<const int64_t*>(ld->ptr) : nullptr, uc.data(), rp, rp + b, nullptr, b, k, v));
  std::vector<int64_t> all((size_t)(b + b * rows));
  hip_check(oxi_hip_memcpy_d2h(all.data(), res.ptr, sizeof(int64_t) * all.size()));
  std::copy(all.begin(), all.begin() + b, accepted.begin());
  std::copy(all.begin() + b, all.end(), out.begin());
  return {accepted, out};
}

}  // namespace oxt
