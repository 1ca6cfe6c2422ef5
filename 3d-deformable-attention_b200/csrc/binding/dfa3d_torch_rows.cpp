// Native host path of the row operators: dropout without a stored mask, LayerNorm(residual + dropout(x)), group norm over the
// levels of a feature pyramid.  Same contract as dfa3d_torch.cpp: NotImplemented means that the Python code has to take the call.
#include <ATen/cuda/EmptyTensor.h>

#include "dfa3d_torch.h"

using namespace dfa3d_torch;

namespace {

// a gradient as the kernels take it: of the forward's type, contiguous
Tensor like_forward(const Tensor &g, at::ScalarType type) {
  if (g.scalar_type() == type) return g.contiguous();
  if (type == at::kFloat) return f32(g);
  return g.to(type).contiguous();
}

bool stored_tensor(PyObject *o, Tensor &t) { return plain_tensor(o, t) && storage_type(t.scalar_type()); }

// Memory for a result, on a's device: what at::empty ends in, without the way through the dispatcher (a call has up to six of them).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor &a) {
  return Tensor(at::detail::empty_cuda(sizes, type, a.device(), std::nullopt));
}
Tensor fresh(const Tensor &a) { return fresh(a.sizes(), a.scalar_type(), a); }

bool same_kind(const Tensor &a, const Tensor &b) {
  return a.scalar_type() == b.scalar_type() && a.sizes() == b.sizes() && a.device() == b.device();
}

// ------------------------------------------------------------------------------------------------
// dropout
// ------------------------------------------------------------------------------------------------
Tensor dropout_forward(const Tensor &x, const Tensor &res, const Tensor &seed, const Rule &r, bool relu) {
  Tensor y = fresh(x);
  check(lib.dfa3d_dropout_forward(vp(x), vp(res), dtype_code(x), x.numel(), relu ? DFA3D_ROW_RELU : DFA3D_ROW_NONE, r.p,
                                  seed_of(seed), (int32_t)r.site, vpm(y), stream_of(x)),
        "dfa3d_dropout_forward");
  return y;
}

struct DropoutFn : torch::autograd::Function<DropoutFn> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &res, const std::optional<Tensor> &seed,
                        const c10::intrusive_ptr<Rule> &r, bool relu) {
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor s = seed ? *seed : Tensor();
    Tensor y = dropout_forward(x, res ? *res : Tensor(), s, *r, relu);
    r->residual = res.has_value();
    r->by_result = relu && !res;
    r->type = x.scalar_type();
    keep(ctx, r, {s, relu ? (r->by_result ? y : x) : Tensor()});
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list v;
    const auto r = kept<Rule>(ctx, v);
    Tensor gx;
    if (ctx->needs_input_grad(0)) {
      const Tensor g = like_forward(grads[0], r->type);
      c10::cuda::CUDAGuard guard(g.device());
      gx = fresh(g);
      check(lib.dfa3d_dropout_backward(vp(g), vp(v[1]), r->by_result, dtype_code(g), g.numel(), r->p, seed_of(v[0]),
                                       (int32_t)r->site, vpm(gx), stream_of(g)),
            "dfa3d_dropout_backward");
    }
    Tensor gr = r->residual && ctx->needs_input_grad(1) ? grads[0] : Tensor();
    return once({gx, gr, Tensor(), Tensor(), Tensor()}, grads);
  }
};

PyObject *run_dropout(PyObject *const *a, Py_ssize_t n) {
  // x, residual or None, seed, p, site, activation
  if (n != 6 || !plain_mode()) return not_plain();
  Tensor x, res, seed;
  auto r = c10::make_intrusive<Rule>();
  const bool with = a[1] != Py_None, relu = a[5] != Py_None;
  if (!stored_tensor(a[0], x) || (with && (!stored_tensor(a[1], res) || !same_kind(x, res))) ||
      (relu && (!PyUnicode_CheckExact(a[5]) || PyUnicode_CompareWithASCIIString(a[5], "relu") != 0)) ||
      !rule_arguments(a[2], a[3], a[4], x, seed, *r))
    return not_plain();
  Tensor y;
  {
    pybind11::gil_scoped_release nogil;
    if (wants_grad(x) || (with && wants_grad(res))) {
      y = DropoutFn::apply(x, given(res), given(seed), r, relu);
    } else {
      c10::cuda::CUDAGuard guard(x.device());
      y = dropout_forward(x, res, seed, *r, relu);
    }
  }
  return THPVariable_Wrap(y);
}

// ------------------------------------------------------------------------------------------------
// LayerNorm(residual + dropout(x))
// ------------------------------------------------------------------------------------------------
Tensor drop_norm_forward(const Tensor &x, const Tensor &res, const Tensor &w, const Tensor &b, const Tensor &seed, const Rule &r,
                         double eps, const Tensor &stats) {
  const int64_t E = x.size(-1), rows = x.numel() / E;
  Tensor y = fresh(x);
  float *mean = stats.defined() ? fpm(stats) : nullptr;
  check(lib.dfa3d_dropout_add_layer_norm_forward(vp(x), vp(res), fp(w), fp(b), dtype_code(x), rows, (int32_t)E, r.p, seed_of(seed),
                                                 (int32_t)r.site, (float)eps, vpm(y), mean, mean ? mean + rows : nullptr,
                                                 stream_of(x)),
        "dfa3d_dropout_add_layer_norm_forward");
  return y;
}

struct DropNormFn : torch::autograd::Function<DropNormFn> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &res, const Tensor &w, const Tensor &b,
                        const std::optional<Tensor> &seed, const c10::intrusive_ptr<Rule> &r, double eps) {
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor s = seed ? *seed : Tensor();
    Tensor stats = fresh({2, x.numel() / x.size(-1)}, at::kFloat, x);
    Tensor y = drop_norm_forward(x, res, w, b, s, *r, eps, stats);
    keep(ctx, r, {x, res, w, stats, s});
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list v;
    const auto r = kept<Rule>(ctx, v);
    const Tensor &x = v[0], &res = v[1], &w = v[2], &stats = v[3], &seed = v[4];
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t E = w.numel(), rows = x.numel() / E;       // counts that a saved-tensor hook cannot change, as it can a shape
    const Tensor g = like_forward(grads[0], x.scalar_type());
    const bool params = ctx->needs_input_grad(2) || ctx->needs_input_grad(3);
    Tensor gx, gr, gw, gb, work;
    if (ctx->needs_input_grad(0)) gx = fresh(g);
    if (ctx->needs_input_grad(1)) gr = fresh(g);
    if (params) {
      gw = fresh({E}, at::kFloat, x);
      gb = fresh({E}, at::kFloat, x);
      work = fresh({lib.dfa3d_dropout_add_layer_norm_workspace(rows, (int32_t)E)}, at::kByte, x);
    }
    check(lib.dfa3d_dropout_add_layer_norm_backward(vp(g), vp(x), vp(res), fp(w), fp(stats), fp(stats) + rows, dtype_code(x), rows,
                                                    (int32_t)E, r->p, seed_of(seed), (int32_t)r->site, vpm(gx), vpm(gr),
                                                    (float *)vpm(gw), (float *)vpm(gb), vpm(work), params ? work.numel() : 0,
                                                    stream_of(x)),
          "dfa3d_dropout_add_layer_norm_backward");
    if (params && !ctx->needs_input_grad(2)) gw = Tensor();
    if (params && !ctx->needs_input_grad(3)) gb = Tensor();
    return once({gx, gr, gw, gb, Tensor(), Tensor(), Tensor()}, grads);
  }
};

PyObject *run_drop_norm(PyObject *const *a, Py_ssize_t n) {
  // x, residual, weight, bias, seed, p, site, eps
  double eps;
  if (n != 8 || !plain_mode() || !number(a[7], eps) || !(eps >= 0)) return not_plain();
  Tensor x, res, w, b, seed;
  auto r = c10::make_intrusive<Rule>();
  if (!stored_tensor(a[0], x) || x.dim() < 1 || x.numel() == 0 || !stored_tensor(a[1], res) || !same_kind(x, res) ||
      !float_tensor(a[2], w, 1) || !float_tensor(a[3], b, 1) || !rule_arguments(a[4], a[5], a[6], x, seed, *r))
    return not_plain();
  const int64_t E = x.size(-1);
  if (w.numel() != E || b.numel() != E || E > 1024 || !one_device(x, w, b)) return not_plain();
  Tensor y;
  {
    pybind11::gil_scoped_release nogil;
    if (wants_grad(x, res, w, b)) {
      y = DropNormFn::apply(x, res, w, b, given(seed), r, eps);
    } else {
      c10::cuda::CUDAGuard guard(x.device());
      y = drop_norm_forward(x, res, w, b, seed, *r, eps, Tensor());
    }
  }
  return THPVariable_Wrap(y);
}

// ------------------------------------------------------------------------------------------------
// group norm
// ------------------------------------------------------------------------------------------------
struct Levels : Kept {
  int32_t B = 0, N = 0, C = 0, G = 0, L = 1, stride = 0, rows = 1, act = 0;
  float eps = 0;
};

Tensor level_workspace(const Levels &s, const Tensor &like, bool backward) {
  const int64_t bytes = lib.dfa3d_group_norm_workspace(s.B, s.N, s.C, s.G, s.L, backward);
  TORCH_CHECK(bytes >= 0, "dfa3d_group_norm_workspace failed: ", lib.dfa3d_last_error());
  return bytes == 0 ? Tensor() : fresh({bytes}, at::kByte, like);
}

Tensor group_norm_forward(const Levels &s, const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &shapes,
                          const Tensor &lsi, const Tensor &stats) {
  Tensor y = fresh(x), work = level_workspace(s, x, false);
  float *mean = stats.defined() ? fpm(stats) : nullptr;
  check(lib.dfa3d_group_norm_forward(vp(x), dtype_code(x), s.B, s.N, s.C, s.G, (const int64_t *)vp(shapes), s.stride,
                                     (const int64_t *)vp(lsi), s.L, fp(w), fp(b), s.rows, s.eps, s.act, vpm(y), mean,
                                     mean ? mean + (int64_t)s.B * s.L * s.G : nullptr, vpm(work), work.defined() ? work.numel() : 0,
                                     stream_of(x)),
        "dfa3d_group_norm_forward");
  return y;
}

struct GroupNormFn : torch::autograd::Function<GroupNormFn> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const Tensor &b, const std::optional<Tensor> &shapes,
                        const std::optional<Tensor> &lsi, const c10::intrusive_ptr<Levels> &s) {
    c10::cuda::CUDAGuard guard(x.device());
    Tensor stats = fresh({2, s->B, s->L, s->G}, at::kFloat, x), sh = shapes ? *shapes : Tensor(), st = lsi ? *lsi : Tensor();
    Tensor y = group_norm_forward(*s, x, w, b, sh, st, stats);
    keep(ctx, s, {x, w, b, sh, st, stats});
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list v;
    const auto s = kept<Levels>(ctx, v);
    const Tensor &x = v[0], &w = v[1], &b = v[2], &shapes = v[3], &lsi = v[4], &stats = v[5];
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor g = like_forward(grads[0], x.scalar_type());
    const bool params = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    Tensor gx, gw, gb, work = level_workspace(*s, x, true);
    if (ctx->needs_input_grad(0)) gx = fresh(g);
    if (params) {
      gw = fresh(w);
      gb = fresh(w);
    }
    check(lib.dfa3d_group_norm_backward(vp(g), vp(x), dtype_code(x), s->B, s->N, s->C, s->G, (const int64_t *)vp(shapes), s->stride,
                                        (const int64_t *)vp(lsi), s->L, fp(w), fp(b), s->rows, s->act, fp(stats),
                                        fp(stats) + (int64_t)s->B * s->L * s->G, vpm(gx), (float *)vpm(gw), (float *)vpm(gb),
                                        vpm(work), work.numel(), stream_of(x)),
          "dfa3d_group_norm_backward");
    if (params && !ctx->needs_input_grad(1)) gw = Tensor();
    if (params && !ctx->needs_input_grad(2)) gb = Tensor();
    return once({gx, gw, gb, Tensor(), Tensor(), Tensor()}, grads);
  }
};

PyObject *run_group_norm(PyObject *const *a, Py_ssize_t n) {
  // x (B, ..., C), weight, bias, spatial_shapes or None, level_start_index or None, num_groups, eps, activation
  int64_t G;
  double eps;
  if (n != 8 || !plain_mode() || !integer(a[5], G) || !number(a[6], eps) || !(eps >= 0)) return not_plain();
  Tensor x, w, b, shapes, lsi;
  const bool table = a[3] != Py_None;
  if (table != (a[4] != Py_None) || !stored_tensor(a[0], x) || x.dim() < 2 || x.numel() == 0 || !float_tensor(a[1], w, -1) ||
      !float_tensor(a[2], b, -1) || (table && (!long_tensor(a[3], shapes, 2) || !long_tensor(a[4], lsi, 1))))
    return not_plain();
  auto s = c10::make_intrusive<Levels>();
  const int64_t B = x.size(0), C = x.size(-1), N = x.numel() / B / C, L = table ? shapes.size(0) : 1;
  if (B * std::max(std::min<int64_t>(N, 2052), L * C) >= (int64_t(1) << 31) || N >= (1 << 30) || C > 1024 || G <= 0 || C % G != 0 || L < 1 || L > DFA3D_MAX_LEVELS ||
      w.sizes() != b.sizes() || !one_device(x, w, b))
    return not_plain();
  if (table && (!one_device(x, shapes, lsi) || (shapes.size(1) != 2 && shapes.size(1) != 3) || lsi.numel() != L)) return not_plain();
  if (w.dim() == 1 ? w.size(0) != C : w.dim() != 2 || w.size(0) != L || w.size(1) != C) return not_plain();
  if (a[7] != Py_None) {
    if (!PyUnicode_CheckExact(a[7])) return not_plain();
    if (PyUnicode_CompareWithASCIIString(a[7], "relu") == 0) s->act = DFA3D_ROW_RELU;
    else if (PyUnicode_CompareWithASCIIString(a[7], "silu") == 0) s->act = DFA3D_ROW_SILU;
    else return not_plain();
  }
  s->B = (int32_t)B; s->N = (int32_t)N; s->C = (int32_t)C; s->G = (int32_t)G; s->L = (int32_t)L;
  s->stride = table ? (int32_t)shapes.size(1) : 0;
  s->rows = w.dim() == 1 ? 1 : (int32_t)L;
  s->eps = (float)eps;
  Tensor y;
  {
    pybind11::gil_scoped_release nogil;
    if (wants_grad(x, w, b)) {
      y = GroupNormFn::apply(x, w, b, given(shapes), given(lsi), s);
    } else {
      c10::cuda::CUDAGuard guard(x.device());
      y = group_norm_forward(*s, x, w, b, shapes, lsi, Tensor());
    }
  }
  return THPVariable_Wrap(y);
}

#define FAST(name, expr)                                                             \
  PyObject *py_##name(PyObject *, PyObject *const *a, Py_ssize_t n) {                 \
    HANDLE_TH_ERRORS                                                                  \
    return expr;                                                                      \
    END_HANDLE_TH_ERRORS                                                              \
  }
FAST(dropout, run_dropout(a, n))
FAST(dropout_add_layer_norm, run_drop_norm(a, n))
FAST(group_norm, run_group_norm(a, n))
#undef FAST

}  // namespace

namespace dfa3d_torch {
#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef row_methods[] = {
    FAST(dropout), FAST(dropout_add_layer_norm), FAST(group_norm), {nullptr, nullptr, 0, nullptr},
};
#undef FAST
}  // namespace dfa3d_torch
