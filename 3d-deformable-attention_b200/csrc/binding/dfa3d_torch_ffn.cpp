// Native host path of the feed-forward block in 16 bits: products with bias, activation and residual, the gated block, inputs kept in
// 8 bits.  Same contract as dfa3d_torch.cpp: NotImplemented means that the Python code has to take the call.
#include <ATen/cuda/EmptyTensor.h>
#include <torch/csrc/Dtype.h>

#include "dfa3d_torch.h"

using namespace dfa3d_torch;

namespace {

Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor &a) {
  return Tensor(at::detail::empty_cuda(sizes, type, a.device(), std::nullopt));
}

int64_t pitch_of(int64_t cols) { return (cols + 7) / 8 * 8; }

// A matrix as the products read it.
struct Rows {
  Tensor t;
  int64_t pitch = 0;
  const void *data() const { return vp(t); }
};

// What is not a 16-bit matrix whose rows begin on a 16-byte boundary is copied, all of it with one launch.
struct Operands {
  explicit Operands(at::ScalarType t) : type(t) {}
  Rows add(const Tensor &m, int64_t rows, int64_t cols) {
    if (m.scalar_type() == type && cols % 8 == 0 && aligned(m, 16)) return {m, cols};
    Rows r{fresh({rows, pitch_of(cols)}, type, m), pitch_of(cols)};
    table[n++] = {vp(m), vpm(r.t), rows, cols, cols, r.pitch, m.scalar_type() == at::kFloat};
    return r;
  }
  void copy(void *s) {
    if (n) check(lib.dfa3d_copy_rows(table, n, type == at::kHalf ? DFA3D_DTYPE_F16 : DFA3D_DTYPE_BF16, s), "dfa3d_copy_rows");
  }
  at::ScalarType type;
  int32_t n = 0;
  dfa3d_row_copy table[DFA3D_MAX_ROW_COPIES];
};

struct Block : Kept {
  int64_t rows = 0, in = 0, hidden = 0, out = 0;      // a single product: hidden unused
  std::vector<int64_t> shape;                         // of the result
  at::ScalarType type = at::kHalf;
  int32_t dtype = 0, act = 0, format = -1;            // format: how the input is kept; -1 whole
  bool plus_x = false, residual = false;
  bool reads = false;                                 // whether a gradient may be wanted that reads what is kept
  bool bias[3] = {false, false, false};               // of a single product: the first
};

// The input as it is kept for the backward, {x, -} or {codes, scales}.
void keep_input(const Block &b, const Tensor &x, variable_list &v) {
  if (b.format < 0) {
    v = {x, Tensor()};
    return;
  }
  Tensor codes = fresh({b.rows, b.in}, at::kByte, x), scales = fresh({b.rows, (b.in + 31) / 32}, at::kByte, x);
  check(lib.dfa3d_compress8(vp(x), b.dtype, b.rows, (int32_t)b.in, b.format, static_cast<uint8_t *>(vpm(codes)),
                            static_cast<uint8_t *>(vpm(scales)), stream_of(x)),
        "dfa3d_compress8");
  v = {codes, scales};
}
Rows kept_input(const Block &b, const variable_list &v, Operands &o) {
  if (b.format < 0) return o.add(v[0], b.rows, b.in);
  Rows r{fresh({b.rows, pitch_of(b.in)}, b.type, v[0]), pitch_of(b.in)};
  check(lib.dfa3d_decompress8(static_cast<const uint8_t *>(vp(v[0])), static_cast<const uint8_t *>(vp(v[1])), b.format, b.rows,
                              (int32_t)b.in, b.dtype, vpm(r.t), r.pitch, stream_of(v[0])),
        "dfa3d_decompress8");
  return r;
}

int32_t out_code(const Block &b, const Tensor &y) { return y.scalar_type() == at::kFloat ? DFA3D_DTYPE_F32 : b.dtype; }

Tensor gradient(const Tensor &g, at::ScalarType type) {      // contiguous, of the forward's type or float32
  return g.scalar_type() == type || g.scalar_type() == at::kFloat ? g.contiguous() : g.to(type).contiguous();
}

struct Wanted {
  const Rows *g;
  int64_t out;
  const Rows *x;
  int64_t in;
  bool weight, bias;
  Tensor *gw, *gb;
};
void weight_gradients(const Block &b, std::initializer_list<Wanted> all, const Tensor &like) {
  dfa3d_weight_gradient table[DFA3D_MAX_WEIGHT_GRADIENTS];
  Tensor dropped;
  int32_t n = 0;
  variable_list alive;
  for (const Wanted &w : all) {
    if (!w.weight && !w.bias) continue;
    Tensor gw = fresh({w.out, w.in}, b.type, like), gb;
    if (w.bias) gb = fresh({w.out}, b.type, like);
    table[n++] = {w.g->data(), w.x->data(), w.g->pitch, w.x->pitch, vpm(gw), vpm(gb), (int32_t)w.in, (int32_t)w.out};
    alive.push_back(gw);
    if (w.weight) *w.gw = gw;
    if (w.bias) *w.gb = gb;
  }
  if (n == 0) return;
  const int64_t bytes = lib.dfa3d_weight_gradients_workspace(table, n, b.rows);
  TORCH_CHECK(bytes >= 0, "dfa3d_weight_gradients_workspace failed: ", lib.dfa3d_last_error());
  Tensor work = fresh({bytes}, at::kByte, like);
  check(lib.dfa3d_weight_gradients(table, n, b.dtype, b.rows, vpm(work), bytes, stream_of(like)), "dfa3d_weight_gradients");
}

// ------------------------------------------------------------------------------------------------
// act(x W^T + b) + residual
// ------------------------------------------------------------------------------------------------
Tensor linear_act_forward(const Block &b, const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &res) {
  Tensor y = fresh(b.shape, res.defined() ? res.scalar_type() : b.type, x);
  Operands o(b.type);
  const Rows xr = o.add(x, b.rows, b.in), wr = o.add(w, b.out, b.in);
  void *s = stream_of(x);
  o.copy(s);
  check(lib.dfa3d_linear_act_forward(xr.data(), xr.pitch, wr.data(), wr.pitch, vp(bias), vp(res), b.dtype, out_code(b, y), b.rows,
                                     (int32_t)b.in, (int32_t)b.out, b.act, vpm(y), s),
        "dfa3d_linear_act_forward");
  return y;
}

struct LinearActFn : torch::autograd::Function<LinearActFn> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const std::optional<Tensor> &bias,
                        const std::optional<Tensor> &res, const c10::intrusive_ptr<Block> &b) {
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor bt = bias ? *bias : Tensor(), rt = res ? *res : Tensor();
    Tensor y = linear_act_forward(*b, x, w, bt, rt);
    variable_list v;
    if (b->reads) {
      keep_input(*b, x, v);
      v.insert(v.end(), {w, bt});
    }
    keep(ctx, b, std::move(v));
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto b = kept_beside<Block>(ctx);
    const bool gx = ctx->needs_input_grad(0), gw = ctx->needs_input_grad(1), gb = b->bias[0] && ctx->needs_input_grad(2);
    Tensor grad_x, grad_w, grad_b;
    if (gx || gw || gb) {
      variable_list v;
      kept<Block>(ctx, v);
      const Tensor &w = v[2], &bias = v[3];
      c10::cuda::CUDAGuard guard(w.device());
      void *s = stream_of(w);
      const Tensor gt = gradient(grads[0], b->type);
      Operands o(b->type);
      const bool slope = b->act != DFA3D_ROW_NONE;
      Rows xr;
      if (slope || gw || gb) xr = kept_input(*b, v, o);
      const Rows wr = slope || gx ? o.add(w, b->out, b->in) : Rows();
      // a 32-bit gradient is not rounded before the derivative has been applied
      const bool wide = slope && gt.scalar_type() == at::kFloat;
      Rows g;
      if (!wide) {
        g = o.add(gt, b->rows, b->out);
      } else if (b->out % 8 == 0 && aligned(gt, 16)) {
        g = {gt, b->out};
      } else {
        g = {fresh({b->rows, pitch_of(b->out)}, at::kFloat, gt), pitch_of(b->out)};
        at::NoGradGuard none;
        g.t.narrow(1, 0, b->out).copy_(gt.view({b->rows, b->out}));
      }
      o.copy(s);
      if (slope) {
        const Rows z{fresh({b->rows, pitch_of(b->out)}, b->type, w), pitch_of(b->out)};
        check(lib.dfa3d_linear_act_slope(xr.data(), xr.pitch, wr.data(), wr.pitch, vp(bias), g.data(), g.pitch, b->dtype,
                                         wide ? DFA3D_DTYPE_F32 : b->dtype, b->rows, (int32_t)b->in, (int32_t)b->out, b->act,
                                         vpm(z.t), z.pitch, s),
              "dfa3d_linear_act_slope");
        g = z;
      }
      if (gx) {
        std::vector<int64_t> shape = b->shape;
        shape.back() = b->in;
        grad_x = fresh(shape, b->type, w);
        check(lib.dfa3d_linear_input_gradient(g.data(), nullptr, g.pitch, wr.data(), nullptr, wr.pitch, nullptr, 0, b->dtype, b->rows,
                                              (int32_t)b->in, (int32_t)b->out, vpm(grad_x), s),
              "dfa3d_linear_input_gradient");
      }
      weight_gradients(*b, {{&g, b->out, &xr, b->in, gw, gb, &grad_w, &grad_b}}, w);
    }
    return once({grad_x, grad_w, grad_b, b->residual && ctx->needs_input_grad(b->bias[0] ? 3 : 2) ? grads[0] : Tensor(), Tensor()},
                grads);
  }
};

bool half_tensor(PyObject *o, Tensor &t) {
  return plain_tensor(o, t) && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf);
}
// a parameter like x, of these sizes
bool parameter(PyObject *o, Tensor &t, const Tensor &x, at::IntArrayRef sizes) {
  return plain_tensor(o, t) && t.scalar_type() == x.scalar_type() && t.device() == x.device() && t.sizes() == sizes;
}
bool optional_parameter(PyObject *o, Tensor &t, const Tensor &x, at::IntArrayRef sizes) {
  return o == Py_None || parameter(o, t, x, sizes);
}
bool optional_residual(PyObject *o, Tensor &t, const Tensor &x, at::IntArrayRef sizes) {
  if (o == Py_None) return true;
  return plain_tensor(o, t) && (t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat) && t.device() == x.device() &&
         t.sizes() == sizes;
}
bool one_of(PyObject *o, std::initializer_list<const char *> names, int32_t first, int32_t none, int32_t &code) {
  code = none;
  if (o == Py_None) return true;
  if (!PyUnicode_CheckExact(o)) return false;
  code = first;
  for (const char *n : names) {
    if (PyUnicode_CompareWithASCIIString(o, n) == 0) return true;
    ++code;
  }
  return false;
}
bool block_arguments(const Tensor &x, PyObject *act, PyObject *checkpoint, Block &b) {
  if (x.dim() < 1 || x.numel() == 0 || x.size(-1) > (1 << 24)) return false;
  b.in = x.size(-1);
  b.rows = x.numel() / b.in;
  b.type = x.scalar_type();
  b.dtype = dtype_code(x);
  b.shape.assign(x.sizes().begin(), x.sizes().end());
  return b.rows < (int64_t(1) << 31) - 128 && one_of(act, {"relu", "silu", "gelu"}, DFA3D_ROW_RELU, DFA3D_ROW_NONE, b.act) &&
         one_of(checkpoint, {"int8", "e4m3"}, DFA3D_FORMAT_INT8, -1, b.format);
}

PyObject *run_linear_act(PyObject *const *a, Py_ssize_t n) {
  // x, weight, bias or None, residual or None, activation, checkpoint
  if (n != 6 || !plain_mode()) return not_plain();
  Tensor x, w, bias, res;
  auto b = c10::make_intrusive<Block>();
  if (!half_tensor(a[0], x) || !block_arguments(x, a[4], a[5], *b) || !plain_tensor(a[1], w) || w.dim() != 2 || w.size(0) == 0 ||
      w.size(0) > (1 << 24) || !parameter(a[1], w, x, {w.size(0), b->in}) || !optional_parameter(a[2], bias, x, {w.size(0)}))
    return not_plain();
  b->out = w.size(0);
  b->shape.back() = b->out;
  if (!optional_residual(a[3], res, x, b->shape)) return not_plain();
  b->residual = res.defined();
  b->bias[0] = bias.defined();
  b->reads = wants_grad(x, w) || (bias.defined() && wants_grad(bias));
  Tensor y;
  {
    pybind11::gil_scoped_release nogil;
    if (b->reads || (res.defined() && wants_grad(res))) {
      y = LinearActFn::apply(x, w, given(bias), given(res), b);
    } else {
      c10::cuda::CUDAGuard guard(x.device());
      y = linear_act_forward(*b, x, w, bias, res);
    }
  }
  return THPVariable_Wrap(y);
}

// ------------------------------------------------------------------------------------------------
// (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual
// ------------------------------------------------------------------------------------------------
struct Weights {
  Tensor gate, up, down, bias_gate, bias_up, bias_down;
};

Tensor gated_forward(const Block &b, const Tensor &x, const Weights &w, const Tensor &res) {
  Tensor y = fresh(b.shape, res.defined() ? res.scalar_type() : b.type, x);
  Operands o(b.type);
  const Rows xr = o.add(x, b.rows, b.in), wg = o.add(w.gate, b.hidden, b.in), wu = o.add(w.up, b.hidden, b.in),
             wd = o.add(w.down, b.out, b.hidden);
  void *s = stream_of(x);
  o.copy(s);
  if (lib.dfa3d_gated_block_supported(out_code(b, y), b.rows, (int32_t)b.in, (int32_t)b.hidden, (int32_t)b.out) &&
      (!res.defined() || aligned(res, 16))) {
    check(lib.dfa3d_gated_block_forward(xr.data(), xr.pitch, wg.data(), wu.data(), wg.pitch, vp(w.bias_gate), vp(w.bias_up), wd.data(),
                                        wd.pitch, vp(w.bias_down), vp(res), b.dtype, out_code(b, y), b.rows, (int32_t)b.in,
                                        (int32_t)b.hidden, (int32_t)b.out, b.act, vpm(y), s),
          "dfa3d_gated_block_forward");
    return y;
  }
  const Rows h{fresh({b.rows, pitch_of(b.hidden)}, b.type, x), pitch_of(b.hidden)};
  check(lib.dfa3d_gated_hidden_forward(xr.data(), xr.pitch, wg.data(), wu.data(), wg.pitch, vp(w.bias_gate), vp(w.bias_up), b.dtype,
                                       b.rows, (int32_t)b.in, (int32_t)b.hidden, b.act, vpm(h.t), h.pitch, s),
        "dfa3d_gated_hidden_forward");
  check(lib.dfa3d_linear_act_forward(h.data(), h.pitch, wd.data(), wd.pitch, vp(w.bias_down), vp(res), b.dtype, out_code(b, y), b.rows,
                                     (int32_t)b.hidden, (int32_t)b.out, DFA3D_ROW_NONE, vpm(y), s),
        "dfa3d_linear_act_forward");
  return y;
}

struct GatedFn : torch::autograd::Function<GatedFn> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &gate, const Tensor &up, const Tensor &down,
                        const std::optional<Tensor> &bg, const std::optional<Tensor> &bu, const std::optional<Tensor> &bd,
                        const std::optional<Tensor> &res, const c10::intrusive_ptr<Block> &b) {
    c10::cuda::CUDAGuard guard(x.device());
    const Weights w{gate, up, down, bg ? *bg : Tensor(), bu ? *bu : Tensor(), bd ? *bd : Tensor()};
    Tensor y = gated_forward(*b, x, w, b->plus_x ? x : res ? *res : Tensor());
    variable_list v;
    if (b->reads) {
      keep_input(*b, x, v);
      v.insert(v.end(), {w.gate, w.up, w.down, w.bias_gate, w.bias_up});
    }
    keep(ctx, b, std::move(v));
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto b = kept_beside<Block>(ctx);
    bool need[8], any = false;
    size_t edge = 0;      // inputs that are absent have none
    for (int i = 0; i < 8; ++i) {
      const bool there = i < 4 || (i < 7 ? b->bias[i - 4] : b->residual);
      need[i] = there && ctx->needs_input_grad(edge);
      edge += there;
      if (i < 7) any |= need[i];
    }
    Tensor gx, gg, gu, gd, gbg, gbu, gbd;
    if (any) {
      variable_list v;
      kept<Block>(ctx, v);
      const Weights w{v[2], v[3], v[4], v[5], v[6], Tensor()};
      c10::cuda::CUDAGuard guard(w.gate.device());
      void *s = stream_of(w.gate);
      const Tensor gt = gradient(grads[0], b->type);
      Operands o(b->type);
      const Rows xr = kept_input(*b, v, o), wg = o.add(w.gate, b->hidden, b->in), wu = o.add(w.up, b->hidden, b->in),
                 wd = o.add(w.down, b->out, b->hidden), g = o.add(gt, b->rows, b->out);
      o.copy(s);
      const int64_t pitch = pitch_of(b->hidden);
      auto hidden = [&] { return Rows{fresh({b->rows, pitch}, b->type, w.gate), pitch}; };
      const Rows dg = hidden(), du = hidden(), h = hidden();
      check(lib.dfa3d_gated_hidden_backward(xr.data(), xr.pitch, wg.data(), wu.data(), wg.pitch, vp(w.bias_gate), vp(w.bias_up),
                                            g.data(), g.pitch, wd.data(), wd.pitch, b->dtype, b->rows, (int32_t)b->in,
                                            (int32_t)b->hidden, (int32_t)b->out, b->act, vpm(dg.t), vpm(du.t), vpm(h.t), pitch, s),
            "dfa3d_gated_hidden_backward");
      if (need[0]) {
        std::vector<int64_t> shape = b->shape;
        shape.back() = b->in;
        gx = fresh(shape, b->type, w.gate);
        check(lib.dfa3d_linear_input_gradient(dg.data(), du.data(), pitch, wg.data(), wu.data(), wg.pitch, b->plus_x ? g.data() : nullptr,
                                              g.pitch, b->dtype, b->rows, (int32_t)b->in, (int32_t)b->hidden, vpm(gx), s),
              "dfa3d_linear_input_gradient");
      }
      weight_gradients(*b,
                       {{&dg, b->hidden, &xr, b->in, need[1], need[4], &gg, &gbg},
                        {&du, b->hidden, &xr, b->in, need[2], need[5], &gu, &gbu},
                        {&g, b->out, &h, b->hidden, need[3], need[6], &gd, &gbd}},
                       w.gate);
    }
    return once({gx, gg, gu, gd, gbg, gbu, gbd, need[7] ? grads[0] : Tensor(), Tensor()}, grads);
  }
};

PyObject *run_gated(PyObject *const *a, Py_ssize_t n) {
  // x, w_gate, w_up, w_down, b_gate, b_up, b_down (or None), residual or None, plus_x, activation, checkpoint
  if (n != 11 || !plain_mode()) return not_plain();
  Tensor x, res;
  Weights w;
  auto b = c10::make_intrusive<Block>();
  if (!half_tensor(a[0], x) || !block_arguments(x, a[9], a[10], *b) || !plain_tensor(a[1], w.gate) || w.gate.dim() != 2 ||
      !plain_tensor(a[3], w.down) || w.down.dim() != 2 || !PyBool_Check(a[8]))
    return not_plain();
  b->hidden = w.gate.size(0);
  b->out = w.down.size(0);
  b->plus_x = a[8] == Py_True;
  if (b->hidden < 1 || b->out < 1 || b->hidden > (1 << 24) || b->out > (1 << 24) || !parameter(a[1], w.gate, x, {b->hidden, b->in}) ||
      !parameter(a[2], w.up, x, {b->hidden, b->in}) || !parameter(a[3], w.down, x, {b->out, b->hidden}) ||
      !optional_parameter(a[4], w.bias_gate, x, {b->hidden}) || !optional_parameter(a[5], w.bias_up, x, {b->hidden}) ||
      !optional_parameter(a[6], w.bias_down, x, {b->out}) || (b->plus_x && (b->out != b->in || a[7] != Py_None)))
    return not_plain();
  b->shape.back() = b->out;
  if (!optional_residual(a[7], res, x, b->shape)) return not_plain();
  b->residual = res.defined();
  Tensor y;
  {
    pybind11::gil_scoped_release nogil;
    b->reads = wants_grad(x, w.gate, w.up, w.down);
    const Tensor *biases[3] = {&w.bias_gate, &w.bias_up, &w.bias_down};
    for (int i = 0; i < 3; ++i) {
      b->bias[i] = biases[i]->defined();
      b->reads |= b->bias[i] && wants_grad(*biases[i]);
    }
    if (b->reads || (res.defined() && wants_grad(res))) {
      y = GatedFn::apply(x, w.gate, w.up, w.down, given(w.bias_gate), given(w.bias_up), given(w.bias_down), given(res), b);
    } else {
      c10::cuda::CUDAGuard guard(x.device());
      y = gated_forward(*b, x, w, b->plus_x ? x : res);
    }
  }
  return THPVariable_Wrap(y);
}

// ------------------------------------------------------------------------------------------------
// 8 bits by themselves
// ------------------------------------------------------------------------------------------------
bool format_argument(PyObject *o, int32_t &format) {
  return o != Py_None && one_of(o, {"int8", "e4m3"}, DFA3D_FORMAT_INT8, -1, format);
}

PyObject *run_compress8(PyObject *const *a, Py_ssize_t n) {
  // x, format -> (codes, scales)
  int32_t format;
  Tensor x;
  if (n != 2 || !plain_mode() || !plain_tensor(a[0], x) || !storage_type(x.scalar_type()) || x.dim() < 1 || x.numel() == 0 ||
      x.size(-1) > (1 << 30) || !format_argument(a[1], format))
    return not_plain();
  Tensor codes, scales;
  {
    pybind11::gil_scoped_release nogil;
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    codes = fresh({rows, cols}, at::kByte, x);
    scales = fresh({rows, (cols + 31) / 32}, at::kByte, x);
    check(lib.dfa3d_compress8(vp(x), dtype_code(x), rows, (int32_t)cols, format, static_cast<uint8_t *>(vpm(codes)),
                              static_cast<uint8_t *>(vpm(scales)), stream_of(x)),
          "dfa3d_compress8");
  }
  PyObject *t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(codes));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(scales));
  return t;
}

PyObject *run_decompress8(PyObject *const *a, Py_ssize_t n) {
  // codes, scales, shape, dtype, format
  int32_t format;
  Tensor codes, scales;
  if (n != 5 || !plain_mode() || !plain_tensor(a[0], codes) || !plain_tensor(a[1], scales) || codes.scalar_type() != at::kByte ||
      scales.scalar_type() != at::kByte || !one_device(codes, scales) || !PyTuple_Check(a[2]) || PyTuple_GET_SIZE(a[2]) < 1 ||
      !THPDtype_Check(a[3]) || !format_argument(a[4], format))
    return not_plain();
  const at::ScalarType type = reinterpret_cast<THPDtype *>(a[3])->scalar_type;
  std::vector<int64_t> shape((size_t)PyTuple_GET_SIZE(a[2]));
  int64_t count = 1;
  for (size_t i = 0; i < shape.size(); ++i)
    if (!integer(PyTuple_GET_ITEM(a[2], (Py_ssize_t)i), shape[i]) || shape[i] < 1 || shape[i] > codes.numel() ||
        (count *= shape[i]) > codes.numel())
      return not_plain();
  const int64_t cols = shape.back(), rows = count / cols;
  if (!storage_type(type) || cols > (1 << 30) || codes.numel() != count || scales.numel() != rows * ((cols + 31) / 32)) return not_plain();
  Tensor x;
  {
    pybind11::gil_scoped_release nogil;
    c10::cuda::CUDAGuard guard(codes.device());
    x = fresh(shape, type, codes);
    check(lib.dfa3d_decompress8(static_cast<const uint8_t *>(vp(codes)), static_cast<const uint8_t *>(vp(scales)), format, rows,
                                (int32_t)cols, dtype_code(x), vpm(x), cols, stream_of(x)),
          "dfa3d_decompress8");
  }
  return THPVariable_Wrap(x);
}

#define FAST(name, expr)                                                             \
  PyObject *py_##name(PyObject *, PyObject *const *a, Py_ssize_t n) {                 \
    HANDLE_TH_ERRORS                                                                  \
    return expr;                                                                      \
    END_HANDLE_TH_ERRORS                                                              \
  }
FAST(linear_act, run_linear_act(a, n))
FAST(gated_feed_forward, run_gated(a, n))
FAST(compress8, run_compress8(a, n))
FAST(decompress8, run_decompress8(a, n))
#undef FAST

}  // namespace

namespace dfa3d_torch {
#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef ffn_methods[] = {
    FAST(linear_act), FAST(gated_feed_forward), FAST(compress8), FAST(decompress8), {nullptr, nullptr, 0, nullptr},
};
#undef FAST
}  // namespace dfa3d_torch
