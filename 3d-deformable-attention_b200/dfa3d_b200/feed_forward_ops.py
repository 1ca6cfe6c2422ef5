"""The feed-forward block in 16 bits on the tensor cores, on the library's own kernels (C entry points ``dfa3d_linear_*``,
``dfa3d_gated_hidden_*``, ``dfa3d_weight_gradients``).

The reference's layers end in ``norm(x + W2 relu(W1 x))`` (BEVFormer_DFA3D/projects/mmdet3d_plugin/bevformer/modules/
custom_base_transformer_layer.py), float32 products with the bias, the activation and the sum as passes of their own.  Here

  * ``linear_act(x, weight, bias, activation, residual)``: act(x W^T + b) + residual, one kernel;
  * ``gated_feed_forward(x, w_gate, w_up, w_down, ...)``: (act(x Wg^T) * (x Wu^T)) Wd^T + residual, two kernels;

with sums, bias, activation, residual and derivatives in 32 bits and one rounding at the end of a kernel.  Both keep their input for
the backward and nothing else: what the activation's derivative needs is formed again by the kernel that applies it, which reads
less than it would if it had been kept.  With ``checkpoint="int8"`` or ``"e4m3"`` the input is kept in 8 bits (``checkpoint_ops``);
the backward is then the gradient at what the 8 bits stand for, the forward is not touched.

bfloat16 and float16 CUDA tensors; the residual and with it the result may be float32, so that a residual stream is never rounded.
Under autocast everything but the residual is cast to autocast's type.  ``LinearAct`` and ``GatedFeedForward`` hold float32 parameters
and cast them.  There is no fallback path; float32 products are ``layer_ops.Linear``'s.
"""
import ctypes

import torch
import torch.nn as nn
from torch.autograd.function import Function, once_differentiable

from . import _lib
from .checkpoint_ops import Compressed8, check_format, compress8, into
from .dropout_ops import CounterDropout, keep, kept
from .layer_ops import runs_forward_only

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_ACTS = {None: _lib.ROW_NONE, "relu": _lib.ROW_RELU, "silu": _lib.ROW_SILU, "gelu": _lib.ROW_GELU}


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check_matrix(t, name, shape, like):
    if t.dtype != like.dtype or t.device != like.device or tuple(t.shape) != shape:
        raise RuntimeError(f"{name} must be {shape} {like.dtype} on {like.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")


def _rows_of(t, name):
    if t.dim() != 2 or t.shape[0] == 0:
        raise RuntimeError(f"{name} must have two dimensions and at least one row, got {tuple(t.shape)}")
    return t.shape[0]


def _check_input(x, activation, checkpoint):
    if not x.is_cuda or x.dtype not in _DTYPES:
        raise RuntimeError(f"x must be a bfloat16 or float16 CUDA tensor, got {x.dtype} on {x.device}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError(f"x must have rows of at least one element, got {tuple(x.shape)}")
    if activation not in _ACTS:
        raise ValueError(f"activation must be one of {list(_ACTS)}, got {activation!r}")
    if checkpoint is not None:
        check_format(checkpoint, "checkpoint")


def _check_residual(residual, shape, x):
    if residual.dtype not in (x.dtype, torch.float32) or residual.device != x.device or tuple(residual.shape) != shape:
        raise RuntimeError(f"residual must be {shape} {x.dtype} or float32 on {x.device}, got {tuple(residual.shape)} "
                           f"{residual.dtype} on {residual.device}")


def _rows(t):
    return t.reshape(-1, t.shape[-1])


def _pitch(cols):
    return (cols + 7) // 8 * 8


def _workspace(rows, cols, like):
    """Rows that begin on a 16-byte boundary: (tensor, pitch)."""
    return torch.empty((rows, _pitch(cols)), dtype=like.dtype, device=like.device), _pitch(cols)


def _operands(dtype, *matrices):
    """Each (rows, cols) matrix as the products read it, (tensor, pitch): itself where its rows begin on a 16-byte boundary, a copy
    otherwise; float32 ones rounded to dtype.  All copies with one launch."""
    out, copies = [], []
    for m in matrices:
        m = m.contiguous()
        if m.dtype == dtype and m.shape[1] % 8 == 0 and m.data_ptr() % 16 == 0:
            out.append((m, m.shape[1]))
            continue
        to = torch.empty((m.shape[0], _pitch(m.shape[1])), dtype=dtype, device=m.device)
        out.append((to, to.shape[1]))
        copies.append((m, to))
    if copies:
        table = (_lib.RowCopy * len(copies))(*[
            _lib.RowCopy(m.data_ptr(), to.data_ptr(), m.shape[0], m.shape[1], m.shape[1], to.shape[1], int(m.dtype == torch.float32))
            for m, to in copies])
        _lib.call_plain("dfa3d_copy_rows", ctypes.byref(table), len(copies), _DTYPES[dtype], _stream(copies[0][0]))
    return out


def _keep_input(ctx, x, checkpoint, *others):
    """Keeps x, whole or in 8 bits, and the other tensors."""
    ctx.kept_as = None
    if checkpoint is None:
        keep(ctx, x, None, *others)
    else:
        c = compress8(x, checkpoint)
        ctx.kept_as = (c.shape, c.dtype, c.format)
        keep(ctx, c.codes, c.scales, *others)


def _kept_input(ctx):
    """(x as an operand, its pitch), and the other tensors."""
    a, b, *others = kept(ctx)
    if ctx.kept_as is None:
        return _operands(a.dtype, _rows(a))[0], others
    shape, dtype, fmt = ctx.kept_as
    x, pitch = torch.empty((a.shape[0], _pitch(shape[-1])), dtype=dtype, device=a.device), _pitch(shape[-1])
    into(Compressed8(a, b, shape, dtype, fmt), x, pitch)
    return (x, pitch), others


def _weight_gradients(dtype, rows, problems):
    """problems: (grad, pitch, out, x, pitch, in, want bias); the gradients of each, [weight, bias or None]."""
    out = []
    table = (_lib.WeightGradient * len(problems))()
    for t, (g, gp, n, x, xp, k, bias) in zip(table, problems):
        gw = torch.empty((n, k), dtype=dtype, device=g.device)
        gb = torch.empty(n, dtype=dtype, device=g.device) if bias else None
        out.append((gw, gb))
        t.grad, t.x, t.grad_pitch, t.x_pitch, t.out_features, t.in_features = g.data_ptr(), x.data_ptr(), gp, xp, n, k
        t.grad_weight, t.grad_bias = gw.data_ptr(), _ptr(gb)
    g = problems[0][0]
    work = torch.empty(_lib.size("dfa3d_weight_gradients_workspace", ctypes.byref(table), len(problems), rows), dtype=torch.uint8,
                       device=g.device)
    _lib.call_plain("dfa3d_weight_gradients", ctypes.byref(table), len(problems), _DTYPES[dtype], rows, work.data_ptr(), work.numel(),
                    _stream(g))
    return out


@_lib.native_apply("linear_act")
class LinearActFunction(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, checkpoint):
        """act(x W^T + b) + residual."""
        _check_input(x, activation, checkpoint)
        K, N = x.shape[-1], _rows_of(weight, "weight")
        _check_matrix(weight, "weight", (N, K), x)
        if bias is not None:
            _check_matrix(bias, "bias", (N,), x)
            bias = bias.contiguous()
        shape = tuple(x.shape[:-1]) + (N,)
        if residual is not None:
            _check_residual(residual, shape, x)
            residual = residual.contiguous()
        x, weight = x.contiguous(), weight.contiguous()
        y = torch.empty(shape, dtype=x.dtype if residual is None else residual.dtype, device=x.device)
        rows = x.numel() // K
        if y.numel():
            with torch.cuda.device(x.device):
                (xo, xp), (wo, wp) = _operands(x.dtype, _rows(x), weight)
                _lib.call_plain("dfa3d_linear_act_forward", xo.data_ptr(), xp, wo.data_ptr(), wp, _ptr(bias), _ptr(residual),
                                _DTYPES[x.dtype], _lib.DTYPE_F32 if y.dtype == torch.float32 else _DTYPES[x.dtype], rows, K, N,
                                _ACTS[activation], y.data_ptr(), _stream(x))
        if any(ctx.needs_input_grad[:3]):
            _keep_input(ctx, x, checkpoint, weight, bias)
        ctx.act, ctx.has_residual = _ACTS[activation], residual is not None
        ctx.sizes, ctx.x_shape, ctx.dtype = (rows, K, N), x.shape, x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        need = ctx.needs_input_grad
        grad_x = grad_w = grad_b = None
        rows, K, N = ctx.sizes
        if any(need[:3]):
            with torch.cuda.device(grad_y.device):
                (x, xp), (weight, bias) = _kept_input(ctx)
                g = grad_y if grad_y.dtype in (ctx.dtype, torch.float32) else grad_y.to(ctx.dtype)
                g, wide = _rows(g).contiguous(), _DTYPES[ctx.dtype]
                if ctx.act != _lib.ROW_NONE and g.dtype == torch.float32:
                    (w, wp), = _operands(ctx.dtype, weight)           # not rounded before the derivative has been applied
                    wide, gp = _lib.DTYPE_F32, _pitch(N)
                    if gp != N or g.data_ptr() % 16:
                        on_grid = torch.empty((rows, gp), dtype=torch.float32, device=g.device)
                        on_grid[:, :N].copy_(g)
                        g = on_grid
                else:
                    (w, wp), (g, gp) = _operands(ctx.dtype, weight, g)
                st = _stream(g)
                if ctx.act != _lib.ROW_NONE:
                    dz, zp = _workspace(rows, N, x)
                    _lib.call_plain("dfa3d_linear_act_slope", x.data_ptr(), xp, w.data_ptr(), wp, _ptr(bias), g.data_ptr(), gp,
                                    _DTYPES[ctx.dtype], wide, rows, K, N, ctx.act, dz.data_ptr(), zp, st)
                    g, gp = dz, zp
                if need[0]:
                    grad_x = torch.empty(ctx.x_shape, dtype=ctx.dtype, device=g.device)
                    _lib.call_plain("dfa3d_linear_input_gradient", g.data_ptr(), None, gp, w.data_ptr(), None, wp, None, 0,
                                    _DTYPES[ctx.dtype], rows, K, N, grad_x.data_ptr(), st)
                if need[1] or need[2]:
                    (grad_w, grad_b), = _weight_gradients(ctx.dtype, rows, [(g, gp, N, x, xp, K, need[2])])
                    grad_w = grad_w if need[1] else None
        return grad_x, grad_w, grad_b, (grad_y if ctx.has_residual and need[3] else None), None, None


@_lib.native_apply("gated_feed_forward")
class GatedFeedForwardFunction(Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual, plus_x, activation, checkpoint):
        """(act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd [+ residual, or + x]."""
        _check_input(x, activation, checkpoint)
        E, F, N = x.shape[-1], _rows_of(w_gate, "w_gate"), _rows_of(w_down, "w_down")
        _check_matrix(w_gate, "w_gate", (F, E), x)
        _check_matrix(w_up, "w_up", (F, E), x)
        _check_matrix(w_down, "w_down", (N, F), x)
        for b, n, name in ((b_gate, F, "b_gate"), (b_up, F, "b_up"), (b_down, N, "b_down")):
            if b is not None:
                _check_matrix(b, name, (n,), x)
        shape = tuple(x.shape[:-1]) + (N,)
        x = x.contiguous()
        if plus_x:
            residual = x
        if residual is not None:
            _check_residual(residual, shape, x)
            residual = residual.contiguous()
        w_gate, w_up, w_down = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
        b_gate, b_up, b_down = (None if b is None else b.contiguous() for b in (b_gate, b_up, b_down))
        y = torch.empty(shape, dtype=x.dtype if residual is None else residual.dtype, device=x.device)
        rows, dt = x.numel() // E, _DTYPES[x.dtype]
        if y.numel():
            with torch.cuda.device(x.device):
                (xo, xp), (wg, wp), (wu, _), (wd, dp) = _operands(x.dtype, _rows(x), w_gate, w_up, w_down)
                out, st = _lib.DTYPE_F32 if y.dtype == torch.float32 else dt, _stream(x)
                if _lib.load().dfa3d_gated_block_supported(out, rows, E, F, N) and (residual is None or residual.data_ptr() % 16 == 0):
                    _lib.call_plain("dfa3d_gated_block_forward", xo.data_ptr(), xp, wg.data_ptr(), wu.data_ptr(), wp, _ptr(b_gate),
                                    _ptr(b_up), wd.data_ptr(), dp, _ptr(b_down), _ptr(residual), dt, out, rows, E, F, N,
                                    _ACTS[activation], y.data_ptr(), st)
                else:
                    h, hp = _workspace(rows, F, x)
                    _lib.call_plain("dfa3d_gated_hidden_forward", xo.data_ptr(), xp, wg.data_ptr(), wu.data_ptr(), wp, _ptr(b_gate),
                                    _ptr(b_up), dt, rows, E, F, _ACTS[activation], h.data_ptr(), hp, st)
                    _lib.call_plain("dfa3d_linear_act_forward", h.data_ptr(), hp, wd.data_ptr(), dp, _ptr(b_down), _ptr(residual), dt,
                                    out, rows, F, N, _lib.ROW_NONE, y.data_ptr(), st)
        if any(ctx.needs_input_grad[:7]):
            _keep_input(ctx, x, checkpoint, w_gate, w_up, w_down, b_gate, b_up)
        ctx.act, ctx.plus_x = _ACTS[activation], plus_x
        ctx.sizes, ctx.x_shape, ctx.dtype = (rows, E, F, N), x.shape, x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        need = ctx.needs_input_grad
        rows, E, F, N = ctx.sizes
        grad_x = gg = gu = gd = bg = bu = bd = None
        if any(need[:7]):
            with torch.cuda.device(grad_y.device):
                (x, xp), (w_gate, w_up, w_down, b_gate, b_up) = _kept_input(ctx)
                g = grad_y if grad_y.dtype in (ctx.dtype, torch.float32) else grad_y.to(ctx.dtype)
                (wg, wp), (wu, _), (wd, dp), (g, gp) = _operands(ctx.dtype, w_gate, w_up, w_down, _rows(g))
                dt, st = _DTYPES[ctx.dtype], _stream(g)
                (dg, hp), (du, _), (h, _) = (_workspace(rows, F, g) for _ in range(3))
                _lib.call_plain("dfa3d_gated_hidden_backward", x.data_ptr(), xp, wg.data_ptr(), wu.data_ptr(), wp, _ptr(b_gate),
                                _ptr(b_up), g.data_ptr(), gp, wd.data_ptr(), dp, dt, rows, E, F, N, ctx.act, dg.data_ptr(),
                                du.data_ptr(), h.data_ptr(), hp, st)
                if need[0]:
                    grad_x = torch.empty(ctx.x_shape, dtype=ctx.dtype, device=g.device)
                    _lib.call_plain("dfa3d_linear_input_gradient", dg.data_ptr(), du.data_ptr(), hp, wg.data_ptr(), wu.data_ptr(), wp,
                                    g.data_ptr() if ctx.plus_x else None, gp, dt, rows, E, F, grad_x.data_ptr(), st)
                wanted = [(need[1] or need[4], (dg, hp, F, x, xp, E, need[4])), (need[2] or need[5], (du, hp, F, x, xp, E, need[5])),
                          (need[3] or need[6], (g, gp, N, h, hp, F, need[6]))]
                if any(w for w, _ in wanted):
                    got = iter(_weight_gradients(ctx.dtype, rows, [p for w, p in wanted if w]))
                    (gg, bg), (gu, bu), (gd, bd) = (next(got) if w else (None, None) for w, _ in wanted)
                    gg, gu, gd = gg if need[1] else None, gu if need[2] else None, gd if need[3] else None
        return grad_x, gg, gu, gd, bg, bu, bd, (grad_y if need[7] else None), None, None, None


def _autocast(*tensors):
    """The tensors as autocast wants them."""
    if not torch.is_autocast_enabled("cuda"):
        return tensors
    dt = torch.get_autocast_dtype("cuda")
    return tuple(t if t is None or not t.is_floating_point() else t.to(dt) for t in tensors)


def linear_act(x, weight, bias=None, activation=None, residual=None, checkpoint=None):
    """act(x W^T + b) + residual for x (..., in), weight (out, in), bias (out,), residual (..., out): bfloat16 or float16, the
    residual also float32; the result has the residual's type.  activation: None, "relu", "silu" or "gelu" (with erf).  checkpoint:
    None, "int8" or "e4m3", how x is kept for the backward."""
    x, weight, bias = _autocast(x, weight, bias)
    return LinearActFunction.apply(x, weight, bias, residual, activation, checkpoint)


def gated_feed_forward(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu", residual=None, checkpoint=None):
    """(act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual for x (..., in), w_gate and w_up (hidden, in), w_down (out, hidden).
    The types, activations and checkpoints of ``linear_act``.  The hidden rows are rounded to x's type between the two products.
    residual may be x itself: its gradient is then added inside the last kernel."""
    plus_x = residual is x and x.dtype in _DTYPES
    x2, w_gate, w_up, w_down, b_gate, b_up, b_down = _autocast(x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    plus_x = plus_x and x2 is x
    return GatedFeedForwardFunction.apply(x2, w_gate, w_up, w_down, b_gate, b_up, b_down, None if plus_x else residual, plus_x,
                                          activation, checkpoint)


class _Computed(nn.Module):
    """float32 parameters, computed with in 16 bits: x's type where it has one, autocast's under autocast, compute_dtype otherwise."""

    compute_dtype = torch.bfloat16

    def _type(self, x):
        if torch.is_autocast_enabled("cuda"):
            return torch.get_autocast_dtype("cuda")
        return x.dtype if x.dtype in _DTYPES else self.compute_dtype


def _plain_product(m):
    """Whether calling m is a product with its weight and bias and nothing else."""
    return (type(m).forward is nn.Linear.forward or (type(m).forward is LinearAct.forward and m.activation is None)) \
        and runs_forward_only(m)


def _to(t, dtype):
    return None if t is None else t.to(dtype)


class LinearAct(nn.Linear, _Computed):
    """``torch.nn.Linear`` (same parameters and state-dict keys), an activation and a residual on ``linear_act``.  Unlike it, a float32 x
    without a residual gives a result of compute_dtype: a float32 result takes a float32 residual."""

    def __init__(self, in_features, out_features, bias=True, activation=None, checkpoint=None, compute_dtype=torch.bfloat16):
        super().__init__(in_features, out_features, bias)
        self.activation, self.checkpoint, self.compute_dtype = activation, checkpoint, compute_dtype

    def forward(self, x, residual=None):
        dt = self._type(x)
        return linear_act(x.to(dt), self.weight.to(dt), _to(self.bias, dt), self.activation, residual, self.checkpoint)


_PLAIN_ACTS = {None: lambda z: z, "relu": torch.relu, "silu": nn.functional.silu, "gelu": nn.functional.gelu}


class GatedFeedForward(_Computed):
    """``dropout((act(gate(x)) * up(x)) down) [+ residual]`` on ``gated_feed_forward``.  A float32 residual is added unrounded.  Where
    ``gate``, ``up`` or ``down`` is more than a product with its parameters (hooks on it, a module that has replaced it), the three are
    called one by one instead: their results are rounded in between too, and they keep their inputs whole."""

    def __init__(self, embed_dims, hidden_dims, activation="silu", bias=True, dropout=0.0, counter_dropout=False, checkpoint=None,
                 compute_dtype=torch.bfloat16):
        super().__init__()
        self.gate = LinearAct(embed_dims, hidden_dims, bias)
        self.up = LinearAct(embed_dims, hidden_dims, bias)
        self.down = LinearAct(hidden_dims, embed_dims, bias)
        self.dropout = CounterDropout(dropout) if counter_dropout else nn.Dropout(dropout)
        self.activation, self.checkpoint, self.compute_dtype = activation, checkpoint, compute_dtype

    def drops(self):
        """Whether the dropout does anything, so that the residual has to wait for it."""
        return not runs_forward_only(self.dropout) or (self.dropout.training and self.dropout.p > 0)

    def _one_by_one(self, x, residual):
        if self.activation not in _ACTS:
            raise ValueError(f"activation must be one of {list(_ACTS)}, got {self.activation!r}")
        h = _PLAIN_ACTS[self.activation](self.gate(x).float()) * self.up(x).float()
        y = self.down(h.to(x.dtype))
        return y if residual is None else residual + y

    def branch(self, x, residual=None):
        """The block without its dropout."""
        dt = self._type(x)
        narrow = x.to(dt)
        if not all(_plain_product(m) for m in (self.gate, self.up, self.down)):
            return self._one_by_one(narrow, residual)
        w = [t for m in (self.gate, self.up, self.down) for t in (m.weight.to(dt), _to(m.bias, dt))]
        return gated_feed_forward(narrow, w[0], w[2], w[4], w[1], w[3], w[5], self.activation,
                                  narrow if residual is x and narrow is x else residual, self.checkpoint)

    def forward(self, x, residual=None):
        if not self.drops():
            return self.branch(x, residual)
        y = self.dropout(self.branch(x))
        return y if residual is None else residual + y
