"""Dropout whose mask is never stored, alone and at the end of a residual block, on the library's own kernels (C entry points
``dfa3d_dropout_*`` and ``dfa3d_dropout_add_layer_norm_*``).

The reference trains with dropout in every block of its layers (BEVFormer_DFA3D/projects/mmdet3d_plugin/bevformer/modules/
spatial_cross_attention.py:616-751, temporal_self_attention.py:26-272, decoder.py:133-345, and the feed-forward block): torch's
keeps a byte for every element until the backward and is a pass of its own over the tensor each way.  Here the mask is a
function of (seed, site, element), formed by a counter-based generator inside whichever kernel needs it:

  * ``dropout(x, p, seed, site, activation, residual)``: [residual +] dropout(act(x)), one pass each way;
  * ``dropout_add_layer_norm(x, residual, weight, bias, p, seed, site, eps)``: LayerNorm(residual + dropout(x));
  * ``CounterDropout``: a ``torch.nn.Dropout`` that draws a seed of torch's generator for every call.

``seed`` is one int64 on the device, so that a captured graph that draws it (``draw_seed``) has a new mask in every replay; a
caller that wants the same mask again passes the same seed and site.  Element i of the tensor in row-major order, whatever its
strides, takes word i mod 4 of Philox4x32-7 (Salmon et al., SC 2011) at counter (i / 4 low, i / 4 high, site, 0) and is kept
where the word is >= p * 2^32.  A dropped element is 0 whatever it was.

CUDA tensors of float32, bfloat16 or float16; arithmetic is float32.  There is no fallback path.
"""
import torch
import torch.nn as nn
from torch.autograd.function import Function, once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_ACTS = {None: _lib.ROW_NONE, "relu": _lib.ROW_RELU}


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _check_tensor(t, name, like=None):
    if not t.is_cuda or t.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be a float32, bfloat16 or float16 CUDA tensor, got {t.dtype} on {t.device}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape != like.shape):
        raise RuntimeError(f"{name} {tuple(t.shape)} {t.dtype} on {t.device} does not match x {tuple(like.shape)} {like.dtype} "
                           f"on {like.device}")


def _check_rule(p, seed, site, x):
    """(p, site) as the kernels take them."""
    p, site = float(p), int(site)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability has to be between 0 and 1, but got {p}")
    if not 0 <= site < 2 ** 31:
        raise ValueError(f"site has to be in [0, 2^31), but got {site}")
    if seed is None:
        if p > 0.0:
            raise RuntimeError("seed must be one int64 on the device where p > 0")
    elif seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
        raise RuntimeError(f"seed must be one int64 on {x.device}, got {tuple(seed.shape)} {seed.dtype} on {seed.device}")
    return p, site


def _ptr(t):
    return None if t is None else t.data_ptr()


def keep(ctx, *tensors):
    """Keeps tensors for the backward, and what they are beside them."""
    ctx.save_for_backward(*tensors)
    ctx.was = [None if t is None else (t.shape, t.dtype, t.device) for t in tensors]


def kept(ctx):
    """The tensors of ``keep``, contiguous.  The kernels read them by address: what a saved-tensor hook handed back instead has to be
    of the same type, size and device."""
    out = []
    for t, was in zip(ctx.saved_tensors, ctx.was):
        if (None if t is None else (t.shape, t.dtype, t.device)) != was:
            raise RuntimeError("a saved-tensor hook returned a tensor of another type, size or device than it was given")
        out.append(None if t is None else t.contiguous())
    return out


def draw_seed(device="cuda", generator=None):
    """A seed for one pass, drawn on the device from torch's generator (or the given one): follows ``torch.manual_seed``, and in
    a captured graph every replay draws another."""
    return torch.empty(1, dtype=torch.int64, device=device).random_(generator=generator)


@_lib.native_apply("dropout")
class DropoutFunction(Function):
    @staticmethod
    def forward(ctx, x, residual, seed, p, site, activation):
        """y = [residual +] keep * act(x) / (1 - p); residual None or like x, activation None or "relu"."""
        _check_tensor(x, "x")
        if residual is not None:
            _check_tensor(residual, "residual", x)
            residual = residual.contiguous()
        if activation not in _ACTS:
            raise ValueError("activation must be None or 'relu'")
        p, site = _check_rule(p, seed, site, x)
        x = x.contiguous()
        y = torch.empty_like(x)
        with torch.cuda.device(x.device):
            _lib.call_plain("dfa3d_dropout_forward", x.data_ptr(), _ptr(residual), _DTYPES[x.dtype], x.numel(), _ACTS[activation],
                            p, _ptr(seed), site, y.data_ptr(), _stream(x))
        # a ReLU's zeros and the dropped elements are the zeros of the result, unless a residual was added
        ctx.by_result = activation is not None and residual is None
        keep(ctx, seed, None if activation is None else y if ctx.by_result else x)
        ctx.has_residual, ctx.p, ctx.site, ctx.dtype = residual is not None, p, site, x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        seed, ref = kept(ctx)
        grad_x = None
        if ctx.needs_input_grad[0]:
            g = grad_y.to(ctx.dtype).contiguous()
            grad_x = torch.empty_like(g)
            with torch.cuda.device(g.device):
                _lib.call_plain("dfa3d_dropout_backward", g.data_ptr(), _ptr(ref), int(ctx.by_result), _DTYPES[g.dtype],
                                g.numel(), ctx.p, _ptr(seed), ctx.site, grad_x.data_ptr(), _stream(g))
        return grad_x, (grad_y if ctx.has_residual and ctx.needs_input_grad[1] else None), None, None, None, None


def dropout(x, p, seed, site=0, activation=None, residual=None):
    """[residual +] dropout(act(x)): elements are kept with probability 1 - p and scaled by 1 / (1 - p).  seed: one int64 on x's
    device (None where p is 0); site tells the calls that share a seed apart."""
    return DropoutFunction.apply(x, residual, seed, p, site, activation)


@_lib.native_apply("dropout_add_layer_norm")
class DropoutAddLayerNormFunction(Function):
    @staticmethod
    @torch.amp.custom_fwd(device_type="cuda", cast_inputs=torch.float32)
    def forward(ctx, x, residual, weight, bias, seed, p, site, eps):
        """LayerNorm(residual + keep * x / (1 - p)) over the last dimension."""
        _check_tensor(x, "x")
        _check_tensor(residual, "residual", x)
        p, site = _check_rule(p, seed, site, x)
        if x.dim() == 0:
            raise RuntimeError("x must have at least one dimension")
        E = x.shape[-1]
        for t, n in ((weight, "weight"), (bias, "bias")):
            if t.dtype != torch.float32 or t.device != x.device or t.numel() != E:
                raise RuntimeError(f"{n} must be {E} float32 elements on {x.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
        rows = x.numel() // E if E else 0
        _lib.size("dfa3d_dropout_add_layer_norm_workspace", rows, E)          # refuses sizes before anything is copied
        x, residual, weight, bias = x.contiguous(), residual.contiguous(), weight.contiguous(), bias.contiguous()
        y = torch.empty_like(x)
        stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)
        with torch.cuda.device(x.device):
            _lib.call_plain("dfa3d_dropout_add_layer_norm_forward", x.data_ptr(), residual.data_ptr(), weight.data_ptr(),
                            bias.data_ptr(), _DTYPES[x.dtype], rows, E, p, _ptr(seed), site, float(eps), y.data_ptr(),
                            stats[0].data_ptr(), stats[1].data_ptr(), _stream(x))
        keep(ctx, x, residual, weight, stats, seed)
        ctx.p, ctx.site, ctx.bias_shape = p, site, bias.shape
        return y

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    @once_differentiable
    def backward(ctx, grad_y):
        x, residual, weight, stats, seed = kept(ctx)
        E, rows = x.shape[-1], stats.shape[1]
        g = grad_y.to(x.dtype).contiguous()
        need = ctx.needs_input_grad
        grad_x = torch.empty_like(x) if need[0] else None
        grad_r = torch.empty_like(x) if need[1] else None
        params = grad_wb = work = None
        if need[2] or need[3]:
            grad_wb = torch.empty((2, (E + 3) // 4 * 4), dtype=torch.float32, device=x.device)
            params = grad_wb[:, :E]
            work = torch.empty(_lib.size("dfa3d_dropout_add_layer_norm_workspace", rows, E), dtype=torch.uint8, device=x.device)
        with torch.cuda.device(x.device):
            _lib.call_plain("dfa3d_dropout_add_layer_norm_backward", g.data_ptr(), x.data_ptr(), residual.data_ptr(),
                            weight.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), _DTYPES[x.dtype], rows, E, ctx.p,
                            _ptr(seed), ctx.site, _ptr(grad_x), _ptr(grad_r), None if params is None else params[0].data_ptr(),
                            None if params is None else params[1].data_ptr(), _ptr(work), 0 if work is None else work.numel(),
                            _stream(x))
        grad_w = params[0].view(weight.shape) if need[2] else None
        grad_b = params[1].view(ctx.bias_shape) if need[3] else None
        return grad_x, grad_r, grad_w, grad_b, None, None, None, None


def dropout_add_layer_norm(x, residual, weight, bias, p, seed, site=0, eps=1e-5):
    """LayerNorm(residual + dropout(x)) over the last dimension (up to 1024 columns): the end of a post-norm residual block.  x and
    residual of one type; weight and bias float32."""
    return DropoutAddLayerNormFunction.apply(x, residual, weight, bias, seed, p, site, eps)


class CounterDropout(nn.Dropout):
    """``torch.nn.Dropout`` on ``dropout``: no stored mask.  Every call in training mode draws a seed from torch's generator."""

    def __init__(self, p=0.5):
        super().__init__(p)

    def forward(self, x):
        if not self.training or self.p == 0.0:
            return x
        return dropout(x, self.p, draw_seed(x.device))
