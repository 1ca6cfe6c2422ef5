"""Group norm of channels-last feature pyramids with an activation, on the library's own kernels (C entry points
``dfa3d_group_norm_*``).

The attention reads its features as (B, N, C): the N rows of all levels, channels innermost (``value`` of the operator;
BEVFormer_DFA3D/projects/mmdet3d_plugin/bevformer/modules/transformer.py:368-391 flattens them so).  ``group_norm`` works on that
layout: every (image, level, group of channels) is normalised by itself, all levels in one launch, and the activation is applied
on the way out, so that projected features go to the attention without a transpose or a pass per level.

CUDA tensors of float32, bfloat16 or float16 with float32 weights; statistics are float32 and merged in a fixed order (the same
bits in every run).  Under autocast the input is cast to float32, as torch does for its norms.  There is no fallback path.
"""
import torch
import torch.nn as nn
from torch.autograd.function import Function, once_differentiable

from . import _lib
from .dropout_ops import keep, kept

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_ACTS = {None: _lib.ROW_NONE, "relu": _lib.ROW_RELU, "silu": _lib.ROW_SILU}


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _table(shapes, lsi, x):
    if (shapes is None) != (lsi is None):
        raise RuntimeError("spatial_shapes and level_start_index must be given together or not at all")
    if shapes is None:
        return None, None, 0, 1
    if shapes.dtype != torch.int64 or lsi.dtype != torch.int64 or shapes.dim() != 2 or shapes.shape[1] not in (2, 3) \
            or lsi.numel() != shapes.shape[0]:
        raise RuntimeError("spatial_shapes must be int64 (L, 2|3) and level_start_index int64 (L)")
    if shapes.device != x.device or lsi.device != x.device:
        raise RuntimeError("all tensors must be on one device")
    return shapes.contiguous(), lsi.contiguous(), shapes.shape[1], shapes.shape[0]


@_lib.native_apply("group_norm")
class GroupNormFunction(Function):
    @staticmethod
    @torch.amp.custom_fwd(device_type="cuda", cast_inputs=torch.float32)
    def forward(ctx, x, weight, bias, spatial_shapes, level_start_index, num_groups, eps, activation):
        """x (B, ..., C); weight, bias (C) or (L, C)."""
        if not x.is_cuda or x.dtype not in _DTYPES or x.dim() < 2:
            raise RuntimeError("x must be a float32, bfloat16 or float16 CUDA tensor (B, ..., C), got "
                               f"{tuple(x.shape)} {x.dtype} on {x.device}")
        if activation not in _ACTS:
            raise ValueError("activation must be None, 'relu' or 'silu'")
        shapes, lsi, stride, L = _table(spatial_shapes, level_start_index, x)
        C, G = x.shape[-1], int(num_groups)
        for t, n in ((weight, "weight"), (bias, "bias")):
            if t.dtype != torch.float32 or t.device != x.device or tuple(t.shape) not in ((C,), (L, C)) or t.shape != weight.shape:
                raise RuntimeError(f"{n} must be float32 ({C}) or ({L}, {C}) on {x.device}, got {tuple(t.shape)} {t.dtype} on "
                                   f"{t.device}")
        B, N, rows = x.shape[0], x[0].numel() // C if x.numel() else 0, 1 if weight.dim() == 1 else L
        size = _lib.size("dfa3d_group_norm_workspace", B, N, C, G, L, 0)      # refuses sizes before anything is copied
        x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
        y = torch.empty_like(x)
        stats = torch.empty((2, B, L, G), dtype=torch.float32, device=x.device)
        work = torch.empty(size, dtype=torch.uint8, device=x.device)
        with torch.cuda.device(x.device):
            _lib.call_plain("dfa3d_group_norm_forward", x.data_ptr(), _DTYPES[x.dtype], B, N, C, G, _ptr(shapes), stride, _ptr(lsi),
                            L, weight.data_ptr(), bias.data_ptr(), rows, float(eps), _ACTS[activation], y.data_ptr(),
                            stats[0].data_ptr(), stats[1].data_ptr(), work.data_ptr(), work.numel(), _stream(x))
        keep(ctx, x, weight, bias, shapes, lsi, stats)
        ctx.sizes, ctx.act = (B, N, C, G, stride, L, rows), _ACTS[activation]
        return y

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    @once_differentiable
    def backward(ctx, grad_y):
        x, weight, bias, shapes, lsi, stats = kept(ctx)
        B, N, C, G, stride, L, rows = ctx.sizes
        g = grad_y.to(x.dtype).contiguous()
        need = ctx.needs_input_grad
        grad_x = torch.empty_like(x) if need[0] else None
        grad_wb = None
        if need[1] or need[2]:
            grad_wb = [torch.empty_like(weight), torch.empty_like(weight)]
        work = torch.empty(_lib.size("dfa3d_group_norm_workspace", B, N, C, G, L, 1), dtype=torch.uint8, device=x.device)
        with torch.cuda.device(x.device):
            _lib.call_plain("dfa3d_group_norm_backward", g.data_ptr(), x.data_ptr(), _DTYPES[x.dtype], B, N, C, G, _ptr(shapes),
                            stride, _ptr(lsi), L, weight.data_ptr(), bias.data_ptr(), rows, ctx.act, stats[0].data_ptr(),
                            stats[1].data_ptr(), _ptr(grad_x), None if grad_wb is None else grad_wb[0].data_ptr(),
                            None if grad_wb is None else grad_wb[1].data_ptr(), work.data_ptr(), work.numel(), _stream(x))
        return (grad_x, grad_wb[0] if need[1] else None, grad_wb[1] if need[2] else None) + (None,) * 5


def group_norm(x, num_groups, weight, bias, eps=1e-5, activation=None, spatial_shapes=None, level_start_index=None):
    """act(GroupNorm(x)) of channels-last features x (B, ..., C), up to 1024 channels.

    With ``spatial_shapes`` (L, 2|3) and ``level_start_index`` (L), int64 on the device as the operator takes them, the N rows of an
    image are L levels, ascending, each normalised by itself; rows that belong to no level become 0.  Without them an image is
    one level (x.permute(0, 2, 3, 1) of a channels_last (B, C, H, W) tensor is read where it lies).  weight and bias (C), or
    (L, C) for weights of each level's own.  activation: None, "relu" or "silu"."""
    return GroupNormFunction.apply(x, weight, bias, spatial_shapes, level_start_index, num_groups, eps, activation)


class LevelGroupNorm(nn.GroupNorm):
    """``torch.nn.GroupNorm`` for channels-last features (B, ..., C) with an activation, over the levels of a feature pyramid.
    Parameters and state dict are GroupNorm's; with ``num_levels`` they are (num_levels, C), a norm of each level's own."""

    def __init__(self, num_groups, num_channels, eps=1e-5, activation=None, num_levels=None):
        if activation not in _ACTS:
            raise ValueError("activation must be None, 'relu' or 'silu'")
        super().__init__(num_groups, num_channels, eps=eps)
        self.activation, self.num_levels = activation, num_levels
        if num_levels is not None:
            self.weight = nn.Parameter(torch.ones(num_levels, num_channels))
            self.bias = nn.Parameter(torch.zeros(num_levels, num_channels))

    def forward(self, x, spatial_shapes=None, level_start_index=None):
        return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation, spatial_shapes, level_start_index)
