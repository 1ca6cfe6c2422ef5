"""Activations kept in 8 bits until the backward, on the library's own kernels (C entry points ``dfa3d_compress8``,
``dfa3d_decompress8``).

Blocks of 32 neighbours of a row share one power of two, the smallest for which no element is beyond the format's largest number
(127 of "int8", 448 of "e4m3"); an element is x / 2^e rounded to nearest even.  33 bytes for 32 elements, half of a 16-bit tensor and
a quarter of a 32-bit one.  int8 is off by at most half a step of its block, e4m3 by 2^-4 of an element: int8 is nearer for rows
without outliers, e4m3 where a block spans orders of magnitude.  Because the factor is a power of two, what a code stands for is a
number of bfloat16 and float16 too, and the products of a backward read it without another rounding.  A block that holds an infinity
or NaN comes back as NaN.

``feed_forward_ops`` keeps inputs this way (``checkpoint=``); the functions here are for a program's own Functions.  They are storage,
not operations of the graph: no gradient passes.
"""
from typing import NamedTuple

import torch

from . import _lib

FORMATS = {"int8": _lib.FORMAT_INT8, "e4m3": _lib.FORMAT_E4M3}
_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


class Compressed8(NamedTuple):
    """A tensor in 8 bits: codes (rows, cols) and scales (rows, ceil(cols / 32)), both uint8, and what it was."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype
    format: str


def check_format(format, name="format"):
    if format not in FORMATS:
        raise ValueError(f"{name} must be one of {sorted(FORMATS)}, got {format!r}")


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def compress8(x, format="int8"):
    """x (..., cols), float32, bfloat16 or float16 on a CUDA device, in 8 bits."""
    check_format(format)
    got = _lib.native().compress8(x, format)
    if got is not NotImplemented:
        return Compressed8(*got, x.shape, x.dtype, format)
    if not x.is_cuda or x.dtype not in _DTYPES:
        raise RuntimeError(f"x must be a float32, bfloat16 or float16 CUDA tensor, got {x.dtype} on {x.device}")
    if x.dim() == 0:
        raise RuntimeError("x must have at least one dimension")
    x = x.detach().contiguous()
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    codes = torch.empty((rows, cols), dtype=torch.uint8, device=x.device)
    scales = torch.empty((rows, (cols + 31) // 32), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _lib.call_plain("dfa3d_compress8", x.data_ptr(), _DTYPES[x.dtype], rows, cols, FORMATS[format], codes.data_ptr(),
                        scales.data_ptr(), _stream(x))
    return Compressed8(codes, scales, x.shape, x.dtype, format)


def check_compressed(c):
    """Refuses what the kernels would read out of range."""
    check_format(c.format)
    cols = c.shape[-1] if len(c.shape) else 0
    rows = c.shape.numel() // cols if cols else 0
    for t, n, name in ((c.codes, cols, "codes"), (c.scales, (cols + 31) // 32, "scales")):
        if t.dtype != torch.uint8 or not t.is_cuda or t.device != c.codes.device or t.numel() != rows * n:
            raise RuntimeError(f"{name} must be {rows} x {n} uint8 on one CUDA device, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if c.dtype not in _DTYPES:
        raise RuntimeError(f"dtype must be float32, bfloat16 or float16, got {c.dtype}")
    return rows, cols


def decompress8(c):
    """What a ``compress8`` stands for, of the shape and type that it was given."""
    got = _lib.native().decompress8(*c)
    if got is not NotImplemented:
        return got
    rows, cols = check_compressed(c)
    out = torch.empty(c.shape, dtype=c.dtype, device=c.codes.device)
    into(c, out, cols)
    return out


def into(c, out, pitch):
    """The same into rows that are `pitch` elements apart."""
    rows, cols = check_compressed(c)
    codes, scales = c.codes.contiguous(), c.scales.contiguous()
    with torch.cuda.device(codes.device):
        _lib.call_plain("dfa3d_decompress8", codes.data_ptr(), scales.data_ptr(), FORMATS[c.format], rows, cols, _DTYPES[c.dtype],
                        out.data_ptr(), pitch, _stream(codes))
