"""Gradients of a group norm where 1 / sqrt(var) squared does not fit 32 bits though the gradient does: eps = 0 and features that hardly
differ; and where it is next to nothing: features that differ a lot, small gradients."""
import pytest
import torch

import row_reference as R
from test_gpu_group_norm import BOTH, DEV, apply, table

pytestmark = pytest.mark.gpu


@BOTH
@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("spread,size", [(1e-18, 1e4), (2e-18, 1e3), (1e-16, 1e6), (1e-17, 1e-3), (1e15, 1e-12), (1e12, 1e-20)])
@pytest.mark.parametrize("B,N,C,G,levels", [(2, 60, 32, 4, None), (1, 40, 15, 3, None), (2, 1100, 64, 16, [(30, 30), (10, 20)]),
                                            (1, 70, 24, 6, [(5, 10), (4, 5)])])
def test_gradients_at_the_ends_of_the_range(lib_built, B, N, C, G, levels, spread, size, activation, native):
    """spread^2 of the smallest is 1e-36, a normal number; its inverse times a mean of d * xhat of 1e4 is 1e40."""
    gen = torch.Generator().manual_seed(N + C)
    x = (spread * torch.randn(B, N, C, generator=gen)).to(DEV)
    w, b = (1 + 0.3 * torch.randn(C, generator=gen)).to(DEV), (0.5 * torch.randn(C, generator=gen)).to(DEV)
    # a gradient with a part along the normalised features: its mean of d * xhat is about `size`
    hat = x / spread
    g = (size * (hat + torch.randn(B, N, C, generator=gen).to(DEV))).contiguous()
    shapes = lsi = None
    segments = [(0, N)]
    if levels:
        shapes, lsi = table(levels)
        ends = torch.tensor([h * v for h, v in levels]).cumsum(0).tolist()
        segments = list(zip([0] + ends[:-1], ends))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = apply(native, *leaves, G, activation, shapes, lsi, eps=0.0)
    gx, gw, gb = torch.autograd.grad(y, leaves, g)
    k = R.group_norm(x, w, b, G, 0.0, activation, segments, g)
    R.assert_within("y", y, k["y"], k["tol_y"] + R.tiny(torch.float32))
    R.assert_within("grad_x", gx, k["gx"], k["tol_gx"] + R.tiny(torch.float32))
    R.assert_within("grad_weight", gw, k["gw"], k["tol_w"] + R.tiny(torch.float32))
    R.assert_within("grad_bias", gb, k["gb"], k["tol_b"] + R.tiny(torch.float32))
    inside = torch.zeros(N, dtype=torch.bool)
    for lo, hi in segments:
        inside[lo:hi] = True
    assert (k["gx"].abs() > k["tol_gx"])[:, inside].double().mean() > 0.9
