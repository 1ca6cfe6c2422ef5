"""Group norm against the definition with the bounds of its own summation (row_bounds): the statistics that it keeps, results and
gradients at these statistics; long images, whose tiles have many rows, and features far from zero."""
import pytest
import torch

import row_bounds as Bo
import row_reference as R
from test_gpu_group_norm import DEV, EPS, apply, inputs, table
from test_gpu_native_path import _python

pytestmark = pytest.mark.gpu


def check(tensors, g, G, activation=None, levels=None):
    from dfa3d_b200.group_norm_ops import GroupNormFunction
    x, w, b = tensors
    dtype, N = x.dtype, x.shape[1]
    h = 0 if dtype == torch.float32 else R.half_step(dtype)
    shapes = lsi = None
    segments = [(0, N)]
    if levels:
        shapes, lsi = table(levels)
        ends = torch.tensor([r * c for r, c in levels]).cumsum(0).tolist()
        segments = list(zip([0] + ends[:-1], ends))
    leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
    y = _python(GroupNormFunction).apply(*leaves, shapes, lsi, G, EPS, activation)
    stats = y.grad_fn.saved_tensors[5].clone()
    got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, g)), y=y.detach())

    mean, off, rstd, rho = Bo.group_stats(x, G, EPS, segments)
    R.assert_within("mean", stats[0], mean, off)
    R.assert_within("rstd", stats[1], rstd, rho * rstd)
    k = Bo.group_given(x, w, b, G, activation, segments, stats, g)
    stored = lambda name: k[name][1] + h * k[name][0].abs() + R.tiny(dtype)
    for name in ("y", "gx"):
        R.assert_within(name, got[name], k[name][0], stored(name))
    for name in ("gw", "gb"):
        R.assert_within(name, got[name], *k[name])
    # a normalisation that was lost, and gradients that were, would not pass
    lost = torch.nn.functional.silu(k["norm"]) if activation else k["norm"]
    Bo.assert_refutes("y", lost, k["y"][0], stored("y"))
    Bo.assert_refutes("gx", torch.zeros_like(k["gx"][0]), k["gx"][0], stored("gx"))
    Bo.assert_refutes("gw", torch.zeros_like(k["gw"][0]), *k["gw"])
    Bo.assert_refutes("gb", torch.zeros_like(k["gb"][0]), *k["gb"])

    leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
    y = apply(True, *leaves, G, activation, shapes, lsi)
    native = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, g)), y=y.detach())
    assert all(torch.equal(native[n], got[n]) for n in got)


@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("B,N,C,G", [(2, 77, 96, 32), (1, 100, 90, 6), (2, 375, 256, 32), (3, 64, 513, 27), (1, 1500, 256, 32),
                                     (2, 3001, 90, 9), (1, 2000, 45, 5)])
def test_statistics_and_results_at_them(lib_built, B, N, C, G, activation, dtype):
    tensors, g = inputs(B, N, C, dtype)
    check(tensors, g, G, activation)


@pytest.mark.parametrize("levels,B,C,G", [([(30, 40), (15, 20), (8, 10)], 6, 64, 8), ([(60, 100), (30, 50)], 2, 256, 32)])
def test_levels_with_weights_of_their_own(lib_built, levels, B, C, G):
    N = sum(h * w for h, w in levels)
    tensors, g = inputs(B, N, C, torch.float32, len(levels))
    check(tensors, g, G, "silu", levels)


@pytest.mark.parametrize("spread,mean", [(1.0, 1000.0), (1e-3, 0.0), (1e4, 0.0), (1e-2, -50.0)])
@pytest.mark.parametrize("B,N", [(2, 700), (2, 4000)])
def test_features_far_from_zero(lib_built, B, N, spread, mean):
    tensors, g = inputs(B, N, 64, torch.float32, spread=spread, mean=mean)
    check(tensors, g, 8)


@pytest.mark.parametrize("B,N,C,G", [(6, 5000, 256, 32), (2, 70000, 256, 32), (1, 90000, 200, 25), (1, 150000, 96, 3), (200, 1100, 64, 8)])
def test_long_images_and_many_of_them(lib_built, B, N, C, G):
    tensors, g = inputs(B, N, C, torch.float32)
    check(tensors, g, G)
