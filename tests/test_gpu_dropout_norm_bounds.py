"""LayerNorm(residual + dropout(x)) against the definition with the bounds of its own summation (row_bounds): the statistics that it
keeps, results and gradients at these statistics; rows far from zero; enough rows that a lane group takes several, in every layout.

Lane groups of a launch: 296 CTAs of 8 warps with 32 / lanes groups each (444 CTAs for a forward on the grid), so that a second row is
taken above 9472 rows of 8 lanes, 4736 of 16, 2368 of 32 (14208, 7104, 3552)."""
import pytest
import torch

import row_bounds as Bo
import row_reference as R
from test_gpu_dropout_norm import DEV, EPS, apply, inputs, seed_tensor
from test_gpu_native_path import _python

pytestmark = pytest.mark.gpu
SEED, SITE = 41, 4


def check(tensors, g, p=0.2):
    from dfa3d_b200.dropout_ops import DropoutAddLayerNormFunction
    dtype = tensors[0].dtype
    rows, E = tensors[0].shape
    h = 0 if dtype == torch.float32 else R.half_step(dtype)
    leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
    y = _python(DropoutAddLayerNormFunction).apply(*leaves, seed_tensor(SEED), p, SITE, EPS)
    stats = y.grad_fn.saved_tensors[3].clone()
    got = dict(zip(("gx", "gr", "gw", "gb"), torch.autograd.grad(y, leaves, g)), y=y.detach())

    f = Bo.norm_forward(*tensors, p, SEED, SITE, EPS)
    mean, off, rstd, rho = Bo.norm_stats(f, EPS)
    R.assert_within("mean", stats[0], mean, off)
    R.assert_within("rstd", stats[1], rstd, rho * rstd)
    k = Bo.norm_given(f, stats, tensors[2], tensors[3], g, -(-rows // 2368))
    stored = lambda name: k[name][1] + h * k[name][0].abs() + R.tiny(dtype)
    for name in ("y", "gr", "gx"):
        R.assert_within(name, got[name], k[name][0], stored(name))
    for name in ("gw", "gb"):
        R.assert_within(name, got[name], *k[name])
    # a normalisation that was lost, and gradients that were, would not pass
    if E > 1:
        Bo.assert_refutes("y", tensors[3].cpu().double().expand(rows, E), k["y"][0], stored("y"))
        Bo.assert_refutes("gw", torch.zeros(E).double(), *k["gw"])
    if E > 2:      # two elements are normalised to -1 and 1 whatever they are: there is next to no gradient
        Bo.assert_refutes("gr", torch.zeros(rows, E).double(), k["gr"][0], stored("gr"))

    leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
    y = apply(True, *leaves, seed_tensor(SEED), p, SITE)
    native = dict(zip(("gx", "gr", "gw", "gb"), torch.autograd.grad(y, leaves, g)), y=y.detach())
    assert all(torch.equal(native[n], got[n]) for n in got)


@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("rows,E", [(7, 12), (50, 96), (120, 256), (65, 514), (40, 1024), (33, 1023)])
def test_statistics_and_results_at_them(lib_built, rows, E, dtype):
    check(*inputs(rows, E, dtype))


@pytest.mark.parametrize("spread,mean", [(1.0, 100.0), (1e-2, 10.0), (1e-3, 100.0), (1e3, -1e4)])
@pytest.mark.parametrize("rows,E", [(50, 256), (50, 203)])
def test_rows_far_from_zero(lib_built, rows, E, spread, mean):
    check(*inputs(rows, E, torch.float32, spread=spread, mean=mean))


# Off the grid: a row's words lie on 8 lanes (one each, two), 16 (two), 32 (two, four, six, nine).  The last turn is not full.
@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("rows,E", [(20011, 27), (20011, 53), (10007, 101), (5003, 203), (5003, 455), (5003, 701), (5003, 1021)])
def test_several_rows_a_lane_group_off_the_grid(lib_built, rows, E, dtype):
    check(*inputs(rows, E, dtype))


# Two and six elements beyond a multiple of four: a row begins at an even place of its word.
@pytest.mark.parametrize("rows,E", [(19001, 6), (5003, 202), (4999, 1022)])
def test_several_rows_that_begin_at_even_places(lib_built, rows, E):
    check(*inputs(rows, E, torch.float16))


@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("rows,E", [(29003, 32), (15001, 128), (15001, 256), (7411, 512), (7411, 1024)])
def test_several_rows_a_lane_group_on_the_grid(lib_built, rows, E, dtype):
    check(*inputs(rows, E, dtype))


@pytest.mark.parametrize("p", [0.1, 0.2])
@pytest.mark.parametrize("rows,E", [(300007, 2), (200003, 3), (150001, 4)])
def test_many_narrow_rows(lib_built, rows, E, p):
    """Among so many rows of two or three there are some where residual and dropped part cancel and some that have next to no spread: what
    the sum is off by is a rounding of its parts, times rstd.  1 / 0.9 is rounded too, 1 / 0.8 is not."""
    check(*inputs(rows, E, torch.float32), p=p)
