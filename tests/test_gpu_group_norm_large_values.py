"""Group norm of features whose square does not fit 32 bits, though what is normalised (their distance from the mean) does.

A part of the rows that is empty, a lane without rows or the first rows that a thread sees, has a mean of its own that counts for
nothing: its distance from the others' mean may not enter the sum of squares."""
import pytest
import torch

import row_reference as R
from test_gpu_group_norm import BOTH, DEV, EPS, apply, table

pytestmark = pytest.mark.gpu

# mean^2 > 3.4e38.  The spread leaves a group's sum of squares (`n` of them, at most 4200 here) inside of 32 bits, and is above the
# step of a bf16 number of that size (2^57 = 1.4e17).
MEAN, SPREAD = 3e19, 2e17
CASES = [
    (1, 3, 8, 2, None),                                  # most row lanes have no rows
    (2, 60, 32, 4, None),
    (1, 40, 15, 3, None),                                # words of one channel
    (2, 50, 30, 5, None),                                # of two
    (1, 300, 24, 12, [(3, 5), (1, 1), (15, 17)]),        # levels of a few rows: CTAs of a cluster without any
    (2, 1025, 256, 64, None),                            # tiles and their merge
    (1, 2000, 256, 128, [(3, 4), (1, 1), (40, 40), (1, 2)]),      # levels that one or two tiles have a piece of
]


@BOTH
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("sign", [1, -1], ids=["above", "below"])
@pytest.mark.parametrize("B,N,C,G,levels", CASES)
def test_features_whose_square_overflows(lib_built, B, N, C, G, levels, sign, dtype, native):
    gen = torch.Generator().manual_seed(N + C)
    x = ((sign * MEAN + SPREAD * torch.randn(B, N, C, generator=gen, dtype=torch.float64)).to(dtype)).to(DEV)
    w, b = ((1 + 0.3 * torch.randn(C, generator=gen)).to(DEV) for _ in range(2))
    g = torch.randn(B, N, C, generator=gen).to(dtype).to(DEV)
    shapes = lsi = None
    segments = [(0, N)]
    if levels:
        shapes, lsi = table(levels)
        ends = torch.tensor([h * v for h, v in levels]).cumsum(0).tolist()
        segments = list(zip([0] + ends[:-1], ends))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = apply(native, *leaves, G, None, shapes, lsi)
    gx, gw, gb = torch.autograd.grad(y, leaves, g)
    k = R.group_norm(x, w, b, G, EPS, None, segments, g)
    h = 0 if dtype == torch.float32 else R.half_step(dtype)
    R.assert_within("y", y, k["y"], k["tol_y"] + h * k["y"].abs() + R.tiny(dtype))
    R.assert_within("grad_x", gx, k["gx"], k["tol_gx"] + h * k["gx"].abs() + R.tiny(dtype))
    R.assert_within("grad_weight", gw, k["gw"], k["tol_w"])
    R.assert_within("grad_bias", gb, k["gb"], k["tol_b"])
    # what is compared is the normalisation: the bias alone would not do
    inside = torch.zeros(N, dtype=torch.bool)
    for lo, hi in segments:
        inside[lo:hi] = hi - lo > 2
    assert ((k["y"] - b.cpu().double()).abs() > k["tol_y"] + h * k["y"].abs())[:, inside].double().mean() > 0.8


@pytest.mark.parametrize("N", [50, 3000])
def test_a_spread_whose_square_overflows_leaves_the_bias(lib_built, N):
    """The variance does not fit 32 bits: 1 / sqrt of it is 0, and so is every gradient but the bias's."""
    gen = torch.Generator().manual_seed(1)
    x = (1e25 * torch.randn(2, N, 64, generator=gen)).to(DEV)
    w, b = (torch.randn(64, generator=gen).to(DEV) for _ in range(2))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = apply(True, *leaves, 8)
    assert torch.equal(y, b.expand_as(y))
    gx, gw, gb = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert not gx.any() and not gw.any() and torch.equal(gb, torch.full_like(gb, 2 * N))
