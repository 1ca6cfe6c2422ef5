"""Dropout without a stored mask: values and gradients against the definition in 64 bits, the mask's independence of everything but
(seed, site, element), refusals."""
import pytest
import torch

import row_reference as R
from test_gpu_native_path import _python

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = pytest.mark.parametrize("native", [True, False], ids=["native", "python"])


def seed_tensor(value):
    return torch.tensor([value], dtype=torch.int64, device=DEV)


def values(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def apply(native, x, p, seed, site=0, activation=None, residual=None):
    from dfa3d_b200.dropout_ops import DropoutFunction
    fn = DropoutFunction if native else _python(DropoutFunction)
    return fn.apply(x, residual, seed, p, site, activation)


def check(native, x, p, seed, site=0, activation=None, residual=None):
    """Forward and both gradients.  scale and the product are rounded once each, a residual's sum once, the result to its type."""
    leaves = [x.detach().clone().requires_grad_(True)]
    if residual is not None:
        leaves.append(residual.detach().clone().requires_grad_(True))
    y = apply(native, leaves[0], p, seed_tensor(seed), site, activation, leaves[1] if residual is not None else None)
    assert y.dtype == x.dtype and y.shape == x.shape
    want, slope = R.dropout(x, p, seed, site, activation, residual)
    kept_part = want if residual is None else (want - residual.cpu().double())
    h = 0 if x.dtype == torch.float32 else R.half_step(x.dtype)
    tol = 2 * R.U * kept_part.abs() + (R.U + h) * want.abs() + R.tiny(x.dtype)
    R.assert_within("y", y, want, tol)
    g = values(x.shape, x.dtype, 77)
    grads = torch.autograd.grad(y, leaves, g)
    want_g = g.cpu().double() * slope
    R.assert_within("grad_x", grads[0], want_g, (2 * R.U + h) * want_g.abs() + R.tiny(x.dtype))
    if residual is not None:
        assert torch.equal(grads[1], g)
    return y


@BOTH
@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 17, 1023, 2048, 4099, 70001])
def test_lengths(lib_built, n, dtype, native):
    check(native, values((n,), dtype, n), 0.3, 1234567 + n, site=2)


@BOTH
@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("activation", [None, "relu"])
@pytest.mark.parametrize("with_residual", [False, True], ids=["plain", "residual"])
@pytest.mark.parametrize("p", [0.0, 1e-12, 0.1, 0.5, 0.97, 1.0])
def test_rates_activation_residual(lib_built, p, with_residual, activation, dtype, native):
    x = values((37, 129), dtype, 5)
    x[3, :40] = 0.0
    check(native, x, p, -5, 7, activation, values((37, 129), dtype, 6) if with_residual else None)


@pytest.mark.parametrize("seed,site", [(0, 0), (-1, 1), (2 ** 63 - 1, 2 ** 31 - 1), (-2 ** 63, 40), (2 ** 32, 3)])
def test_seeds_and_sites(lib_built, seed, site):
    check(True, values((41, 100), torch.float32, 5), 0.4, seed, site)


@BOTH
@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_addresses_off_the_grid_and_strides(lib_built, offset, dtype, native):
    """The mask belongs to the element's number in row-major order, wherever the element lies."""
    base = values((30 * 31 + 4,), dtype, 5)
    whole = check(native, base[:930].clone().view(30, 31), 0.3, 9)
    moved = torch.empty(934, dtype=dtype, device=DEV)[offset:offset + 930].view(30, 31)
    moved.copy_(base[:930].view(30, 31))
    assert torch.equal(check(native, moved, 0.3, 9), whole)
    turned = base[:930].view(30, 31).t().contiguous().t()
    assert not turned.is_contiguous()
    assert torch.equal(apply(native, turned, 0.3, seed_tensor(9)), whole)
    res = values((31, 30), dtype, 6).t()
    assert torch.equal(apply(native, moved, 0.3, seed_tensor(9), residual=res),
                       apply(native, base[:930].view(30, 31), 0.3, seed_tensor(9), residual=res.contiguous()))


@pytest.mark.parametrize("shape", [(), (0,), (3, 0, 5), (2, 3, 4, 5, 6)])
def test_shapes(lib_built, shape):
    y = check(True, values(shape, torch.float32, 1), 0.5, 3)
    assert y.shape == shape


@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
def test_dropped_elements_are_zero_whatever_they_were(lib_built, dtype):
    x = values((64, 33), dtype, 1)
    bad = torch.tensor([float("nan"), float("inf"), float("-inf")])
    keep = R.kept((64, 33), 0.5, 11, 0)
    x.view(-1)[::7] = bad.repeat(400)[:x.view(-1)[::7].numel()].to(dtype).to(DEV)
    r = values((64, 33), dtype, 2)
    y, yr = apply(True, x, 0.5, seed_tensor(11)), apply(True, x, 0.5, seed_tensor(11), residual=r)
    assert (y.cpu()[~keep] == 0).all() and torch.equal(yr.cpu()[~keep], r.cpu()[~keep])
    assert torch.equal(torch.isnan(y.cpu()), keep & torch.isnan(x.cpu()))
    assert torch.equal(torch.isinf(y.cpu()), keep & torch.isinf(x.cpu()))
    # a gradient that is not finite stays where its element was kept
    xg = x.clone().requires_grad_(True)
    g = torch.full_like(x, float("inf"))
    gx, = torch.autograd.grad(apply(True, xg, 0.5, seed_tensor(11)), xg, g)
    assert torch.equal(torch.isinf(gx.cpu()), keep) and (gx.cpu()[~keep] == 0).all()


@pytest.mark.parametrize("with_residual", [False, True])
def test_a_nan_passes_the_relu_as_in_torch(lib_built, with_residual):
    x = values((40, 33), torch.float32, 1)
    x[::3, ::2] = float("nan")
    x.requires_grad_(True)
    keep = R.kept((40, 33), 0.5, 11, 0).to(DEV)
    y = apply(True, x, 0.5, seed_tensor(11), activation="relu", residual=torch.zeros_like(x) if with_residual else None)
    want = torch.where(keep, torch.relu(x) * 2, torch.zeros_like(x))
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(9.0), want.nan_to_num(9.0))
    g = torch.ones_like(x)
    assert torch.equal(torch.autograd.grad(y, x, g)[0], torch.autograd.grad(want, x, g)[0])


def test_smallest_values_keep_their_gradient(lib_built):
    """The backward of ReLU + dropout reads the result's sign: no positive element that is kept may have become 0."""
    x = torch.full((64,), torch.finfo(torch.float16).smallest_normal * torch.finfo(torch.float16).eps, device=DEV).half()
    for t in (x, torch.full((64,), 1e-45, device=DEV), torch.full((64,), 1e-40, device=DEV).bfloat16()):
        t.requires_grad_(True)
        assert (t > 0).all()
        y = apply(True, t, 0.01, seed_tensor(4), activation="relu")
        gx, = torch.autograd.grad(y, t, torch.ones_like(t))
        assert torch.equal(gx > 0, R.kept((64,), 0.01, 4, 0).to(DEV))


def test_keeps_the_fraction_and_no_two_sites_agree(lib_built):
    n, p = 4000000, 0.1
    x = torch.ones(n, device=DEV)
    masks = [apply(True, x, p, seed_tensor(s), site) > 0 for s, site in ((1, 0), (1, 1), (2, 0))]
    for m in masks:      # five standard deviations
        assert abs(float(m.float().mean()) - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
    q = p * p + (1 - p) ** 2
    for a, b in ((0, 1), (0, 2), (1, 2)):
        assert abs(float((masks[a] == masks[b]).float().mean()) - q) < 5 * (q * (1 - q) / n) ** 0.5


def test_elements_past_two_to_the_31(lib_built):
    n = (1 << 31) + 37
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    x.requires_grad_(True)
    y = apply(True, x, 0.5, seed_tensor(21), 3)
    gx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(gx, y)
    first = (n - 4000) // 4 * 4
    words = torch.from_numpy(_words_from(first, n, 21, 3) >= (1 << 31))
    assert torch.equal(y[first:].cpu() > 0, words)


def _words_from(first, last, seed, site):
    """Words first ... last - 1 (first a multiple of 4)."""
    import numpy as np
    m, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    block = np.arange(first // 4, (last + 3) // 4, dtype=np.uint64)
    c, k = [block & m, block >> s32, np.full_like(block, site), np.zeros_like(block)], [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(7):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s32) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> s32) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[:last - first]


@BOTH
def test_gradient_of_the_residual_alone_and_of_nothing(lib_built, native):
    x, r = values((8, 16), torch.float32, 1), values((8, 16), torch.float32, 2).requires_grad_(True)
    y = apply(native, x, 0.5, seed_tensor(1), residual=r)
    g = torch.ones_like(y)
    assert torch.equal(torch.autograd.grad(y, r, g)[0], g)
    with torch.no_grad():
        assert not apply(native, x.requires_grad_(True), 0.5, seed_tensor(1)).requires_grad


@BOTH
def test_one_tensor_as_both_summands(lib_built, native):
    x = values((8, 16), torch.float32, 1).requires_grad_(True)
    y = apply(native, x, 0.5, seed_tensor(1), residual=x)
    gx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(gx, 1 + 2 * R.kept((8, 16), 0.5, 1, 0).to(DEV).float())


@BOTH
def test_a_seed_that_changes_before_the_backward_is_noticed(lib_built, native):
    x, s = values((8, 16), torch.float32, 1).requires_grad_(True), seed_tensor(1)
    y = apply(native, x, 0.5, s)
    s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@BOTH
def test_no_second_derivative(lib_built, native):
    x = values((8, 16), torch.float32, 1).requires_grad_(True)
    g = torch.ones(8, 16, device=DEV, requires_grad=True)
    gx, = torch.autograd.grad(apply(native, x, 0.5, seed_tensor(1)), x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        gx.sum().backward()


def test_refusals(lib_built):
    from dfa3d_b200 import dropout
    x, s = torch.zeros(4, 8, device=DEV), seed_tensor(1)
    for bad in (torch.zeros(4, 8), x.double(), x.int()):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            dropout(bad, 0.5, s)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="between 0 and 1"):
            dropout(x, p, s)
    for site in (-1, 2 ** 31):
        with pytest.raises(ValueError, match="site"):
            dropout(x, 0.5, s, site)
    for bad in (None, s.cpu(), s.int(), torch.zeros(2, dtype=torch.int64, device=DEV)):
        with pytest.raises(RuntimeError, match="seed must be one int64"):
            dropout(x, 0.5, bad)
    with pytest.raises(ValueError, match="activation"):
        dropout(x, 0.5, s, activation="silu")
    for r in (x[:3], x.half(), x.cpu()):
        with pytest.raises(RuntimeError, match="residual"):
            dropout(x, 0.5, s, residual=r)
    assert torch.equal(dropout(x + 1, 0, None), x + 1)           # an integer rate, no seed needed


def test_another_stream(lib_built):
    x, s = values((500, 300), torch.float32, 1), seed_tensor(3)
    want = apply(True, x, 0.5, s)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = apply(True, x * 1, 0.5, s)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(got, want)


def test_captured_passes_draw_new_masks_and_keep_them_for_the_backward(lib_built):
    from dfa3d_b200 import draw_seed, dropout
    x = torch.ones(300, 100, device=DEV, requires_grad=True)

    def step():
        seed = draw_seed()
        y = dropout(x, 0.5, seed, activation="relu")
        z = dropout(x, 0.5, seed, 1, residual=y)
        return seed, y, z, torch.autograd.grad(z, x, torch.ones_like(z))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seed, y, z, g = step()
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        value = int(seed)
        a, b = R.kept((300, 100), 0.5, value, 0).to(DEV).float(), R.kept((300, 100), 0.5, value, 1).to(DEV).float()
        assert torch.equal(y, 2 * a) and torch.equal(z, 2 * a + 2 * b) and torch.equal(g, 2 * a + 2 * b)
        seen.append(value)
    assert len(set(seen)) == 3


def test_module_is_a_dropout(lib_built):
    from dfa3d_b200 import CounterDropout
    m = CounterDropout(0.25)
    assert isinstance(m, torch.nn.Dropout) and m.p == 0.25
    x = values((64, 64), torch.float32, 1)
    torch.manual_seed(5)
    a, b = m(x), m(x)
    torch.manual_seed(5)
    assert torch.equal(m(x), a) and not torch.equal(a, b)
    assert torch.equal(a[a != 0], (x * (4.0 / 3.0))[a != 0])
    m.eval()
    assert m(x) is x
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        CounterDropout(0.25)(x.cpu())
