"""LayerNorm(residual + dropout(x)): values and gradients against the definition in 64 bits and against differences, refusals."""
import pytest
import torch

import row_reference as R
from test_gpu_native_path import _python

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-5
BOTH = pytest.mark.parametrize("native", [True, False], ids=["native", "python"])


def seed_tensor(value):
    return torch.tensor([value], dtype=torch.int64, device=DEV)


def inputs(rows, E, dtype, seed=0, spread=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed + rows + E)
    x, r = (torch.randn(rows, E, generator=g) * spread).to(dtype), (torch.randn(rows, E, generator=g) * spread + mean).to(dtype)
    w, b = 1 + 0.3 * torch.randn(E, generator=g), torch.randn(E, generator=g)
    return [t.to(DEV) for t in (x, r, w, b)], torch.randn(rows, E, generator=g).to(dtype).to(DEV)


def apply(native, x, r, w, b, seed, p, site=0, eps=EPS):
    from dfa3d_b200.dropout_ops import DropoutAddLayerNormFunction
    fn = DropoutAddLayerNormFunction if native else _python(DropoutAddLayerNormFunction)
    return fn.apply(x, r, w, b, seed, p, site, eps)


def check(native, tensors, g, p, seed, site=0):
    leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
    y = apply(native, *leaves, seed_tensor(seed), p, site)
    dtype = tensors[0].dtype
    assert y.dtype == dtype and y.shape == tensors[0].shape
    f = R.norm_forward(*tensors, p, seed, site, EPS)
    h = 0 if dtype == torch.float32 else R.half_step(dtype)
    tol = f["w"].abs() * R.hat_error(f) + (4 * R.U + h) * f["y"].abs() + 4 * R.U * tensors[3].cpu().double().abs() + R.tiny(dtype)
    R.assert_within("y", y, f["y"], tol)
    gx, gr, gw, gb = torch.autograd.grad(y, leaves, g)
    k = R.norm_backward(f, g)
    R.assert_within("grad_residual", gr, k["gr"], k["tol"] + h * k["gr"].abs() + R.tiny(dtype))
    R.assert_within("grad_x", gx, k["gx"], k["tol"] * f["slope"] + (h + 2 * R.U) * k["gx"].abs() + R.tiny(dtype))
    R.assert_within("grad_weight", gw, k["gw"], k["tol_w"])
    R.assert_within("grad_bias", gb, k["gb"], k["tol_b"])
    assert gw.dtype == gb.dtype == torch.float32
    return [y, gx, gr, gw, gb]


@BOTH
@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("rows,E", [(1, 1), (1, 256), (3, 4), (2, 8), (5, 7), (9, 30), (17, 64), (33, 127), (20, 128), (50, 132),
                                    (77, 200), (1000, 256), (301, 257), (100, 384), (65, 514), (130, 640), (64, 1000), (40, 1023),
                                    (40, 1024)])
def test_matches_definition(lib_built, rows, E, dtype, native):
    tensors, g = inputs(rows, E, dtype)
    check(native, tensors, g, 0.2, 31 + rows, 4)


@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("p", [0.0, 1e-12, 0.5, 0.95, 1.0])
def test_rates(lib_built, p, dtype):
    tensors, g = inputs(120, 96, dtype)
    check(True, tensors, g, p, -7)


@pytest.mark.parametrize("rows,E", [(5003, 256), (20011, 64), (2500, 1024)])
def test_many_rows(lib_built, rows, E):
    tensors, g = inputs(rows, E, torch.float32)
    got = check(True, tensors, g, 0.1, 3)
    again = check(True, tensors, g, 0.1, 3)
    assert all(torch.equal(a, b) for a, b in zip(got, again))          # sums over rows too


@pytest.mark.parametrize("spread,mean", [(1e-3, 100.0), (1e3, 0.0), (1e-6, 0.0)])
def test_rows_far_from_zero_and_tiny_ones(lib_built, spread, mean):
    tensors, g = inputs(50, 256, torch.float32, spread=spread, mean=mean)
    check(True, tensors, g, 0.1, 3)


def test_constant_rows(lib_built):
    """No spread at all: the result is the bias, gradients are finite."""
    x, r = torch.zeros(6, 64, device=DEV), torch.full((6, 64), 3.0, device=DEV)
    (_, _, w, b), g = inputs(6, 64, torch.float32)
    check(True, [x, r, w, b], g, 0.5, 1)


@BOTH
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("E", [30, 64])
def test_addresses_off_the_grid_and_strides(lib_built, E, dtype, native):
    tensors, g = inputs(40, E, dtype)
    want = check(native, tensors, g, 0.3, 9)
    moved = [torch.empty(t.numel() + 3, dtype=t.dtype, device=DEV)[1:1 + t.numel()].view(t.shape).copy_(t) for t in tensors]
    assert moved[0].data_ptr() % 8 != 0
    got = check(native, moved, g, 0.3, 9)
    assert torch.equal(got[0], want[0])
    turned = [t.t().contiguous().t() if t.dim() == 2 else t for t in tensors]
    assert torch.equal(apply(native, *turned, seed_tensor(9), 0.3), want[0])


@BOTH
def test_more_dimensions_and_no_rows(lib_built, native):
    tensors, g = inputs(24, 32, torch.float32)
    want = apply(native, *tensors, seed_tensor(2), 0.5)
    x, r, w, b = tensors
    assert torch.equal(apply(native, x.view(2, 3, 4, 32), r.view(2, 3, 4, 32), w, b, seed_tensor(2), 0.5).view(24, 32), want)
    assert torch.equal(apply(native, x[0], r[0], w, b, seed_tensor(2), 0.5), want[0])
    leaves = [t.clone().requires_grad_(True) for t in (x[:0], r[:0], w, b)]
    y = apply(native, *leaves, seed_tensor(2), 0.5)
    assert y.shape == (0, 32)
    gw, gb = torch.autograd.grad(y, leaves[2:], y.detach())
    assert not gw.any() and not gb.any()


@BOTH
@pytest.mark.parametrize("needed", [(0,), (1,), (2,), (3,), (0, 3), (1, 2)])
def test_some_gradients_only(lib_built, needed, native):
    tensors, g = inputs(40, 64, torch.float32)
    full = [t.clone().requires_grad_(True) for t in tensors]
    want = torch.autograd.grad(apply(native, *full, seed_tensor(1), 0.5), full, g)
    part = [t.clone().requires_grad_(i in needed) for i, t in enumerate(tensors)]
    got = torch.autograd.grad(apply(native, *part, seed_tensor(1), 0.5), [part[i] for i in needed], g)
    assert all(torch.equal(a, want[i]) for a, i in zip(got, needed))


def test_without_gradients_the_result_is_the_same(lib_built):
    tensors, _ = inputs(40, 64, torch.float32)
    with torch.no_grad():
        a = apply(True, *tensors, seed_tensor(1), 0.5)
    assert torch.equal(a, apply(True, *[t.clone().requires_grad_(True) for t in tensors], seed_tensor(1), 0.5))


def test_gradient_against_differences(lib_built):
    """(f(t + hv) - f(t - hv)) / 2h of the kernel's own forward against its gradient: what the difference misses of the slope is
    computed in 64 bits, what its two results are rounded by is 2 U |y| and the normalisation's error each, over 2h."""
    tensors, g = inputs(30, 64, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    grads = torch.autograd.grad(apply(True, *leaves, seed_tensor(5), 0.25), leaves, g)
    gen = torch.Generator().manual_seed(1)
    h, g64 = 2.0 ** -6, g.cpu().double()
    for i, t in enumerate(tensors):
        v = torch.randint(0, 2, t.shape, generator=gen).double() * 2 - 1
        up, down = ([u if j != i else u + s * h * v.float().to(DEV) for j, u in enumerate(tensors)] for s in (1, -1))
        # t + hv is rounded: the step that was taken is what counts, the same for both sides of the comparison
        got = [(apply(True, *a, seed_tensor(5), 0.25).cpu().double() * g64).sum() for a in (up, down)]
        f = [R.norm_forward(*a, 0.25, 5, 0, EPS) for a in (up, down)]
        exact = [(k["y"] * g64).sum() for k in f]
        rounding = sum(((k["w"].abs() * R.hat_error(k) + 6 * R.U * k["y"].abs()) * g64.abs()).sum() for k in f)
        slope = (grads[i].cpu().double() * v).sum()
        missed = abs((exact[0] - exact[1]) / (2 * h) - (_exact_gradient(tensors, g, i) * v).sum())
        k = R.norm_backward(R.norm_forward(*tensors, 0.25, 5, 0, EPS), g)
        own = [(k["tol"] * 1.34).sum(), k["tol"].sum(), k["tol_w"].sum(), k["tol_b"].sum()][i]
        assert abs((got[0] - got[1]) / (2 * h) - slope) <= rounding / (2 * h) + missed + own


def _exact_gradient(tensors, g, i):
    leaves = [t.cpu().double().requires_grad_(True) for t in tensors]
    x, r, w, b = leaves
    keep = R.kept(x.shape, 0.25, 5, 0).double() / 0.75
    y = torch.nn.functional.layer_norm(r + x * keep, (x.shape[-1],), w, b, EPS)
    return torch.autograd.grad(y, leaves[i], g.cpu().double())[0]


def test_the_mask_is_that_of_dropout(lib_built):
    from dfa3d_b200 import dropout, dropout_add_layer_norm
    from dfa3d_b200.layer_ops import AddLayerNormFunction
    for E in (64, 37):
        (x, r, w, b), _ = inputs(50, E, torch.float32)
        got = dropout_add_layer_norm(x, r, w, b, 0.3, seed_tensor(8), 6)
        summed = dropout(x, 0.3, seed_tensor(8), 6, residual=r)
        want = torch.nn.functional.layer_norm(summed.double(), (E,), w.double(), b.double(), EPS)
        R.assert_within("y", got, want.cpu(), 1e-5)
        if E % 4 == 0:
            R.assert_within("existing norm", AddLayerNormFunction.apply(summed, None, w, b, EPS), want.cpu(), 1e-5)


@BOTH
def test_autocast_computes_in_float32(lib_built, native):
    tensors, g = inputs(40, 64, torch.float16)
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    with torch.autocast("cuda", dtype=torch.float16):
        y = apply(native, *leaves, seed_tensor(2), 0.5)
    assert y.dtype == torch.float32
    want = apply(native, *[t.float() for t in tensors], seed_tensor(2), 0.5)
    assert torch.equal(y, want)
    grads = torch.autograd.grad(y, leaves, g.float())
    assert [t.dtype for t in grads] == [torch.float16, torch.float16, torch.float32, torch.float32]


def test_refusals(lib_built):
    from dfa3d_b200 import dropout_add_layer_norm as f
    (x, r, w, b), _ = inputs(4, 8, torch.float32)
    s = seed_tensor(1)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        f(x.cpu(), r.cpu(), w.cpu(), b.cpu(), 0.5, s)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        f(x.double(), r.double(), w, b, 0.5, s)
    with pytest.raises(RuntimeError, match="residual"):
        f(x, r.half(), w, b, 0.5, s)
    with pytest.raises(RuntimeError, match="residual"):
        f(x, r[:3], w, b, 0.5, s)
    with pytest.raises(RuntimeError, match="weight must be"):
        f(x, r, w[:4], b, 0.5, s)
    with pytest.raises(RuntimeError, match="bias must be"):
        f(x, r, w, b.half(), 0.5, s)
    with pytest.raises(RuntimeError, match="up to 1024"):
        f(*(torch.zeros(2, 1028, device=DEV),) * 2, *(torch.zeros(1028, device=DEV),) * 2, 0.5, s)
    with pytest.raises(RuntimeError, match="E must be positive"):
        f(x[:, :0], r[:, :0], w[:0], b[:0], 0.5, s)
    with pytest.raises(RuntimeError, match="eps must be"):
        f(x, r, w, b, 0.5, s, eps=-1.0)
    with pytest.raises(ValueError, match="between 0 and 1"):
        f(x, r, w, b, 2.0, s)
    with pytest.raises(RuntimeError, match="seed must be"):
        f(x, r, w, b, 0.5, None)


def test_captured_forward_and_backward(lib_built):
    from dfa3d_b200 import draw_seed, dropout_add_layer_norm
    tensors, g = inputs(500, 128, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in tensors]

    def step():
        seed = draw_seed()
        y = dropout_add_layer_norm(*leaves, 0.5, seed)
        return (seed, y) + torch.autograd.grad(y, leaves, g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        eager = [t.clone().requires_grad_(True) for t in tensors]
        y = dropout_add_layer_norm(*eager, 0.5, out[0].clone())
        for a, b in zip(out[1:], (y,) + torch.autograd.grad(y, eager, g)):
            assert torch.equal(a, b)


def test_rows_past_two_to_the_31_elements(lib_built):
    """The last rows of a tensor that long have the mask of their own element numbers and are normalised like any others."""
    E, rows = 256, (1 << 23) + 11
    last = 40
    g = torch.Generator(device=DEV).manual_seed(3)
    x, r, go = (torch.empty(rows, E, dtype=torch.bfloat16, device=DEV).normal_(generator=g) for _ in range(3))
    w, b = torch.rand(E, device=DEV) + 0.5, torch.randn(E, device=DEV)
    leaves = [x.requires_grad_(True), r.requires_grad_(True)]
    y = apply(True, x, r, w, b, seed_tensor(5), 0.5, 9)
    gx, gr = torch.autograd.grad(y, leaves, go)
    first = (rows - last) * E
    keep = torch.from_numpy(_words(first, rows * E, 5, 9) >= (1 << 31)).view(last, E)
    xs, rs, gs = (t.detach()[-last:].cpu().double() for t in (x, r, go))
    s = rs + torch.where(keep, xs * 2, torch.zeros_like(xs))
    mean, var = s.mean(-1, keepdim=True), s.var(-1, keepdim=True, correction=0)
    rstd = (var + EPS) ** -0.5
    hat = (s - mean) * rstd
    d = gs * w.cpu().double()
    want = rstd * (d - d.mean(-1, keepdim=True) - hat * (d * hat).mean(-1, keepdim=True))
    step = R.half_step(torch.bfloat16)
    R.assert_within("y", y[-last:], hat * w.cpu().double() + b.cpu().double(), (step + 1e-5) * 8 * torch.ones(last, E).double())
    R.assert_within("grad_residual", gr[-last:], want, (step + 1e-4) * want.abs() + 1e-4)
    R.assert_within("grad_x", gx[-last:], torch.where(keep, want * 2, torch.zeros_like(want)), (step + 1e-4) * 2 * want.abs() + 2e-4)
    assert not gx[-last:].cpu()[~keep].any()


@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("rows,E", [(9, 2), (9, 3), (40, 5), (33, 250), (33, 253), (33, 254), (33, 255), (18, 509), (18, 510), (18, 511),
                                    (11, 1021), (11, 1022), (5003, 6), (2500, 61)])
def test_rows_that_begin_inside_of_a_word(lib_built, rows, E, dtype):
    tensors, g = inputs(rows, E, dtype)
    check(True, tensors, g, 0.2, 7, 4)


@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("E", [5, 30, 202, 255, 511, 1022])
def test_rows_without_numbers_spoil_no_neighbour(lib_built, E, dtype):
    tensors, g = inputs(30, E, dtype)
    results = []
    for spoiled in (False, True):
        x, r, w, b = [t.clone() for t in tensors]
        go = g.clone()
        if spoiled:
            x[1::2], r[1::2], go[1::2] = float("nan"), float("inf"), float("nan")
        leaves = [x.requires_grad_(True), r.requires_grad_(True)]
        y = apply(True, x, r, w, b, seed_tensor(3), 0.3, 2)
        results.append([t[::2] for t in (y.detach(), *torch.autograd.grad(y, leaves, go))])
    for a, c in zip(*results):
        assert torch.equal(a, c)


def _words(first, last, seed, site):
    from test_gpu_dropout import _words_from
    return _words_from(first, last, seed, site)
