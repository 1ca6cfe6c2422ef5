"""Group norm of channels-last feature pyramids: values and gradients against the definition in 64 bits and against differences, level
tables of every kind, refusals."""
import pytest
import torch

import row_reference as R
from test_gpu_native_path import _python

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-5
BOTH = pytest.mark.parametrize("native", [True, False], ids=["native", "python"])


def table(levels, start=None, third=None):
    shapes = torch.tensor([list(l) + ([third] if third else []) for l in levels], dtype=torch.int64)
    if start is None:
        hw = shapes[:, 0] * shapes[:, 1]
        start = torch.cat([hw.new_zeros(1), hw.cumsum(0)[:-1]])
    return shapes.to(DEV), torch.as_tensor(start, dtype=torch.int64).to(DEV)


def inputs(B, N, C, dtype, rows=None, spread=1.0, mean=0.0, seed=0):
    g = torch.Generator().manual_seed(seed + N + C)
    x = (torch.randn(B, N, C, generator=g) * (0.5 + torch.rand(C, generator=g)) * spread + torch.randn(C, generator=g) * spread
         + mean).to(dtype)
    size = (C,) if rows is None else (rows, C)
    w, b = 1 + 0.3 * torch.randn(size, generator=g), 0.5 * torch.randn(size, generator=g)
    return [t.to(DEV) for t in (x, w, b)], torch.randn(B, N, C, generator=g).to(dtype).to(DEV)


def apply(native, x, w, b, G, activation=None, shapes=None, lsi=None, eps=EPS):
    from dfa3d_b200.group_norm_ops import GroupNormFunction
    fn = GroupNormFunction if native else _python(GroupNormFunction)
    return fn.apply(x, w, b, shapes, lsi, G, eps, activation)


def check(native, tensors, g, G, activation=None, shapes=None, lsi=None, segments=None):
    """Compares y and the gradients; a ReLU's gradient is left out where z is within its own error of the border."""
    x = tensors[0]
    leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
    y = apply(native, *leaves, G, activation, shapes, lsi)
    assert y.dtype == x.dtype and y.shape == x.shape
    segments = [(0, x.shape[1])] if segments is None else segments
    k = R.group_norm(*tensors, G, EPS, activation, segments, g)
    h = 0 if x.dtype == torch.float32 else R.half_step(x.dtype)
    R.assert_within("y", y, k["y"], k["tol_y"] + h * k["y"].abs() + R.tiny(x.dtype))
    gx, gw, gb = torch.autograd.grad(y, leaves, g)
    if activation == "relu":
        z = R.group_norm(*tensors, G, EPS, None, segments)
        assert (z["y"].abs() > z["tol_y"])[z["tol_y"] > 0].all(), "the test's inputs have an element on the ReLU's border"
    R.assert_within("grad_x", gx, k["gx"], k["tol_gx"] + h * k["gx"].abs() + R.tiny(x.dtype))
    R.assert_within("grad_weight", gw, k["gw"], k["tol_w"])
    R.assert_within("grad_bias", gb, k["gb"], k["tol_b"])
    return [y, gx, gw, gb]


SIZES = [(1, 1, 4, 2), (2, 1, 8, 1), (1, 2, 1, 1), (3, 5, 7, 7), (2, 33, 6, 3), (1, 50, 30, 2), (2, 77, 96, 32), (1, 100, 90, 6),
         (2, 375, 256, 32), (1, 920, 256, 32), (3, 64, 513, 27), (1, 40, 1024, 1), (2, 31, 1023, 3), (1, 300, 1000, 8), (5, 9, 20, 5)]


@BOTH
@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("B,N,C,G", SIZES)
def test_one_level(lib_built, B, N, C, G, dtype, native):
    tensors, g = inputs(B, N, C, dtype)
    check(native, tensors, g, G)


@BOTH
@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("own_weights", [False, True], ids=["shared", "own"])
@pytest.mark.parametrize("B,levels,C,G", [(2, [(11, 13), (6, 7), (3, 4), (1, 1)], 64, 8), (1, [(1, 1), (20, 31)], 30, 3),
                                          (3, [(40, 50), (20, 25)], 256, 32), (7, [(2, 2), (1, 2), (1, 1)], 36, 4)])
def test_levels(lib_built, B, levels, C, G, own_weights, activation, dtype, native):
    N = sum(h * w for h, w in levels)
    shapes, lsi = table(levels, third=9 if C == 30 else None)
    tensors, g = inputs(B, N, C, dtype, len(levels) if own_weights else None)
    ends = torch.tensor([h * w for h, w in levels]).cumsum(0).tolist()
    check(native, tensors, g, G, activation, shapes, lsi, list(zip([0] + ends[:-1], ends)))


@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("B,N,C,G,seed", [(2, 60, 32, 4, 0), (1, 111, 15, 3, 0)])
def test_relu(lib_built, B, N, C, G, seed, dtype):
    tensors, g = inputs(B, N, C, dtype, seed=seed)
    got = check(True, tensors, g, G, "relu")
    assert (got[0] == 0).any() and (got[0] >= 0).all()


def test_relu_lets_a_nan_pass_as_torch_does(lib_built):
    (x, w, b), g = inputs(2, 40, 16, torch.float32)
    x[0, 3, 5] = float("nan")                       # its group of its image, and nothing else
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = apply(True, *leaves, 4, "relu")
    bad = torch.zeros(2, 40, 16, dtype=torch.bool)
    bad[0, :, 4:8] = True
    assert torch.equal(y.isnan().cpu(), bad)
    gx, = torch.autograd.grad(y, leaves[0], g)
    assert torch.equal(gx.isnan().cpu(), bad)


@pytest.mark.parametrize("spread,mean", [(1.0, 1000.0), (1e-3, 0.0), (1e4, 0.0), (1e-2, -50.0)])
def test_features_far_from_zero(lib_built, spread, mean):
    """Statistics are kept around their own mean: the error is that of the inputs' rounding, not of a difference of squares."""
    tensors, g = inputs(2, 700, 64, torch.float32, spread=spread, mean=mean)
    check(True, tensors, g, 8)


def test_rows_that_stand_out_at_the_beginning(lib_built):
    """Zero padding before features far from zero: no row may serve as the others' origin."""
    tensors, g = inputs(1, 4000, 32, torch.float32, mean=300.0)
    tensors[0][:, :40] = 0
    check(True, tensors, g, 4)


def test_constant_features(lib_built):
    tensors, g = inputs(2, 90, 16, torch.float32)
    tensors[0][:] = 7.0
    y, gx, gw, gb = check(True, tensors, g, 4)
    assert torch.equal(y, tensors[2].expand_as(y)) and not gw.any()


@BOTH
@pytest.mark.parametrize("levels,start,N,segments", [
    ([(4, 5), (3, 3)], [2, 30], 45, [(2, 22), (30, 39)]),            # gaps and rows behind the last level
    ([(4, 5), (0, 7), (2, 2)], [0, 20, 20], 24, [(0, 20), (20, 20), (20, 24)]),
    ([(4, 5)], [0], 12, [(0, 12)]),                                  # more than there is
    ([(4, 5), (4, 5)], [0, 10], 40, [(0, 20), (20, 20 + 0)]),        # the second begins inside of the first
    ([(2, 2)], [50], 40, [(40, 40)]),
])
def test_level_tables_that_leave_rows_out(lib_built, levels, start, N, segments, native):
    if levels == [(4, 5), (4, 5)]:
        segments = [(0, 20), (20, 30)]
    shapes, lsi = table(levels, start)
    tensors, g = inputs(2, N, 24, torch.float32, len(levels))
    y, gx, gw, gb = check(native, tensors, g, 3, "silu", shapes, lsi, segments)
    out = torch.ones(N, dtype=torch.bool)
    for lo, hi in segments:
        out[lo:hi] = False
    assert not y[:, out].any() and not gx[:, out].any()
    for l, (lo, hi) in enumerate(segments):
        assert hi > lo or not gw[l].any()


@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("B,C,G,levels,start,N", [
    (2, 96, 12, [(60, 70), (30, 35), (8, 9), (1, 1)], [5, 4300, 5360, 5432], 5500),      # gaps and rows behind the last level
    (1, 90, 6, [(41, 70), (0, 3), (30, 30)], [0, 2870, 2900], 3800),
    (1, 15, 5, [(120, 130), (50, 60)], [100, 15700], 19000),
    (3, 256, 32, [(20, 30), (20, 30)], [0, 500], 1500),                                   # the second begins inside of the first
    (2, 256, 32, [(20, 30), (10, 15), (5, 8)], [0, 600, 750], 1024),                      # the last size of one launch, and the first
    (2, 256, 32, [(20, 30), (10, 15), (5, 8)], [0, 600, 750], 1025),                      # of three
])
def test_level_tables_of_larger_images(lib_built, B, C, G, levels, start, N, dtype):
    shapes, lsi = table(levels, start)
    tensors, g = inputs(B, N, C, dtype, len(levels))
    segments, at = [], 0
    for (h, w), first in zip(levels, start):
        lo = max(first, at)
        at = max(lo, min(first + h * w, N))
        segments.append((lo, at))
    y, gx, _, _ = check(True, tensors, g, G, "silu", shapes, lsi, segments)
    out = torch.ones(N, dtype=torch.bool)
    for lo, hi in segments:
        out[lo:hi] = False
    assert not y[:, out].any() and not gx[:, out].any()


@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
@pytest.mark.parametrize("B,N,C,G", [(6, 5000, 256, 32), (1, 23000, 128, 16), (200, 40, 64, 8), (2, 3001, 90, 9)])
def test_larger_calls_and_the_same_bits_again(lib_built, B, N, C, G, dtype):
    tensors, g = inputs(B, N, C, dtype)
    got = check(True, tensors, g, G, "silu")
    again = check(True, tensors, g, G, "silu")
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("B,N,C,G", [(2, 70000, 256, 32), (1, 90000, 200, 25), (1, 150000, 96, 3)])
def test_images_that_are_cut_into_slabs_of_channels(lib_built, B, N, C, G):
    """Images too large for one batch of work; the last slab is narrower than the others in one of the directions."""
    tensors, g = inputs(B, N, C, torch.float32)
    check(True, tensors, g, G)


@BOTH
@pytest.mark.parametrize("dtype", R.DTYPES, ids=str)
def test_addresses_off_the_grid_and_strides(lib_built, dtype, native):
    tensors, g = inputs(2, 60, 32, dtype)
    check(native, tensors, g, 4)
    x = tensors[0]
    moved = torch.empty(x.numel() + 3, dtype=dtype, device=DEV)[1:1 + x.numel()].view(x.shape).copy_(x)
    check(native, [moved] + tensors[1:], g, 4)
    turned = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert not turned.is_contiguous()
    assert torch.equal(apply(native, turned, *tensors[1:], 4), apply(native, *tensors, 4))


def test_images_in_channels_last_order(lib_built):
    """A (B, C, H, W) tensor in channels_last memory is read where it lies, and agrees with torch's group norm."""
    from dfa3d_b200 import LevelGroupNorm
    m = LevelGroupNorm(4, 32).to(DEV)
    ref = torch.nn.GroupNorm(4, 32).to(DEV)
    ref.load_state_dict(m.state_dict())
    x = torch.randn(2, 32, 9, 11, device=DEV).contiguous(memory_format=torch.channels_last)
    y = m(x.permute(0, 2, 3, 1))
    assert y.shape == (2, 9, 11, 32)
    want = torch.nn.functional.group_norm(x.double(), 4, ref.weight.double(), ref.bias.double(), ref.eps)
    R.assert_within("y", y.permute(0, 3, 1, 2), want.cpu(), 1e-5)


@BOTH
@pytest.mark.parametrize("needed", [(0,), (1,), (2,), (0, 2)])
def test_some_gradients_only(lib_built, needed, native):
    tensors, g = inputs(2, 50, 24, torch.float32)
    full = [t.clone().requires_grad_(True) for t in tensors]
    want = torch.autograd.grad(apply(native, *full, 4, "silu"), full, g)
    part = [t.clone().requires_grad_(i in needed) for i, t in enumerate(tensors)]
    got = torch.autograd.grad(apply(native, *part, 4, "silu"), [part[i] for i in needed], g)
    assert all(torch.equal(a, want[i]) for a, i in zip(got, needed))
    with torch.no_grad():
        assert torch.equal(apply(native, *part, 4, "silu"), apply(native, *full, 4, "silu"))


@BOTH
def test_nothing_to_do(lib_built, native):
    for shape in ((0, 5, 8), (2, 0, 8)):
        leaves = [torch.zeros(shape, device=DEV, requires_grad=True), torch.ones(8, device=DEV, requires_grad=True),
                  torch.ones(8, device=DEV, requires_grad=True)]
        y = apply(native, *leaves, 2)
        assert y.shape == shape
        grads = torch.autograd.grad(y, leaves, y.detach())
        assert not grads[1].any() and not grads[2].any()


def test_gradient_against_differences(lib_built):
    """As for the other norm: what the difference misses of the slope is computed in 64 bits."""
    levels, segments = [(5, 6), (3, 4)], [(0, 30), (30, 42)]
    shapes, lsi = table(levels)
    tensors, g = inputs(2, 42, 16, torch.float32, 2)
    g64, h = g.cpu().double(), 2.0 ** -6
    f = lambda t: apply(True, *t, 4, "silu", shapes, lsi)
    exact = lambda t: R.group_norm(*t, 4, EPS, "silu", segments, g)
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    grads = torch.autograd.grad(f(leaves), leaves, g)
    k = exact(tensors)
    gen = torch.Generator().manual_seed(1)
    for i, (t, name) in enumerate(zip(tensors, ("gx", "gw", "gb"))):
        v = torch.randint(0, 2, t.shape, generator=gen).double() * 2 - 1
        up, down = ([u if j != i else u + s * h * v.float().to(DEV) for j, u in enumerate(tensors)] for s in (1, -1))
        a, b = exact(up), exact(down)
        got = ((f(up).cpu().double() - f(down).cpu().double()) * g64).sum() / (2 * h)
        rounding = ((a["tol_y"] + b["tol_y"] + R.U * (a["y"].abs() + b["y"].abs())) * g64.abs()).sum() / (2 * h)
        missed = abs(((a["y"] - b["y"]) * g64).sum() / (2 * h) - (k[name] * v).sum())
        own = k[{"gx": "tol_gx", "gw": "tol_w", "gb": "tol_b"}[name]].sum()
        assert abs(got - (grads[i].cpu().double() * v).sum()) <= rounding + missed + own


def test_more_than_two_to_the_31_elements(lib_built):
    """The last image of a batch that long is the image by itself, but for the order in which its rows were summed."""
    B, N, C = 3, 2900000, 256
    assert B * N * C > 1 << 31
    x = torch.empty(B, N, C, dtype=torch.bfloat16, device=DEV)
    for i in range(B):
        x[i].normal_(i, 1 + i)
    w, b = torch.rand(C, device=DEV) + 0.5, torch.randn(C, device=DEV)
    with torch.no_grad():
        y = apply(True, x, w, b, 8)[-1]
        alone = apply(True, x[-1:].clone(), w, b, 8)[0]
    step = R.half_step(torch.bfloat16)
    # one rounding each, and a statistic that differs by (chain of sums) U
    bound = (2 * step + 1e-4) * alone.abs().float() + 1e-3
    assert ((y.float() - alone.float()).abs() <= bound).all()
    mean = alone.float().view(N, 8, 32)
    hat = (mean - b.view(8, 32)) / w.view(8, 32)
    assert hat.mean((0, 2)).abs().max() < 1e-3


@BOTH
def test_autocast_computes_in_float32(lib_built, native):
    (x, w, b), g = inputs(2, 50, 24, torch.float16)
    leaf = x.clone().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.float16):
        y = apply(native, leaf, w, b, 4)
    assert y.dtype == torch.float32 and torch.equal(y, apply(native, x.float(), w, b, 4))
    assert torch.autograd.grad(y, leaf, g.float())[0].dtype == torch.float16


def test_refusals(lib_built):
    from dfa3d_b200 import LevelGroupNorm, group_norm
    (x, w, b), _ = inputs(2, 20, 24, torch.float32)
    shapes, lsi = table([(4, 5)])
    for bad in (x.cpu(), x.double(), x[0, 0]):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            group_norm(bad, 4, w, b)
    for G in (5, 0, -1):
        with pytest.raises(RuntimeError, match="groups"):
            group_norm(x, G, w, b)
    with pytest.raises(ValueError, match="activation"):
        group_norm(x, 4, w, b, activation="gelu")
    with pytest.raises(RuntimeError, match="weight must be"):
        group_norm(x, 4, w[:20], b)
    with pytest.raises(RuntimeError, match="bias must be"):
        group_norm(x, 4, w, b.half())
    with pytest.raises(RuntimeError, match="weight must be"):
        group_norm(x, 4, w.expand(2, 24), b.expand(2, 24), spatial_shapes=shapes, level_start_index=lsi)
    with pytest.raises(RuntimeError, match="together"):
        group_norm(x, 4, w, b, spatial_shapes=shapes)
    with pytest.raises(RuntimeError, match="int64"):
        group_norm(x, 4, w, b, spatial_shapes=shapes.int(), level_start_index=lsi)
    with pytest.raises(RuntimeError, match="one device"):
        group_norm(x, 4, w, b, spatial_shapes=shapes.cpu(), level_start_index=lsi.cpu())
    with pytest.raises(RuntimeError, match="eps must be"):
        group_norm(x, 4, w, b, eps=-1.0)
    with pytest.raises(RuntimeError, match="exceeds 1024"):
        group_norm(torch.zeros(1, 2, 1028, device=DEV), 4, *(torch.zeros(1028, device=DEV),) * 2)
    with pytest.raises(RuntimeError, match="MAX_LEVELS"):
        many = table([(1, 1)] * 33)
        group_norm(torch.zeros(1, 33, 24, device=DEV), 4, w, b, spatial_shapes=many[0], level_start_index=many[1])
    with pytest.raises(ValueError, match="activation"):
        LevelGroupNorm(4, 24, activation="tanh")


def test_module(lib_built):
    from dfa3d_b200 import LevelGroupNorm
    shapes, lsi = table([(4, 5), (2, 3)])
    (x, w, b), _ = inputs(2, 26, 24, torch.float32, 2)
    m = LevelGroupNorm(4, 24, activation="silu", num_levels=2).to(DEV)
    assert list(m.state_dict()) == list(torch.nn.GroupNorm(4, 24).state_dict()) and m.weight.shape == (2, 24)
    with torch.no_grad():
        m.weight.copy_(w); m.bias.copy_(b)
    y = m(x, shapes, lsi)
    assert torch.equal(y, apply(True, x, w, b, 4, "silu", shapes, lsi))
    y.sum().backward()
    assert m.weight.grad.shape == (2, 24)


def test_captured_forward_and_backward_in_two_graphs(lib_built):
    """Two captured passes have workspaces of their own: replayed one after the other and again, each gives its eager results."""
    cases = []
    for B, N, C, G in ((2, 900, 64, 8), (3, 500, 96, 6)):
        tensors, g = inputs(B, N, C, torch.float32)
        leaves = [t.clone().requires_grad_(True) for t in tensors]
        step = lambda leaves=leaves, g=g, G=G: (lambda y: (y,) + torch.autograd.grad(y, leaves, g))(apply(True, *leaves, G, "silu"))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [t.detach().clone() for t in step()]      # no eager graph outlives this
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        cases.append((graph, out, want))
    for _ in range(2):
        for graph, out, want in cases:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out, want in cases:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
