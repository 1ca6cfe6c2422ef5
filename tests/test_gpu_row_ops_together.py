"""Dropout, dropout + LayerNorm and group norm as programs run them: on two streams at once, with saved-tensor hooks, traced, in a
captured training step of a layer, beside rows that hold no numbers."""
import pytest
import torch

import test_gpu_counter_dropout_modules as layers
from dfa3d_b200 import CounterDropout, dropout, dropout_add_layer_norm, group_norm, layer_ops
from dfa3d_b200.dropout_ops import DropoutAddLayerNormFunction, DropoutFunction
from dfa3d_b200.group_norm_ops import GroupNormFunction
from dfa3d_b200.rebatch import RebatchPlan
from test_gpu_native_path import _python

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = ["dropout", "relu", "residual", "norm", "group", "linear"]
BOTH = pytest.mark.parametrize("native", [True, False], ids=["native", "python"])


def call(kind, native=True, rows=37, E=32, seed=5):
    """A function of no arguments that runs the forward, and its leaves."""
    g = torch.Generator().manual_seed(1)
    s = torch.tensor([seed], device=DEV)
    x, r = (torch.randn(rows, E, generator=g).to(DEV).requires_grad_(True) for _ in range(2))
    w, b = ((torch.randn(E, generator=g) + 1).to(DEV).requires_grad_(True) for _ in range(2))
    image = torch.randn(2, rows, E, generator=g).to(DEV).requires_grad_(True)
    shapes, start = torch.tensor([[5, 6], [1, 4]], device=DEV), torch.tensor([0, 30], device=DEV)
    linear, relu = layer_ops.Linear(E, 2 * E).to(DEV), torch.nn.ReLU()
    drop, norm, group = (f if native else _python(f) for f in (DropoutFunction, DropoutAddLayerNormFunction, GroupNormFunction))
    return {
        "dropout": (lambda: drop.apply(x, None, s, 0.3, 1, None), [x]),
        "relu": (lambda: drop.apply(x, None, s, 0.3, 1, "relu"), [x]),
        "residual": (lambda: drop.apply(x, r, s, 0.3, 1, "relu"), [x, r]),
        "norm": (lambda: norm.apply(x, r, w, b, s, 0.3, 2, 1e-5), [x, r, w, b]),
        "group": (lambda: group.apply(image, w, b, shapes, start, 4, 1e-5, "silu"), [image, w, b]),
        "linear": (lambda: layer_ops.linear_relu_dropout(x, linear, relu, CounterDropout(0.3), lambda device: s, 2), [x, linear.weight, linear.bias]),
    }[kind]


@BOTH
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hook", ["cpu", "layout"])
def test_hooks_that_hand_back_equal_tensors(lib_built, kind, hook, native):
    f, leaves = call(kind, native)
    out = f()
    go = torch.randn(out.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = torch.autograd.grad(out, leaves, go)
    pack, unpack = {"cpu": (lambda t: t.cpu(), lambda t: t.to(DEV)),
                    "layout": (lambda t: t.clone(), lambda t: t.transpose(0, -1).contiguous().transpose(0, -1))}[hook]
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        out = f()
    for a, b in zip(torch.autograd.grad(out, leaves, go), want):
        # the same kernels on the same numbers; "linear" has products and a sum over rows whose order is not fixed: 37 terms
        torch.testing.assert_close(a, b, rtol=1e-5 if kind == "linear" else 0, atol=1e-5 if kind == "linear" else 0)


@BOTH
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hook", ["type", "size"])
def test_hooks_that_hand_back_other_tensors(lib_built, kind, hook, native):
    if kind == "linear" and not native:
        pytest.skip("its parts are tested by themselves")
    f, leaves = call(kind, native)
    # another type of whatever is saved (the dropout alone keeps an int64 seed), or one element of it too few
    pack = (lambda t: t.half() if t.is_floating_point() else t.int()) if hook == "type" else (lambda t: t.flatten()[1:].clone())
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = f()
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        torch.autograd.grad(out, leaves, torch.ones_like(out))


def test_a_hook_that_changes_the_shape_alone(lib_built):
    """Counts decide what the kernels read, not the shape that a hook hands back."""
    f, leaves = call("norm")
    go = torch.randn(37, 32, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = torch.autograd.grad(f(), leaves, go)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.flatten(), lambda t: t):
        out = f()
    for a, b in zip(torch.autograd.grad(out, leaves, go), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", KINDS[:-1])
def test_calls_on_two_streams_at_once(lib_built, kind):
    calls = [call(kind, rows=2000, E=64, seed=i) for i in (1, 2)]
    streams = [torch.cuda.Stream() for _ in calls]

    def one(i):
        f, leaves = calls[i]
        y = f()
        return [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))]

    want = [one(0), one(1)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(one(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for tensors in got[i]:
            for a, b in zip(tensors, want[i]):
                assert torch.equal(a, b)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_traced_calls_follow_their_inputs(lib_built):
    s = torch.tensor([3], device=DEV)
    w, b = torch.rand(32, device=DEV), torch.rand(32, device=DEV)

    def run(x):
        x = dropout(x, 0.2, s, 1, "relu", x)
        x = dropout_add_layer_norm(x, x * 2, w, b, 0.2, s, 2)
        return group_norm(x[None], 4, w, b, activation="silu")

    with torch.no_grad():
        traced = torch.jit.trace(run, (torch.randn(9, 32, device=DEV),), check_trace=False)
        x = torch.randn(9, 32, device=DEV)
        want = run(x)
        spoil = [torch.full((9, 32), float("nan"), device=DEV) for _ in range(16)]
        del spoil
        assert torch.equal(traced(x), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("N", [50, 12000])
def test_rows_of_no_level_are_not_looked_at(lib_built, bad, N):
    g = torch.Generator().manual_seed(0)
    x, go = torch.randn(2, N, 24, generator=g).to(DEV), torch.randn(2, N, 24, generator=g).to(DEV)
    w, b = torch.rand(24, device=DEV).requires_grad_(True), torch.rand(24, device=DEV).requires_grad_(True)
    shapes, start = torch.tensor([[2, 7], [4, 4]], device=DEV), torch.tensor([3, 20], device=DEV)
    outside = torch.ones(N, dtype=torch.bool)
    outside[3:17] = outside[20:36] = False
    results = []
    for spoiled in (False, True):
        xs, gs = x.clone(), go.clone()
        if spoiled:
            xs[:, outside], gs[:, outside] = bad, bad
        xs.requires_grad_(True)
        y = group_norm(xs, 3, w, b, 1e-5, "silu", shapes, start)
        results.append([y.detach(), *torch.autograd.grad(y, [xs, w, b], gs)])
    for a, c in zip(*results):
        assert torch.equal(a, c)
    assert not results[1][0][:, outside].any() and not results[1][1][:, outside].any()


def test_one_image_without_numbers_spoils_no_other(lib_built):
    x = torch.randn(3, 40, 32, generator=torch.Generator().manual_seed(0)).to(DEV)
    w, b = torch.rand(32, device=DEV), torch.rand(32, device=DEV)
    want = group_norm(x, 4, w, b)
    x[1, 7, 9] = float("nan")                           # group 1 of image 1
    got = group_norm(x, 4, w, b)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[1, :, 8:16] = True
    assert torch.equal(got[~hit], want[~hit]) and got[hit].isnan().all()
    rows = x.view(-1, 32)
    seed = torch.tensor([3], device=DEV)
    y = dropout_add_layer_norm(rows, torch.zeros_like(rows), w, b, 0.0, seed)
    assert y.isnan().any(1).nonzero().flatten().tolist() == [47]


def test_captured_training_step_of_a_layer(lib_built, monkeypatch):
    """Every replay forms the masks of the seed it finds, in its backward as in its forward."""
    seed = torch.tensor([11], dtype=torch.int64, device=DEV)
    monkeypatch.setattr(layer_ops, "draw_seed", lambda device="cuda", generator=None: seed.clone())
    layer, d = layers._layer("full"), layers._inputs(6)
    kw = {k: d[k] for k in layers.KEYS}
    kw["rebatch_plan"] = RebatchPlan(kw["bev_mask"])           # counted before the capture
    query = d["query"].clone().requires_grad_(True)
    leaves = [query] + list(layer.parameters())
    go = torch.randn(query.shape, generator=torch.Generator().manual_seed(1)).to(DEV)

    def step():
        y = layer(query, **kw)
        return [y.detach(), *torch.autograd.grad(y, leaves, go)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    seen = []
    for value in (11, 12):
        seed.fill_(value)
        graph.replay()
        got = [t.clone() for t in out]
        layers._close(got, step())
        seen.append(got[0])
    assert not torch.equal(*seen)
