"""What the feed-forward operators keep until the backward: nothing where only the residual is trained, and nothing that is not read stands
in the way of a gradient."""
import pytest
import torch

from dfa3d_b200.feed_forward_ops import GatedFeedForwardFunction, LinearActFunction
from test_gpu_native_path import _python

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
KINDS = pytest.mark.parametrize("kind", ["linear", "gated"])
FORMS = pytest.mark.parametrize("checkpoint", [None, "int8"])


def _inputs(rows=64, E=40):
    g = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g).bfloat16().to(DEV)
    return dict(x=n(rows, E), w=[n(E, E) for _ in range(3)], b=[n(E) for _ in range(3)], r=torch.randn(rows, E, generator=g).to(DEV))


def _call(kind, native, d, checkpoint):
    linear, gated = (f if native else _python(f) for f in (LinearActFunction, GatedFeedForwardFunction))
    if kind == "linear":
        return linear.apply(d["x"], d["w"][0], d["b"][0], d["r"], "gelu", checkpoint)
    return gated.apply(d["x"], *d["w"], *d["b"], d["r"], False, "silu", checkpoint)


@BOTH
@KINDS
@FORMS
def test_nothing_where_only_the_residual_is_trained(lib_built, native, kind, checkpoint):
    """The input may be changed before the backward: nothing of it is read."""
    d = _inputs()
    d["r"].requires_grad_(True)
    y = _call(kind, native, d, checkpoint)
    d["x"].zero_()
    for t in d["w"] + d["b"]:
        t.zero_()
    go = torch.randn_like(y)
    y.backward(go)
    assert torch.equal(d["r"].grad, go)


@BOTH
@KINDS
@FORMS
def test_no_memory_either(lib_built, native, kind, checkpoint):
    d = _inputs(rows=8192, E=256)
    d["r"].requires_grad_(True)
    x = d.pop("x")
    _call(kind, native, dict(d, x=x), checkpoint)               # what a first call sets up
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = _call(kind, native, dict(d, x=x.clone()), checkpoint)
    assert torch.cuda.memory_allocated() - before <= y.numel() * 4 + 4096


@KINDS
@FORMS
def test_a_gradient_of_the_residual_alone(lib_built, kind, checkpoint):
    """Asked for by itself of a call that keeps its input for others."""
    d = _inputs()
    for t in [d["x"], d["r"]] + d["w"] + d["b"]:
        t.requires_grad_(True)
    y = _call(kind, True, d, checkpoint)
    with torch.no_grad():
        d["x"].zero_()
        d["w"][0].zero_()
    go = torch.randn_like(y)
    got, = torch.autograd.grad(y, d["r"], go)
    assert torch.equal(got, go)


@BOTH
@KINDS
@pytest.mark.parametrize("trained", ["x", "w", "b"])
def test_what_is_read_is_kept(lib_built, native, kind, trained):
    d = _inputs()
    t = d[trained] if trained == "x" else d[trained][0]
    t.requires_grad_(True)
    want, = torch.autograd.grad(_call(kind, native, d, None), t, torch.ones_like(d["r"]))
    y = _call(kind, native, d, None)
    with torch.no_grad():
        d["w"][0].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, t, torch.ones_like(y))
    assert (want != 0).any()


@KINDS
def test_biases_that_are_absent(lib_built, kind):
    """Gradients are those of the inputs that they belong to, whichever are there."""
    d = _inputs()
    d["b"] = [None, None, d["b"][2]]
    leaves = [d["x"], d["r"]] + d["w"] + ([d["b"][2]] if kind == "gated" else [])
    for t in leaves:
        t.requires_grad_(True)
    leaves = leaves if kind == "gated" else leaves[:3]
    go = torch.randn_like(d["r"])
    a, b = (torch.autograd.grad(_call(kind, native, d, None), leaves, go) for native in (True, False))
    assert all(torch.equal(s, t) for s, t in zip(a, b)) and torch.equal(a[1], go)
