"""Hooks on the gated block's three products and modules in their place: they run, as they do for a block of torch's own modules."""
import pytest
import torch
import torch.nn as nn

import ffn_reference as ref
from dfa3d_b200 import GatedFeedForward, LinearAct

pytestmark = pytest.mark.gpu
DEV = "cuda"
CHILDREN = ("gate", "up", "down")


def _block(rows=70, E=40, F=56, act="silu", dtype=torch.bfloat16, **kw):
    torch.manual_seed(4)
    block = GatedFeedForward(E, F, activation=act, compute_dtype=dtype, **kw).to(DEV)
    return block, torch.randn(rows, E, device=DEV)


@pytest.mark.parametrize("child", CHILDREN)
@pytest.mark.parametrize("autocast", [False, True])
def test_a_hook_changes_what_it_returns_another_value_for(lib_built, child, autocast):
    block, x = _block()
    seen = []

    def twice(m, a, y):
        seen.append(y.dtype)
        return 2 * y

    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        block.get_submodule(child).register_forward_hook(twice)
        got = block(x)
    assert seen == [torch.bfloat16]
    with torch.no_grad():
        m = block.get_submodule(child)
        m._forward_hooks.clear()
        m.weight.mul_(2)
        m.bias.mul_(2)
    want = block(x)
    # twice a parameter is twice its product, exactly; gate, up, hidden row and result are rounded apart from the one form
    scale = float(want.detach().float().abs().max())
    assert float((got.float() - want.float()).detach().abs().max()) <= 0.03 * scale


@pytest.mark.parametrize("child", CHILDREN)
def test_a_weight_that_a_hook_forms_anew(lib_built, child):
    """As torch's weight and spectral norms do."""
    block, x = _block()
    m = block.get_submodule(child)
    raw = m.weight.detach().clone()
    del m._parameters["weight"]
    m.weight = raw * 1e3                                        # stale until the hook has run
    m.raw = nn.Parameter(raw)
    m.register_forward_pre_hook(lambda mod, a: setattr(mod, "weight", mod.raw / mod.raw.norm()))
    y = block(x)
    assert torch.isfinite(y.float()).all() and float(y.detach().float().abs().max()) < 10
    y.float().sum().backward()
    assert m.raw.grad is not None and torch.isfinite(m.raw.grad).all() and (m.raw.grad != 0).any()


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("residual", [False, True])
def test_called_one_by_one(lib_built, act, dtype, residual):
    """Every call is seen, and the result is the definition's with gate, up, hidden row and branch rounded."""
    block, x = _block(act=act, dtype=dtype)
    seen = []
    for name in CHILDREN:
        block.get_submodule(name).register_forward_hook(lambda m, a, y, n=name: seen.append(n))
    y = block(x, x if residual else None)
    assert sorted(seen) == sorted(CHILDREN)
    assert y.dtype == (torch.float32 if residual else dtype)
    low = lambda t: ref.exactly(t.detach().to(dtype))
    X = low(x)
    part = lambda m, v: ref.rounded(ref.plus(ref.product(v, ref.transposed(low(m.weight))), low(m.bias)), dtype)
    h = ref.rounded(ref.times(ref.act(part(block.gate, X), act)[0], part(block.up, X)), dtype)
    q = part(block.down, h)
    ref.near("y", y, ref.plus(q, ref.exactly(x)) if residual else q)
    y.float().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in block.parameters())


@pytest.mark.parametrize("child", CHILDREN)
def test_hooks_that_change_nothing(lib_built, child):
    """The same block within the roundings, gradients too."""
    results = []
    for hooked in (False, True):
        block, x = _block(act="gelu", checkpoint="int8")
        if hooked:
            block.get_submodule(child).register_full_backward_hook(lambda m, gi, go: None)
        x.requires_grad_(True)
        y = block(x, x)
        results.append((y,) + torch.autograd.grad(y, [x] + list(block.parameters()), torch.ones_like(y)))
    for a, b in zip(*results):
        assert float((a.double() - b.double()).norm()) <= 0.02 * float(a.double().norm())


class _Adapter(nn.Module):
    """A product with a small one beside it."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner
        self.small = LinearAct(inner.in_features, inner.out_features, bias=False)

    def forward(self, x):
        return self.inner(x) + self.small(x)


@pytest.mark.parametrize("child", CHILDREN)
def test_a_module_in_a_products_place(lib_built, child):
    block, x = _block()
    block.set_submodule(child, _Adapter(block.get_submodule(child)).to(DEV))
    y = block(x)
    y.float().sum().backward()
    small = block.get_submodule(child).small.weight
    assert small.grad is not None and (small.grad != 0).any()
    with torch.no_grad():
        small.zero_()
        inner = block.get_submodule(child).inner
        got = block(x)
        block.set_submodule(child, inner)
        want = block(x)
    assert float((got.float() - want.float()).norm()) <= 0.02 * float(want.float().norm())


def test_an_activation_given_to_a_product(lib_built):
    block, x = _block(act=None)
    block.up = LinearAct(40, 56, activation="relu").to(DEV)
    with torch.no_grad():
        up = block.up(x.bfloat16()).float()
        want = block.down((block.gate(x.bfloat16()).float() * up).bfloat16())
        assert torch.equal(block(x), want)


def test_parametrized_weights_stay_with_one_call(lib_built):
    block, x = _block()
    want = block(x)
    torch.nn.utils.parametrize.register_parametrization(block.gate, "weight", nn.Identity())
    assert torch.equal(block(x), want)


def test_unknown_activations_are_refused_either_way(lib_built):
    block, x = _block(act="tanh")
    with pytest.raises(ValueError, match="activation"):
        block(x)
    block.up.register_forward_hook(lambda m, a, y: None)
    with pytest.raises(ValueError, match="activation"):
        block(x)
