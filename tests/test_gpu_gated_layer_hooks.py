"""Encoder layers with the gated block whose block carries hooks or has been replaced: every hook runs, a replacement is called, and hooks
that change nothing change nothing, in float32 outside autocast too."""
import pytest
import torch
import torch.nn as nn

from dfa3d_b200 import GatedFeedForward
from test_gpu_counter_dropout_modules import KEYS
from test_gpu_feed_forward_together import _layer
from test_gpu_modules import DEV, _inputs

pytestmark = pytest.mark.gpu


def _call(layer, d, q=None):
    return layer(d["query"] if q is None else q, **{k: d[k] for k in KEYS})


def _leaves(layer):
    return [layer.ffn.gate.weight, layer.ffn.up.bias, layer.ffn.down.weight, layer.norm2.weight]


HOOKS = {
    "forward": lambda m, seen: m.register_forward_hook(lambda mod, a, y: seen.append(y.dtype)),
    "pre": lambda m, seen: m.register_forward_pre_hook(lambda mod, a: seen.append(a[0].dtype)),
    "backward": lambda m, seen: m.register_full_backward_hook(lambda mod, gi, go: seen.append(go[0].dtype)),
}


@pytest.mark.parametrize("kind", ["cross", "full"])
@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("autocast", [False, True])
def test_hooks_on_the_block(lib_built, kind, hook, autocast):
    layer, d = _layer(kind, dropout=0.0, gated_feed_forward=dict(activation="gelu")), _inputs(6)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        want, seen = _call(layer, d), []
        HOOKS[hook](layer.ffn, seen)
        got = _call(layer, d)
    assert got.dtype == torch.float32 and torch.equal(got, want)
    g = torch.randn(got.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    grads = []
    for y in (want, got):
        layer.zero_grad()
        y.backward(g)
        grads.append([p.grad for p in _leaves(layer)])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    assert seen == [torch.float32]


@pytest.mark.parametrize("counter", [False, True])
def test_hooks_with_dropout(lib_built, counter):
    layer, d = _layer("cross", dropout=0.2, counter_dropout=counter, gated_feed_forward=True), _inputs(6)
    x, calls = [], []

    def seeded(m, a, y):
        torch.manual_seed(5)
        x.append(y)

    layer.norm1.register_forward_hook(seeded)
    layer.ffn.register_forward_hook(lambda m, a, y: calls.append(y))
    got = _call(layer, d)
    assert len(calls) == 1
    torch.manual_seed(5)
    assert torch.equal(got, layer.norm2(layer.ffn(x[0], x[0])))
    got.sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in layer.ffn.parameters())
    layer.eval()
    hooked = _call(layer, d)
    layer.ffn._forward_hooks.clear()
    assert torch.equal(hooked, _call(layer, d))


def test_hooks_for_all_modules(lib_built):
    layer, d = _layer("cross", dropout=0.0, gated_feed_forward=True), _inputs(6)
    want, seen = _call(layer, d), []
    handle = nn.modules.module.register_module_forward_hook(lambda m, a, y: seen.append(m))
    try:
        got = _call(layer, d)
    finally:
        handle.remove()
    assert got.dtype == torch.float32 and layer.ffn in seen
    # the branch is rounded to 16 bits once more on its way through the hooked modules
    torch.testing.assert_close(got, want, rtol=2e-2, atol=2e-2)


class _Louder(GatedFeedForward):
    def branch(self, x, residual=None):
        return 2 * super().branch(x, residual)


class _Alone(GatedFeedForward):
    def forward(self, x):
        return self.branch(x)


class _Adapter(nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x) * 0.5


@pytest.mark.parametrize("kind", ["branch", "forward", "adapter", "instance"])
def test_replaced_blocks(lib_built, kind):
    layer, d = _layer("cross", dropout=0.0, gated_feed_forward=True), _inputs(6)
    x = []
    layer.norm1.register_forward_hook(lambda m, a, y: x.append(y))
    block = layer.ffn
    if kind == "branch":
        block.__class__ = _Louder
    elif kind == "forward":
        block.__class__ = _Alone
    elif kind == "adapter":
        layer.ffn = _Adapter(block)
    else:
        block.forward = lambda t: block.branch(t) * 0.25
    got = _call(layer, d)
    if kind == "branch":
        want = layer.norm2(layer.ffn(x[0], x[0]))
    else:
        y = layer.ffn(x[0])
        assert y.dtype == torch.bfloat16
        want = layer.norm2(y.float(), x[0])
    assert got.dtype == torch.float32 and torch.equal(got, want)
