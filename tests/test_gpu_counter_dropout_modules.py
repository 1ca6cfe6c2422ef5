"""Encoder layers built with counter_dropout=True: what they run inside their kernels is their blocks applied one by one with the same
masks; blocks that carry hooks are called; layers built without it have torch's dropout as before.  And the row operators
together as a model uses them: group norm of the features, attention, dropout inside norms and feed-forward block."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import row_reference as R
from dfa3d_b200 import CounterDropout, LevelGroupNorm, dropout, layer_ops, modules
from dfa3d_b200.layer_ops import Linear
from test_gpu_modules import DEV, _inputs

pytestmark = pytest.mark.gpu
KEYS = ("value", "value_dpt_dist", "reference_points_cam", "bev_mask", "spatial_shapes", "level_start_index")
P = 0.25


def seed_tensor(value):
    return torch.tensor([value], dtype=torch.int64, device=DEV)


@pytest.fixture
def seed(monkeypatch):
    """Every pass draws this seed."""
    monkeypatch.setattr(layer_ops, "draw_seed", lambda device="cuda", generator=None: seed_tensor(77))
    monkeypatch.setattr("dfa3d_b200.dropout_ops.draw_seed", lambda device="cuda", generator=None: seed_tensor(77))
    return seed_tensor(77)


def _layer(kind, counter=True, p=P):
    torch.manual_seed(2)
    kw = dict(embed_dims=32, ffn_dims=64, num_cams=3, num_heads=2, num_levels=2, num_points=8, dropout=p, counter_dropout=counter)
    if kind == "full":
        kw.update(bev_h=5, bev_w=10)
    layer = (modules.BEVFormerEncoderLayer if kind == "full" else modules.SCAEncoderLayer)(**kw).to(DEV)
    with torch.no_grad():
        for m in layer.modules():
            if isinstance(m, nn.Linear) and not m.weight.any():
                m.weight.normal_(0, 0.05)
    return layer


def _block_by_block(layer, query, seed, kw):
    """The layer's blocks with `dropout` between them, at the sites that the layer uses."""
    def norm(n, branch, residual, site):
        return F.layer_norm(dropout(branch, P, seed, site) + residual, (32,), n.weight, n.bias, n.eps)

    if hasattr(layer, "self_attn"):
        shapes, lsi, cells = layer._bev_tables(query.device, query.dtype)
        branch, residual = layer.self_attn(query, reference_points=cells.expand(2, -1, -1, -1), spatial_shapes=shapes,
                                           level_start_index=lsi, return_residual="undropped")
        query = norm(layer.norm0, branch, residual, 0)
    branch, residual = layer.cross_attn(query, return_residual="undropped", **kw)
    query = norm(layer.norm1, branch, residual, 1)
    h = dropout(F.linear(query, layer.ffn[0].weight, layer.ffn[0].bias).relu(), P, seed, 2)
    return norm(layer.norm2, F.linear(h, layer.ffn[3].weight, layer.ffn[3].bias), query, 3)


def _close(got, want):
    # products and norms of 32 to 64 elements in another order, through up to three blocks
    for i, (a, b) in enumerate(zip(got, want)):
        scale = float(b.detach().abs().max())
        assert float((a - b).detach().abs().max()) <= 2e-4 * scale + 1e-6, (i, float((a - b).detach().abs().max()), scale)


@pytest.mark.parametrize("kind", ["full", "cross"])
def test_layer_is_its_blocks_with_the_same_masks(lib_built, seed, kind):
    layer, d = _layer(kind), _inputs(6)
    kw = {k: d[k] for k in KEYS}
    g = torch.randn(d["query"].shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    results = []
    for f in (lambda q: layer(q, **kw), lambda q: _block_by_block(layer, q, seed, kw)):
        q = d["query"].clone().requires_grad_(True)
        y = f(q)
        results.append((y.detach(),) + torch.autograd.grad(y, [q] + list(layer.parameters()), g))
    _close(*results)


def test_the_masks_are_those_of_the_definition(lib_built, seed):
    """The last norm's input, seen through an identity of a norm: dropped where the definition says so."""
    layer, d = _layer("cross"), _inputs(6)
    kw = {k: d[k] for k in KEYS}
    hidden = []
    layer.ffn[3].register_forward_hook(lambda m, a, y: hidden.append((a[0].detach(), y.detach())))
    layer(d["query"], **kw)
    h, _ = hidden[0]
    keep = R.kept(h.shape, P, 77, 2).to(DEV)
    assert not h[~keep].any() and (h[keep] > 0).float().mean() > 0.2


@pytest.mark.parametrize("kind", ["full", "cross"])
def test_evaluation_is_that_of_a_layer_without_it(lib_built, kind):
    a, b, d = _layer(kind).eval(), _layer(kind, counter=False).eval(), _inputs(6)
    assert list(a.state_dict()) == list(b.state_dict())
    kw = {k: d[k] for k in KEYS}
    with torch.no_grad():
        assert torch.equal(a(d["query"], **kw), b(d["query"], **kw))


def test_layers_are_built_with_torchs_dropout_unless_asked(lib_built):
    layer = _layer("full", counter=False)
    kinds = [type(m) for m in layer.modules() if isinstance(m, nn.Dropout)]
    assert kinds == [nn.Dropout] * 4
    assert [type(m) for m in _layer("full").modules() if isinstance(m, nn.Dropout)] == [CounterDropout] * 4
    d = _inputs(6)
    kw = {k: d[k] for k in KEYS}
    torch.manual_seed(5)
    got = layer(d["query"], **kw)
    torch.manual_seed(5)
    shapes, lsi, cells = layer._bev_tables(d["query"].device, torch.float32)
    q = layer.norm0(*layer.self_attn(d["query"], reference_points=cells.expand(2, -1, -1, -1), spatial_shapes=shapes,
                                     level_start_index=lsi, return_residual=True))
    q = layer.norm1(*layer.cross_attn(q, return_residual=True, **kw))
    assert torch.equal(got, layer.norm2(layer.ffn(q), q))


def test_every_pass_has_other_masks_and_a_torch_seed_repeats_them(lib_built):
    layer, d = _layer("full"), _inputs(6)
    kw = {k: d[k] for k in KEYS}
    with torch.no_grad():
        torch.manual_seed(3)
        a, b = layer(d["query"], **kw), layer(d["query"], **kw)
        torch.manual_seed(3)
        assert torch.equal(layer(d["query"], **kw), a) and not torch.equal(a, b)


@pytest.mark.parametrize("where", ["norm1", "ffn", "ffn.0", "ffn.2", "ffn.4", "cross_attn", "cross_attn.dropout"])
def test_hooks_see_every_call(lib_built, seed, where):
    layer, d = _layer("cross"), _inputs(6)
    calls = []
    layer.get_submodule(where).register_forward_hook(lambda m, a, y: calls.append(y))
    y = layer(d["query"], **{k: d[k] for k in KEYS})
    y.sum().backward()
    assert len(calls) == 1 and torch.isfinite(y).all()


@pytest.mark.parametrize("kind", ["none", "other dropout", "short"])
def test_replaced_blocks_are_called(lib_built, seed, kind):
    layer, d = _layer("cross"), _inputs(6)
    if kind == "none":
        layer.ffn[2] = nn.Identity()
    elif kind == "other dropout":
        layer.ffn[4] = nn.Dropout(0.0)
    else:
        layer.ffn = nn.Sequential(Linear(32, 32), nn.ReLU()).to(DEV)
    seen = []
    layer.norm1.register_forward_hook(lambda m, a, y: seen.append(y))
    got = layer(d["query"], **{k: d[k] for k in KEYS})
    want = layer.norm2(layer.ffn(seen[0]), seen[0])
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("module", ["cross", "self", "decoder"])
def test_attention_modules_by_themselves(lib_built, seed, module):
    d = _inputs(6)
    torch.manual_seed(4)
    if module == "cross":
        m = modules.SpatialCrossAttention_DFA3D(32, 3, P, modules.MSDeformableAttention3D_DFA3D(32, 2, 2, 8),
                                                counter_dropout=True).to(DEV)
        kw = {k: d[k] for k in KEYS}
    else:
        cls = modules.TemporalSelfAttention if module == "self" else modules.CustomMSDeformableAttention
        m = cls(32, 2, num_levels=1, num_points=4, dropout=P, batch_first=True, counter_dropout=True).to(DEV)
        bs = 2 if module == "self" else 1
        kw = dict(reference_points=modules.bev_reference_points(5, 10, dim="2d", device=DEV).expand(bs, -1, -1, -1),
                  spatial_shapes=torch.tensor([[5, 10]], device=DEV), level_start_index=torch.tensor([0], device=DEV))
    got = m(d["query"], **kw)
    m.eval()
    branch = m(d["query"], **kw) - d["query"]
    want = dropout(branch, P, seed) + d["query"]
    assert torch.equal(got == d["query"], want == d["query"])
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)
    m.train()
    got.sum().backward()
    assert torch.isfinite(m.output_proj.weight.grad).all()


@pytest.mark.parametrize("rows", [1, 77, 16384 + 5])
def test_linear_relu_dropout_is_its_parts(lib_built, rows):
    torch.manual_seed(1)
    linear, drop = Linear(40, 64).to(DEV), CounterDropout(P)
    x, g = torch.randn(rows, 40, device=DEV), torch.randn(rows, 64, device=DEV)
    results = []
    for fused in (True, False):
        xi = x.clone().requires_grad_(True)
        y = layer_ops.linear_relu_dropout(xi, linear, nn.ReLU(), drop, lambda dev: seed_tensor(9), 5) if fused else \
            dropout(layer_ops.linear_relu(xi, linear, nn.ReLU()), P, seed_tensor(9), 5)
        results.append((y.detach(),) + torch.autograd.grad(y, [xi, linear.weight, linear.bias], g))
    assert torch.equal(results[0][0], results[1][0])
    y = layer_ops.linear_relu_dropout(x.requires_grad_(True), linear, nn.ReLU(), drop, lambda dev: seed_tensor(9), 5)
    assert "LinearReluDropout" in y.grad_fn.name()
    # the same products; sums over `rows` in another order
    for a, b in zip(results[0][1:], results[1][1:]):
        assert float((a - b).abs().max()) <= 8 * R.U * max(rows, 16) ** 0.5 * float(b.abs().max())


def test_under_autocast_and_in_half(lib_built, seed):
    layer, d = _layer("cross"), _inputs(6)
    kw = {k: d[k] for k in KEYS}
    want = layer(d["query"], **kw)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = layer(d["query"], **kw)
        got.float().sum().backward()
    assert torch.isfinite(got).all() and torch.isfinite(layer.ffn[0].weight.grad).all()
    # the package's Linear and norms compute in float32 under autocast: the same numbers, other kernels
    _close([got.float()], [want])


def test_checkpointed_layer_has_the_same_masks_in_its_second_forward(lib_built):
    from torch.utils.checkpoint import checkpoint
    layer, d = _layer("cross"), _inputs(6)
    kw = {k: d[k] for k in KEYS}
    g = torch.randn(d["query"].shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    results = []
    for f in (lambda q: layer(q, **kw), lambda q: checkpoint(lambda t: layer(t, **kw), q, use_reentrant=False)):
        torch.manual_seed(9)
        q = d["query"].clone().requires_grad_(True)
        y = f(q)
        results.append((y.detach(),) + torch.autograd.grad(y, [q] + list(layer.parameters()), g))
    assert torch.equal(results[0][0], results[1][0])
    _close(*results)


def test_features_to_layer_in_one_training_pass(lib_built, seed):
    """Projected features of two levels -> group norm with SiLU -> value -> encoder layer with counter dropout, against the same model
    of torch's operators with the masks of the definition."""
    layer, d = _layer("full"), _inputs(6)
    torch.manual_seed(8)
    norm = LevelGroupNorm(4, 32, activation="silu", num_levels=2).to(DEV)
    with torch.no_grad():
        norm.weight.normal_(1, 0.2), norm.bias.normal_(0, 0.2)
    features = d["value"][:, :, 0].clone() * 3 + 1                       # (cams, N, E)
    kw = {k: d[k] for k in KEYS if k != "value"}
    levels = [(int(h), int(w)) for h, w in d["spatial_shapes"].tolist()]
    g = torch.randn(d["query"].shape, generator=torch.Generator().manual_seed(1)).to(DEV)

    def plain_norm(x):
        out, at = [], 0
        for l, (h, w) in enumerate(levels):
            y = F.group_norm(x[:, at:at + h * w].transpose(1, 2), 4, norm.weight[l], norm.bias[l], norm.eps)
            out.append(F.silu(y).transpose(1, 2))
            at += h * w
        return torch.cat(out, 1)

    def model(x, q):
        return layer(q, value=norm(x, d["spatial_shapes"], d["level_start_index"])[:, :, None], **kw)

    def reference(x, q):
        return _block_by_block(layer, q, seed, dict(kw, value=plain_norm(x)[:, :, None]))

    results = []
    for f in (model, reference):
        x, q = features.clone().requires_grad_(True), d["query"].clone().requires_grad_(True)
        y = f(x, q)
        results.append((y.detach(),) + torch.autograd.grad(y, [x, q] + list(norm.parameters()) + list(layer.parameters()), g))
    _close(*results)
