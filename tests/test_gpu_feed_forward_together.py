"""The feed-forward operators as programs run them: refusals on the device, both host paths, streams, graphs, hooks, autocast, 8-bit
checkpoints and their memory, a run of all of them, encoder layers with the gated block."""
import pytest
import torch

import dfa3d_b200 as M
import ffn_reference as ref
import test_gpu_counter_dropout_modules as layers
from dfa3d_b200 import modules
from dfa3d_b200.feed_forward_ops import GatedFeedForwardFunction, LinearActFunction
from test_gpu_native_path import _python

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
KINDS = ["linear", "linear none", "linear wide", "linear int8", "gated", "gated x", "gated e4m3"]


def call(kind, native=True, rows=70, E=40, F=56, dtype=torch.bfloat16, seed=1):
    """A function of no arguments that runs the forward, and its leaves."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV).requires_grad_(True)
    x, wg, wu, wd, bg, bu, bd = n(rows, E), n(F, E), n(F, E), n(E, F), n(F), n(F), n(E)
    r = torch.randn(rows, F, generator=g).to(DEV).requires_grad_(True)
    linear, gated = (f if native else _python(f) for f in (LinearActFunction, GatedFeedForwardFunction))
    all7 = [x, wg, wu, wd, bg, bu, bd]
    return {
        "linear": (lambda: linear.apply(x, wg, bg, None, "silu", None), [x, wg, bg]),
        "linear none": (lambda: linear.apply(x, wg, None, None, None, None), [x, wg]),
        "linear wide": (lambda: linear.apply(x, wg, bg, r, "gelu", None), [x, wg, bg, r]),
        "linear int8": (lambda: linear.apply(x, wg, bg, r, "gelu", "int8"), [x, wg, bg, r]),
        "gated": (lambda: gated.apply(*all7, None, False, "silu", None), all7),
        "gated x": (lambda: gated.apply(*all7, None, True, "gelu", None), all7),
        "gated e4m3": (lambda: gated.apply(x, wg, wu, wd, None, None, None, None, True, "relu", "e4m3"), all7[:4]),
    }[kind]


def grads_of(f, leaves, go=None):
    y = f()
    if go is None:
        go = torch.randn(y.shape, generator=torch.Generator().manual_seed(9)).to(y.dtype).to(DEV)
    return (y.detach(),) + torch.autograd.grad(y, leaves, go)


def equal(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,E,F", [(70, 40, 56), (33, 37, 51)])
def test_both_host_paths_give_the_same_bits(lib_built, kind, rows, E, F):
    assert equal(grads_of(*call(kind, True, rows, E, F)), grads_of(*call(kind, False, rows, E, F)))


def test_the_native_path_takes_the_plain_calls(lib_built):
    for kind in KINDS:
        y = call(kind)[0]()
        assert "Backward" not in y.grad_fn.name() or "Fn" in y.grad_fn.name(), y.grad_fn.name()


@BOTH
@pytest.mark.parametrize("kind", KINDS)
def test_hooks(lib_built, kind, native):
    f, leaves = call(kind, native)
    want = grads_of(f, leaves)
    for pack, unpack in ((lambda t: t.cpu(), lambda t: t.to(DEV)),
                         (lambda t: t.clone(), lambda t: t.transpose(0, -1).contiguous().transpose(0, -1))):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = f()
        go = torch.randn(y.shape, generator=torch.Generator().manual_seed(9)).to(y.dtype).to(DEV)
        assert equal(torch.autograd.grad(y, leaves, go), want[1:])
    for pack in (lambda t: t.float() if t.is_floating_point() else t.int(), lambda t: t.flatten()[1:].clone()):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = f()
        with pytest.raises(RuntimeError, match="saved-tensor hook"):
            torch.autograd.grad(y, leaves, torch.ones_like(y))


@BOTH
@pytest.mark.parametrize("kind", KINDS)
def test_no_second_derivative(lib_built, kind, native):
    f, leaves = call(kind, native)
    y = f()
    go = torch.ones_like(y).requires_grad_(True)
    g = torch.autograd.grad(y, leaves[0], go, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.float().sum().backward()


@pytest.mark.parametrize("kind", KINDS)
def test_inputs_changed_before_the_backward_are_noticed(lib_built, kind):
    if kind.endswith(("int8", "e4m3")):
        pytest.skip("keeps a copy in 8 bits")
    f, leaves = call(kind)
    y = f()
    with torch.no_grad():
        leaves[0].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


@pytest.mark.parametrize("kind", KINDS)
def test_two_streams_at_once(lib_built, kind):
    """Calls that run beside each other share nothing."""
    jobs = [call(kind, rows=5000, E=136, F=264, seed=s) for s in (1, 2)]
    want = [grads_of(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, (s, j) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(s):
                got[i].append(grads_of(*j))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("kind", KINDS)
def test_captured_and_replayed(lib_built, kind):
    """Two graphs of the same call, replayed in turn on other inputs."""
    f, leaves = call(kind, rows=300, E=72, F=96)
    go = torch.randn(f().shape, generator=torch.Generator().manual_seed(9)).to(DEV)
    go = go.to(f().dtype)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            grads_of(f, leaves, go)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = grads_of(f, leaves, go)
        graphs.append((g, out))
    for factor in (1.0, 0.5, 2.0):
        with torch.no_grad():
            leaves[0].mul_(factor)
        for g, _ in graphs:
            g.replay()
        want = grads_of(f, leaves, go)
        for _, out in graphs:
            assert equal(out, want)


def test_inference_mode(lib_built):
    for kind in KINDS:
        f, leaves = call(kind)
        want = f().detach()
        with torch.inference_mode():
            assert torch.equal(f(), want)
        with torch.no_grad():
            assert torch.equal(f(), want)


def test_refusals_on_the_device(lib_built):
    x, w, b = torch.randn(4, 16, device=DEV).bfloat16(), torch.randn(24, 16, device=DEV).bfloat16(), torch.randn(24, device=DEV).bfloat16()
    wd = torch.randn(16, 24, device=DEV).bfloat16()
    for bad in (lambda: M.linear_act(x.float(), w, b), lambda: M.linear_act(x, w.float(), b), lambda: M.linear_act(x, w.half(), b),
                lambda: M.linear_act(x, w[:, :8], b), lambda: M.linear_act(x, w, b[:8]), lambda: M.linear_act(x, w, b.float()),
                lambda: M.linear_act(x, w.cpu(), b), lambda: M.linear_act(x, w, b, residual=x),
                lambda: M.linear_act(x, w, b, residual=torch.zeros(4, 24, device=DEV).half()),
                lambda: M.linear_act(x, w, b, residual=torch.zeros(1, 24, device=DEV)), lambda: M.linear_act(x[:, :0], w[:, :0]),
                lambda: M.linear_act(x, w[:0], b[:0]),
                lambda: M.gated_feed_forward(x, w, w[:8], wd), lambda: M.gated_feed_forward(x, w, w, wd[:, :8]),
                lambda: M.gated_feed_forward(x, w, w, wd, b, b[:8]), lambda: M.gated_feed_forward(x, w, w, wd[:8], residual=x),
                lambda: M.gated_feed_forward(x, w, w, wd.float()), lambda: M.gated_feed_forward(x, w[:0], w[:0], wd[:, :0]),
                lambda: M.decompress8(M.compress8(x)._replace(shape=torch.Size((8, 16)))),
                lambda: M.decompress8(M.compress8(x)._replace(scales=torch.zeros(4, 2, dtype=torch.uint8, device=DEV)))):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: M.linear_act(x, w, b, activation="tanh"), lambda: M.linear_act(x, w, b, checkpoint="int4"),
                lambda: M.gated_feed_forward(x, w, w, wd, activation="swish"), lambda: M.compress8(x, "e5m2")):
        with pytest.raises(ValueError):
            bad()


def test_a_checkpoint_keeps_half(lib_built):
    """Memory between forward and backward: the input in 16 bits, or 33 / 32 bytes an element."""
    rows, E = 8192, 256
    w = torch.randn(64, E, device=DEV).bfloat16().requires_grad_(True)
    held = {}
    for name, fmt in (("whole", None), ("int8", "int8")):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = M.linear_act(torch.randn(rows, E, device=DEV).bfloat16(), w, checkpoint=fmt)
        held[name] = torch.cuda.memory_allocated() - before - y.numel() * 2
        del y
    assert held["whole"] >= rows * E * 2 and held["int8"] <= rows * E * 33 // 32 + 4096


def test_under_autocast(lib_built):
    x = torch.randn(100, 64, device=DEV, requires_grad=True)
    layer = M.LinearAct(64, 48, activation="gelu").to(DEV)
    block = M.GatedFeedForward(48, 80, checkpoint="int8").to(DEV)
    for dt in (torch.bfloat16, torch.float16):
        with torch.autocast("cuda", dtype=dt):
            h = layer(x)
            assert h.dtype == dt
            y = block(h, h)
            assert y.dtype == dt
            stream = block(x[:, :48], x[:, :48])
            assert stream.dtype == torch.float32
        (y.float().sum() + stream.sum()).backward()
        assert all(p.grad is not None and p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all()
                   for p in list(layer.parameters()) + list(block.parameters()))
    want = M.linear_act(x.detach().half(), layer.weight.detach().half(), layer.bias.detach().half(), "gelu")
    assert torch.equal(h, want)


@pytest.mark.parametrize("checkpoint", [None, "int8", "e4m3"])
def test_a_run_of_them(lib_built, checkpoint):
    """Projection -> gated block with a 32-bit residual stream -> product back, as a model runs them, against the definition."""
    g = torch.Generator(device=DEV).manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g, device=DEV)
    rows, E, F, N = 400, 64, 120, 40
    x = n(rows, E).bfloat16()
    w = {k: (n(*s) * s[1] ** -0.5).bfloat16().requires_grad_(True) for k, s in dict(a=(E, E), g=(F, E), u=(F, E), d=(E, F), o=(N, E)).items()}
    go = n(rows, N).bfloat16()
    stream = M.linear_act(x, w["a"], activation="silu", residual=x.float(), checkpoint=checkpoint)
    assert stream.dtype == torch.float32
    stream.retain_grad()
    narrow = stream.bfloat16()
    narrow.retain_grad()
    more = M.gated_feed_forward(narrow, w["g"], w["u"], w["d"], residual=stream, checkpoint=checkpoint)
    y = M.linear_act(more.bfloat16(), w["o"], checkpoint=checkpoint)
    y.backward(go)
    keep = lambda t: None if checkpoint is None else ref.stands_for(t.detach(), checkpoint)
    # each operator by itself, on what it was given
    zero = torch.zeros(rows, E, device=DEV)
    ref.near("stream", stream, ref.linear(x, w["a"], None, "silu", x.float(), zero, keep(x))[0])
    top = ref.linear(more.detach().bfloat16(), w["o"], None, None, None, go, keep(more.detach().bfloat16()))
    ref.near("y", y, top[0])
    ref.near("grad o", w["o"].grad, top[2])
    into = (go.double() @ w["o"].detach().double()).bfloat16()          # the gradient that reached the block, as it was rounded
    mid = ref.gated(narrow.detach(), w["g"], w["u"], w["d"], None, None, None, "silu", stream.detach(), into.float(), keep(narrow))
    ref.near("more", more, mid[0])
    # `into` is a rounding of the exact product, the kernel's of its 32-bit sum: one step of bfloat16 apart where that lies on a border
    for k, q in zip("gud", mid[2:5]):
        got = w[k].grad.double()
        assert ((got - q[0]).norm() <= 0.01 * q[0].norm()).item(), k
    assert torch.isfinite(w["a"].grad).all() and (w["a"].grad != 0).any()


def _layer(kind, **kw):
    torch.manual_seed(3)
    cls = {"cross": modules.SCAEncoderLayer, "full": modules.BEVFormerEncoderLayer}[kind]
    size = dict(bev_h=5, bev_w=10) if kind == "full" else {}
    layer = cls(32, 64, 3, 2, 2, 8, **size, **kw).to(DEV)
    return layer


@pytest.mark.parametrize("kind", ["cross", "full"])
@pytest.mark.parametrize("options", [True, dict(activation="gelu", checkpoint="int8"), dict(compute_dtype=torch.float16, bias=False)])
def test_layers_with_the_gated_block(lib_built, kind, options):
    """The layer is its parts: attention and norms as before, the block on the operator, a float32 stream that is not rounded."""
    layer, d = _layer(kind, dropout=0.0, gated_feed_forward=options), layers._inputs(6)
    kw = {k: d[k] for k in layers.KEYS}
    seen = []
    hook = layer.norm1.register_forward_hook(lambda m, a, out: seen.append(out))
    got = layer(d["query"], **kw)
    hook.remove()
    x = seen[0].detach()
    dt = layer.ffn.compute_dtype
    p = lambda m: None if m is None else m.detach().to(dt)
    f = layer.ffn
    want = layer.norm2(M.gated_feed_forward(x.to(dt), p(f.gate.weight), p(f.up.weight), p(f.down.weight), p(f.gate.bias), p(f.up.bias),
                                            p(f.down.bias), f.activation, residual=x))
    assert got.dtype == torch.float32 and torch.equal(got, want)
    got.sum().backward()
    assert all(q.grad is not None and torch.isfinite(q.grad).all() for q in f.parameters())
    assert set(layer.state_dict()) >= {"ffn.gate.weight", "ffn.up.weight", "ffn.down.weight"}


@pytest.mark.parametrize("counter", [False, True])
def test_layers_with_the_gated_block_and_dropout(lib_built, counter):
    layer, d = _layer("cross", dropout=0.2, counter_dropout=counter, gated_feed_forward=True), layers._inputs(6)
    kw = {k: d[k] for k in layers.KEYS}
    outs = []
    for s in (1, 1, 2):
        torch.manual_seed(s)
        y = layer(d["query"], **kw)
        outs.append(y.detach())
    assert torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], outs[2])
    y.sum().backward()
    assert all(torch.isfinite(q.grad).all() for q in layer.ffn.parameters())
    layer.eval()
    assert torch.equal(layer(d["query"], **kw), layer(d["query"], **kw))


def test_activation_checkpoints_of_a_layer(lib_built):
    from torch.utils.checkpoint import checkpoint
    layer, d = _layer("cross", dropout=0.0, gated_feed_forward=dict(checkpoint="e4m3")), layers._inputs(6)
    kw = {k: d[k] for k in layers.KEYS}
    results = []
    for f in (lambda q: layer(q, **kw), lambda q: checkpoint(lambda t: layer(t, **kw), q, use_reentrant=False)):
        q = d["query"].clone().requires_grad_(True)
        y = f(q)
        results.append(torch.autograd.grad(y, [layer.ffn.gate.weight, layer.ffn.down.bias], torch.ones_like(y)))
    # the rest of the layer adds up in an order that is not fixed
    for a, b in zip(*results):
        torch.testing.assert_close(a, b, rtol=2e-2, atol=2e-2 * float(b.abs().max()))


@pytest.mark.parametrize("kind", KINDS)
def test_captured_behind_a_join(lib_built, kind):
    """The kernels may begin before the one in front of them ends: not before either of two that they follow."""
    f, leaves = call(kind, rows=3000, E=136, F=200)
    go = torch.randn(f().shape, generator=torch.Generator().manual_seed(9)).to(DEV).to(f().dtype)
    base = [t.detach().clone() for t in leaves]
    side = torch.cuda.Stream()

    def run():
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.no_grad():
            leaves[0].copy_(base[0] * 2 - base[0])                      # what the call reads, written on both streams
            with torch.cuda.stream(side):
                for t, b in zip(leaves[1:], base[1:]):
                    t.copy_(b * 2 - b)
        here.wait_stream(side)
        out = grads_of(f, leaves, go)
        with torch.no_grad():
            for t in leaves:                                            # behind it: the call has read all of it
                t.fill_(float("nan"))
        return out

    want = run()
    with torch.no_grad():
        for t, b in zip(leaves, base):
            t.copy_(b)
    assert equal(want, grads_of(f, leaves, go))
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        run()
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(5):
        graph.replay()
        assert equal(out, want)


@BOTH
def test_shared_and_broadcast_inputs(lib_built, native):
    """One tensor in several places, and rows that are one row: gradients add up."""
    g = torch.Generator().manual_seed(4)
    n = lambda *s: torch.randn(*s, generator=g).bfloat16().to(DEV)
    row, w, wd, b, go = n(1, 40), n(56, 40), n(40, 56), n(56), n(70, 40)
    linear, gated = (f if native else _python(f) for f in (LinearActFunction, GatedFeedForwardFunction))
    leaves = [t.clone().requires_grad_(True) for t in (row, w, wd, b)]
    x = leaves[0].expand(70, 40)
    y = gated.apply(x, leaves[1], leaves[1], leaves[2], leaves[3], leaves[3], None, x, False, "silu", None)
    got = torch.autograd.grad(y, leaves, go)
    apart = [t.clone().requires_grad_(True) for t in (row.expand(70, 40), w, w, wd, b, b, row.expand(70, 40))]
    z = gated.apply(*apart[:6], None, apart[6], False, "silu", None)
    each = torch.autograd.grad(z, apart, go)
    assert torch.equal(y, z)
    # two gradients added once in 16 bits; 140 of them added up in 32 and rounded once (2^-8 each, the second of what the first
    # has rounded)
    assert torch.equal(got[1], each[1] + each[2]) and torch.equal(got[2], each[3]) and torch.equal(got[3], each[4] + each[5])
    total = each[0].double() + each[6].double()
    assert ((got[0].double() - total.sum(0)).abs() <= 1.01 * 2 ** -8 * (total.abs().sum(0) + total.sum(0).abs())).all()
    square = n(64, 64).requires_grad_(True)
    y = linear.apply(square, square, None, square, "gelu", None)
    go = n(64, 64)
    got, = torch.autograd.grad(y, square, go)
    three = [square.detach().clone().requires_grad_(True) for _ in range(3)]
    each = torch.autograd.grad(linear.apply(three[0], three[1], None, three[2], "gelu", None), three, go)
    total = sum(t.double() for t in each)
    # two sums in 16 bits, half a step each of at most the terms' magnitudes
    assert ((got.double() - total).abs() <= 1.01 * 2 * 2 ** -8 * sum(t.double().abs() for t in each)).all()
