"""act(x W^T + b) + residual and its gradients, against the definition in 64 bits."""
import pytest
import torch

import ffn_reference as ref

pytestmark = pytest.mark.gpu
TYPES = (torch.bfloat16, torch.float16)


def make(rows, K, N, dtype, bias=True, residual=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    out = {None: dtype, "same": dtype, "wide": torch.float32}[residual]
    return dict(x=n(rows, K).to(dtype), w=(n(N, K) * K ** -0.5).to(dtype), b=(0.3 * n(N)).to(dtype) if bias else None,
                r=n(rows, N).to(out) if residual else None, g=n(rows, N).to(out))


def run(d, act, checkpoint=None):
    import dfa3d_b200 as M
    leaves = {k: d[k].clone().requires_grad_(True) for k in ("x", "w", "b", "r") if d[k] is not None}
    y = M.linear_act(leaves["x"], leaves["w"], leaves.get("b"), activation=act, residual=leaves.get("r"), checkpoint=checkpoint)
    return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), d["g"])))


def check(d, act, checkpoint=None):
    y, grads = run(d, act, checkpoint)
    kept = None if checkpoint is None else ref.stands_for(d["x"], checkpoint)
    q = ref.linear(d["x"], d["w"], d["b"], act, d["r"], d["g"], kept)
    assert y.dtype == d["g"].dtype
    ref.near("y", y, q[0])
    for k, pair in zip(("x", "w", "b"), q[1:]):
        if k in grads:
            assert grads[k].dtype == d["x"].dtype
            ref.near("grad_" + k, grads[k], pair)
    if d["r"] is not None:
        assert torch.equal(grads["r"], d["g"])


# one row and one column, sizes around 32, 64, 128 and 256, odd ones, sums of one and of more than the resident 256 elements
SIZES = [(1, 1, 1), (1, 8, 8), (3, 7, 5), (33, 64, 64), (127, 65, 63), (128, 128, 128), (129, 256, 257), (255, 264, 72), (257, 40, 130),
         (300, 512, 256), (513, 72, 520), (700, 1000, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,N", SIZES)
def test_sizes(rows, K, N, dtype):
    check(make(rows, K, N, dtype, residual="same", seed=rows), "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("residual", [None, "same", "wide"])
def test_forms(act, bias, residual, dtype):
    check(make(150, 96, 200, dtype, bias, residual, seed=1), act)


@pytest.mark.parametrize("N", [203, 100])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_wide_residual_of_odd_rows(act, N):
    check(make(150, 96, N, torch.bfloat16, True, "wide", seed=2), act)


def test_a_wide_gradient_is_rounded_once(lib_built):
    """Rows off the 16-byte grid too: the derivative is applied to 32 bits."""
    check(make(1, 256, 393, torch.bfloat16, False, "wide", seed=2368), "silu", "int8")
    check(make(7, 64, 2051, torch.float16, True, "wide", seed=3), "gelu")


@pytest.mark.parametrize("checkpoint", ["int8", "e4m3"])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("K", [96, 59])
def test_checkpoints(checkpoint, act, K):
    check(make(200, K, 136, torch.bfloat16, seed=3), act, checkpoint)


@pytest.mark.parametrize("rows,K,N", [(20000, 256, 512), (20001, 512, 256), (40000, 64, 64), (9999, 256, 192), (19000, 320, 640)])
def test_many_tiles(rows, K, N):
    """Every pair of CTAs has several tiles: rows that stay, rings and accumulators that come round again."""
    d = make(rows, K, N, torch.bfloat16, residual="wide" if K == 512 else "same", seed=4)
    check(d, "gelu")


def test_weight_gradients_of_wide_results():
    """More tiles of a weight gradient than SMs: one share of the rows each."""
    check(make(70, 2500, 1300, torch.float16, seed=5), None)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
def test_far_values(act):
    """Both tails: results neither overflow nor become NaN where the activation is 0 or the identity."""
    d = make(64, 32, 64, torch.bfloat16, seed=6)
    d["x"] = d["x"] * 300
    check(d, act)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
def test_not_a_number_stays_in_its_rows(act):
    d = make(300, 64, 96, torch.bfloat16, seed=7)
    d["x"][7, 3] = float("nan")
    d["x"][200, 60] = float("inf")
    y, grads = run(d, act)
    bad = ~torch.isfinite(y).all(1)
    assert bad[7] and bad[200] and int(bad.sum()) == 2
    assert torch.isnan(y[7]).all()
    clean = torch.ones(300, dtype=torch.bool, device="cuda")
    clean[7] = clean[200] = False
    assert torch.isfinite(grads["x"][clean]).all()


def test_no_rows_and_shapes():
    import dfa3d_b200 as M
    d = make(0, 16, 24, torch.float16, seed=8)
    y, grads = run(d, "silu")
    assert y.shape == (0, 24) and grads["x"].shape == (0, 16)
    assert (grads["w"] == 0).all() and (grads["b"] == 0).all()
    d = make(24, 16, 8, torch.float16, seed=9)
    y = M.linear_act(d["x"].view(2, 3, 4, 16), d["w"], d["b"], residual=d["g"].view(2, 3, 4, 8))
    assert y.shape == (2, 3, 4, 8)
    assert torch.equal(y.view(24, 8), M.linear_act(d["x"], d["w"], d["b"], residual=d["g"]))
    assert M.linear_act(d["x"][0], d["w"]).shape == (8,)


def test_strides_and_storage_off_the_grid():
    import dfa3d_b200 as M
    d = make(200, 64, 72, torch.bfloat16, residual="same", seed=10)
    want = M.linear_act(d["x"], d["w"], d["b"], "silu", d["r"])
    turned = d["x"].t().contiguous().t()
    off = torch.empty(d["x"].numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(d["x"]).copy_(d["x"])
    w_off = torch.empty(d["w"].numel() + 3, dtype=torch.bfloat16, device="cuda")[3:].view_as(d["w"]).copy_(d["w"])
    r_off = torch.empty(d["r"].numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(d["r"]).copy_(d["r"])
    b_off = torch.empty(73, dtype=torch.bfloat16, device="cuda")[1:].copy_(d["b"])
    for x, w, b, r in ((turned, d["w"], d["b"], d["r"]), (off, w_off, b_off, r_off), (d["x"], d["w"].t().contiguous().t(), d["b"], d["r"])):
        assert torch.equal(M.linear_act(x, w, b, "silu", r), want)
    d["x"], d["r"] = off, r_off
    d["g"] = d["g"][:1].expand(200, 72)          # a broadcast gradient
    check(d, "silu")


@pytest.mark.parametrize("frozen", ["x", "w", "b", "r", "xw", "xb", "wb", "xwb"])
def test_frozen_inputs(frozen):
    import dfa3d_b200 as M
    d = make(100, 40, 48, torch.bfloat16, residual="same", seed=11)
    _, want = run(d, "gelu")
    leaves = {k: d[k].clone().requires_grad_(k not in frozen) for k in "xwbr"}
    y = M.linear_act(leaves["x"], leaves["w"], leaves["b"], "gelu", leaves["r"])
    y.backward(d["g"])
    for k, t in leaves.items():
        assert (t.grad is None) == (k in frozen)
        if k not in frozen:
            assert torch.equal(t.grad, want[k])


@pytest.mark.parametrize("bias", [True, False])
def test_only_the_residual_is_trained(bias):
    import dfa3d_b200 as M
    d = make(100, 40, 48, torch.bfloat16, bias, "same", seed=12)
    d["r"].requires_grad_(True)
    M.linear_act(d["x"], d["w"], d["b"], "gelu", d["r"]).backward(d["g"])
    assert torch.equal(d["r"].grad, d["g"])


def test_same_bits_in_every_run_and_row_by_row():
    """A row's result depends on the row alone, whatever it is computed with."""
    import dfa3d_b200 as M
    d = make(3000, 256, 512, torch.bfloat16, seed=13)
    y, grads = run(d, "silu")
    for _ in range(3):
        y2, grads2 = run(d, "silu")
        assert torch.equal(y, y2) and all(torch.equal(grads[k], grads2[k]) for k in grads)
    part = M.linear_act(d["x"][1000:1100], d["w"], d["b"], "silu")
    assert torch.equal(part, y[1000:1100])


def test_differences():
    """Gradients against differences of the operator itself, in a direction."""
    import dfa3d_b200 as M
    d = make(64, 48, 40, torch.float16, residual="wide", seed=14)
    for act in ("silu", "gelu"):
        _, grads = run(d, act)
        for k in ("x", "w", "b"):
            step = torch.randn_like(d[k], dtype=torch.float32) * 0.05
            hi, lo = dict(d), dict(d)
            hi[k], lo[k] = (d[k] + step).half(), (d[k] - step).half()
            f = lambda e: (M.linear_act(e["x"], e["w"], e["b"], act, e["r"]).double() * d["g"].double()).sum()
            slope = (grads[k].double() * (hi[k].double() - lo[k].double())).sum()
            # rounding of the gradient: 2^-11 of its terms; curvature: third order in the step
            bound = 3e-3 * (grads[k].double().abs() * (hi[k].double() - lo[k].double()).abs()).sum()
            assert abs(f(hi) - f(lo) - slope) <= bound


def test_past_two_to_the_31_elements():
    """The last rows of x and y lie beyond 32-bit offsets."""
    import dfa3d_b200 as M
    rows, K, N = (1 << 25) + 259, 64, 72              # 2.1e9 and 2.4e9 elements, 4.3 and 4.8 GB
    d = make(300, K, N, torch.bfloat16, seed=15)
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device="cuda")
    x[:300], x[-300:] = d["x"], d["x"]
    want = M.linear_act(d["x"], d["w"], d["b"], "gelu")
    y = M.linear_act(x, d["w"], d["b"], "gelu")
    assert torch.equal(y[:300], want) and torch.equal(y[-300:], want)
    assert torch.equal(y[300:400], M.linear_act(x[300:400], d["w"], d["b"], "gelu"))
