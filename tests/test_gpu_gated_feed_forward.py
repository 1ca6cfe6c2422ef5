"""The gated feed-forward block and its gradients, against the definition in 64 bits."""
import pytest
import torch

import ffn_reference as ref

pytestmark = pytest.mark.gpu
TYPES = (torch.bfloat16, torch.float16)
NAMES = ("x", "wg", "wu", "wd", "bg", "bu", "bd")


def make(rows, E, F, N, dtype, bias=True, residual=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    out = torch.float32 if residual == "wide" else dtype
    d = dict(x=n(rows, E).to(dtype), wg=(n(F, E) * E ** -0.5).to(dtype), wu=(n(F, E) * E ** -0.5).to(dtype),
             wd=(n(N, F) * F ** -0.5).to(dtype), g=n(rows, N).to(out))
    for k, m in (("bg", F), ("bu", F), ("bd", N)):
        d[k] = (0.3 * n(m)).to(dtype) if bias else None
    d["r"] = "x" if residual == "x" else None if residual is None else n(rows, N).to(out)
    return d


def run(d, act, checkpoint=None):
    import dfa3d_b200 as M
    leaves = {k: d[k].clone().requires_grad_(True) for k in NAMES + ("r",) if torch.is_tensor(d[k])}
    r = leaves["x"] if d["r"] == "x" else leaves.get("r")
    y = M.gated_feed_forward(*(leaves.get(k) for k in NAMES), activation=act, residual=r, checkpoint=checkpoint)
    return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), d["g"])))


def check(d, act, checkpoint=None):
    y, grads = run(d, act, checkpoint)
    kept = None if checkpoint is None else ref.stands_for(d["x"], checkpoint)
    plus_x = d["r"] == "x" if isinstance(d["r"], str) else False
    q = ref.gated(*(d[k] for k in NAMES), act, None if plus_x else d["r"], d["g"], kept, plus_x)
    assert y.dtype == d["g"].dtype
    ref.near("y", y, q[0])
    for k, pair in zip(NAMES, q[1:]):
        if k in grads:
            assert grads[k].dtype == d["x"].dtype
            ref.near("grad_" + k, grads[k], pair)
    if "r" in grads:
        assert torch.equal(grads["r"], d["g"])


SIZES = [(1, 1, 1, 1), (1, 8, 8, 8), (5, 7, 3, 9), (33, 64, 64, 64), (129, 65, 63, 66), (128, 128, 128, 128), (200, 90, 250, 90),
         (257, 256, 136, 256), (300, 300, 72, 100), (130, 72, 520, 40), (200, 300, 72, 310), (200, 330, 140, 700), (140, 64, 60, 600)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,E,F,N", SIZES)
def test_sizes(rows, E, F, N, dtype):
    check(make(rows, E, F, N, dtype, seed=rows), "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", None])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("residual", [None, "x", "same", "wide"])
def test_forms(act, bias, residual, dtype):
    check(make(150, 96, 200, 96, dtype, bias, residual, seed=1), act)


@pytest.mark.parametrize("residual", ["x", "wide"])
def test_odd_residuals(residual):
    check(make(150, 91, 57, 91, torch.float16, True, residual, seed=2), "gelu")


@pytest.mark.parametrize("checkpoint", ["int8", "e4m3"])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("E", [96, 59])
def test_checkpoints(checkpoint, act, E):
    check(make(200, E, 136, E, torch.bfloat16, residual="x", seed=3), act, checkpoint)


@pytest.mark.parametrize("rows,E,F", [(20000, 256, 512), (10001, 256, 200), (12000, 128, 1024), (9000, 512, 256)])
def test_many_tiles(rows, E, F):
    check(make(rows, E, F, E, torch.bfloat16, residual="x", seed=4), "gelu")


def test_no_rows_and_shapes():
    import dfa3d_b200 as M
    d = make(0, 16, 24, 16, torch.float16, seed=5)
    y, grads = run(d, "silu")
    assert y.shape == (0, 16) and all((grads[k] == 0).all() for k in NAMES[1:])
    d = make(24, 16, 40, 16, torch.float16, residual="x", seed=6)
    flat, _ = run(d, "silu")
    x = d["x"].view(2, 3, 4, 16)
    assert torch.equal(M.gated_feed_forward(x, *(d[k] for k in NAMES[1:]), residual=x).view(24, 16), flat)


@pytest.mark.parametrize("frozen", ["x", "wg", "wu", "wd", "bg", "bu", "bd", "x wg bg", "wg wu wd bg bu bd", "x wg wu wd", "wg bu bd"])
def test_frozen_inputs(frozen):
    import dfa3d_b200 as M
    frozen = frozen.split()
    d = make(100, 40, 48, 40, torch.bfloat16, residual="same", seed=7)
    _, want = run(d, "gelu")
    leaves = {k: d[k].clone().requires_grad_(k not in frozen) for k in NAMES + ("r",)}
    M.gated_feed_forward(*(leaves[k] for k in NAMES), activation="gelu", residual=leaves["r"]).backward(d["g"])
    for k, t in leaves.items():
        assert (t.grad is None) == (k in frozen)
        if k not in frozen:
            assert torch.equal(t.grad, want[k])


def test_some_biases():
    for there in (("bg",), ("bu", "bd"), ("bd",)):
        d = make(100, 40, 48, 40, torch.bfloat16, residual="same", seed=8)
        for k in ("bg", "bu", "bd"):
            if k not in there:
                d[k] = None
        check(d, "silu")


def test_residual_that_is_x_is_a_residual_like_any_other():
    d = make(200, 64, 96, 64, torch.bfloat16, residual="x", seed=9)
    y, grads = run(d, "silu")
    e = dict(d, r=d["x"])
    y2, grads2 = run(e, "silu")
    assert torch.equal(y, y2)
    both = grads2["x"].double() + grads2["r"].double()
    # two roundings against one
    assert ((grads["x"].double() - both).abs() <= 2 ** -7 * (both.abs() + grads2["x"].double().abs())).all()


def test_same_bits_in_every_run():
    d = make(3000, 256, 512, 256, torch.bfloat16, residual="x", seed=10)
    y, grads = run(d, "silu", "e4m3")
    for _ in range(3):
        y2, grads2 = run(d, "silu", "e4m3")
        assert torch.equal(y, y2) and all(torch.equal(grads[k], grads2[k]) for k in grads)


def test_not_a_number_stays_in_its_rows():
    d = make(300, 64, 96, 64, torch.bfloat16, residual="x", seed=11)
    d["x"][7, 3] = float("nan")
    y, grads = run(d, "silu")
    bad = ~torch.isfinite(y).all(1)
    assert bad[7] and int(bad.sum()) == 1
    rows = torch.arange(300, device="cuda") != 7
    assert torch.isfinite(grads["x"][rows]).all()


ONE_KERNEL = 9473      # rows enough for the kernel that keeps the hidden rows on the SMs (37 of 74 pairs with 256 rows each), one more


@pytest.mark.parametrize("E,F,N", [(256, 512, 256), (256, 130, 256), (64, 128, 64), (8, 8, 8), (200, 72, 136), (136, 1000, 24), (96, 200, 248)])
@pytest.mark.parametrize("residual", [None, "same", "wide"])
def test_hidden_rows_that_stay_on_the_sms(lib_built, E, F, N, residual):
    from dfa3d_b200 import _lib
    assert _lib.load().dfa3d_gated_block_supported(_lib.DTYPE_F32, ONE_KERNEL, E, F, N)
    d = make(ONE_KERNEL, E, F, N, torch.bfloat16, residual=residual, seed=12)
    check(d, "gelu")


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", None])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [True, False])
def test_one_kernel_and_two_give_the_same_bits(lib_built, act, dtype, bias):
    """Many rows with one kernel, few with two: a row's result depends on the row alone."""
    import dfa3d_b200 as M
    from dfa3d_b200 import _lib
    d = make(40001, 128, 330, 128, dtype, bias=bias, residual="wide", seed=13)
    assert not _lib.load().dfa3d_gated_block_supported(_lib.DTYPE_F32, 9000, 128, 330, 128)
    f = lambda rows: M.gated_feed_forward(d["x"][rows], *(d[k] for k in NAMES[1:]), activation=act, residual=d["r"][rows])
    whole = f(slice(None))
    for first in range(0, 40001, 9000):
        rows = slice(first, min(first + 9000, 40001))
        assert torch.equal(whole[rows], f(rows))


def test_one_kernel_on_two_streams_and_with_no_numbers(lib_built):
    import dfa3d_b200 as M
    jobs = [make(20000, 256, 256, 256, torch.bfloat16, residual="x", seed=s) for s in (14, 15)]
    f = lambda d: M.gated_feed_forward(*(d[k] for k in NAMES), residual=d["x"])
    want = [f(d) for d in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(f(jobs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
    jobs[0]["x"][777, 5] = float("nan")
    bad = ~torch.isfinite(f(jobs[0])).all(1)
    assert bad[777] and int(bad.sum()) == 1


@pytest.mark.parametrize("case", ["residual", "x", "weights"])
def test_one_kernel_and_storage_off_the_grid(lib_built, case):
    import dfa3d_b200 as M
    d = make(ONE_KERNEL, 64, 96, 64, torch.bfloat16, residual="same", seed=16)
    f = lambda e: M.gated_feed_forward(*(e[k] for k in NAMES), residual=e["r"])
    want = f(d)
    off = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view_as(t).copy_(t)
    moved = {"residual": ("r",), "x": ("x",), "weights": NAMES[1:]}[case]
    assert torch.equal(f(dict(d, **{k: off(d[k]) for k in moved})), want)
