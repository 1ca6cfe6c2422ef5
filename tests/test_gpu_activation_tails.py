"""The activations of the feed-forward products element by element, at every 16-bit number: what a 16-bit result holds far out in a tail is
the activation's value there, not a number of the same smallness.

z passes through a product with the identity, exactly; with a float32 residual of zeros the activation is seen in 32 bits.

Bounds, relative, with U = 2^-24 the rounding of one operation.  SiLU, z e^z / (1 + e^z): the exponent's argument is off by 2 U |A|,
A = z log2 e, which moves e^z by ln 2 times as much, 2 U |z|; exponential 2^-22, reciprocal 2^-23, six roundings: below 2^-20 in all.
GELU, z P(X <= z), for z < 0 a factor exp(-z^2 / 2) whose argument is off by 3 U |A|, A = z^2 / 2 log2 e: 1.5 U z^2; a polynomial
that is fitted to 2^-18, nine of its terms' roundings, exponential and reciprocal as above: below 2^-17.  Results below 2^-118 come from
an exponential that ends at 2^-126."""
import math

import pytest
import torch

from row_reference import assert_within, half_step, tiny

pytestmark = pytest.mark.gpu
TYPES = (torch.bfloat16, torch.float16)
U = 2.0 ** -24
END = 2.0 ** -118


def numbers(dtype, most):
    """Every number of the type up to `most`, (rows, 8)."""
    z = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32, device="cuda").to(torch.int16).view(dtype)
    z = z[torch.isfinite(z) & (z.abs() <= most)]
    return z[:z.numel() // 8 * 8].view(-1, 8).contiguous()


def definition(z, act):
    """Value, derivative, and the bounds of both."""
    v = z.double()
    if act == "silu":
        s, far = torch.sigmoid(v), 1 / (1 + torch.exp(v))          # far = 1 - s
        a, d = v * s, s * (1 + v * far)
        rel = 2.0 ** -20 + 2 * U * v.abs()
        # the derivative's 1 - s is off by what s is off by
        return a, d, rel * a.abs() + END, rel * (s + a.abs() * far) + a.abs() * 2.0 ** -21 + END
    p = 0.5 * torch.special.erfc(-v / math.sqrt(2))
    bell = v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    rel = 2.0 ** -17 + 1.5 * U * v * v
    # on the positive side it is 1 - P(X <= -z)
    off = rel * 0.5 * torch.special.erfc(v.abs() / math.sqrt(2)) + torch.where(v > 0, 2.0 ** -23, 0.0)
    return v * p, p + bell, v.abs() * off + 2 * U * (v * p).abs() + END, off + (rel + 2.0 ** -20) * bell.abs() + 2 * U + END


def run(z, act, wide):
    import dfa3d_b200 as M
    x = z.clone().requires_grad_(True)
    one = torch.eye(8, device="cuda").to(z.dtype)
    r = torch.zeros(z.shape, device="cuda") if wide else None
    y = M.linear_act(x, one, activation=act, residual=r)
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    return y.detach(), g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act,most", [("silu", 300.0), ("gelu", 40.0)])
def test_every_number(lib_built, dtype, act, most):
    z = numbers(dtype, most)
    a, d, ea, ed = definition(z, act)
    y, g = run(z, act, True)
    assert y.dtype == torch.float32
    assert_within("y", y, a.cpu(), ea.cpu())
    stored = lambda v, e: (e + half_step(dtype) * (v.abs() + e) + tiny(dtype)).cpu()
    assert_within("slope", g, d.cpu(), stored(d, ed))
    y, _ = run(z, act, False)
    assert_within("16-bit y", y, a.cpu(), stored(a, ea))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_far_on_the_negative_side_nothing_is_left(lib_built, act):
    """Where the value is below what 32 bits hold it is 0."""
    z = -torch.logspace(2.5, 30, 64, device="cuda").bfloat16().view(8, 8)
    y, g = run(z, act, True)
    assert (y == 0).all() and (g == 0).all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gate_times_large_up(lib_built, act):
    """A gate far out in the tail closes whatever it stands before: act(gate) up is right relative to itself."""
    import dfa3d_b200 as M
    z = torch.linspace(-70, -1, 64, device="cuda").bfloat16().view(8, 8)
    up = torch.full((8, 1), 2.0 ** 40, device="cuda").bfloat16()
    x = torch.cat([z, up, torch.zeros(8, 7, device="cuda").bfloat16()], 1)
    eye = torch.eye(8, device="cuda")
    gate = torch.cat([eye, torch.zeros(8, 8, device="cuda")], 1).bfloat16()
    ups = torch.zeros(8, 16, device="cuda").bfloat16()
    ups[:, 8] = 1
    y = M.gated_feed_forward(x, gate, ups, eye.bfloat16(), activation=act)
    a, _, ea, _ = definition(z, act)
    want = a * 2.0 ** 40
    e = ea * 2.0 ** 40
    e = e + half_step(torch.bfloat16) * (want.abs() + e)          # the hidden row is rounded, then passes the identity
    assert_within("y", y, want.cpu(), (e + tiny(torch.bfloat16)).cpu())
