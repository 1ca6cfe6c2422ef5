"""The feed-forward operators by their definitions in 64 bits, with a bound of how far a computation of 16-bit products, 32-bit sums
and one rounding at the end of a kernel may be from them.

A quantity is a pair (value, error bound).  Products of 16-bit numbers are exact in 32 bits; a sum of n of them in any order, each
addition off by at most 2^-23 relative (a tensor core may cut where the standard rounds: half a step more), is off by at most
n 2^-23 times the sum of the magnitudes.  Exponential and reciprocal are off by 2^-22 and 2^-23 relative, the polynomial behind GELU by
1.5e-7 of the bell curve; four such operations in a row are below `ACT` relative to the result plus 2e-7 |z|.
`half_step(dtype)` is the rounding of a result to its type, `tiny(dtype)` what a result near 0 is off by at least."""
import math

import torch

from row_reference import assert_within, half_step, tiny  # noqa: F401

STEP = 2.0 ** -23
ACT = 2.0 ** -19


def wide(t):
    return None if t is None else t.detach().double()


def exactly(t):
    t = wide(t)
    return t, torch.zeros_like(t)


def rounded(q, dtype):
    """A result that is stored."""
    v, e = q
    return v, e + half_step(dtype) * (v.abs() + e) + tiny(dtype)


def product(a, b):
    """a (m, k) @ b (k, n) of pairs."""
    (x, ex), (y, ey) = a, b
    size = (x.abs() + ex) @ (y.abs() + ey)
    return x @ y, ex @ (y.abs() + ey) + x.abs() @ ey + (x.shape[1] + 2) * STEP * size


def plus(a, b):
    if b is None:
        return a
    v = a[0] + b[0]
    e = a[1] + b[1]
    return v, e + STEP * (v.abs() + e)


def times(a, b):
    (x, ex), (y, ey) = a, b
    v = x * y
    e = ex * (y.abs() + ey) + x.abs() * ey
    return v, e + STEP * (v.abs() + e)


def transposed(q):
    return q[0].t(), q[1].t()


def act(z, name):
    """act(z) and its derivative.  Both change by at most 1.13 and 1 times what z changes by, but for the ReLU's derivative."""
    v, e = z
    if name is None:
        return z, (torch.ones_like(v), torch.zeros_like(v))
    if name == "relu":
        return (v.clamp(min=0), e), ((v > 0).double(), (v.abs() <= e).double())
    if name == "silu":
        s = torch.sigmoid(v)
        a, d = v * s, s * (1 + v * (1 - s))
    else:
        p = 0.5 * torch.special.erfc(-v / math.sqrt(2))
        a, d = v * p, p + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    return (a, 1.13 * e + ACT * a.abs() + 2e-7 * (v.abs() + e)), (d, e + ACT * (1 + v.abs()) * 0.25 + 2e-7 * (1 + v.abs()))


def linear(x, w, b, name, residual, grad, kept=None):
    """Pairs of y, grad_x, grad_w, grad_b.  kept: what the backward reads in place of x."""
    dt = x.dtype
    out = dt if residual is None else residual.dtype
    W = exactly(w)
    bias = None if b is None else exactly(b)
    z = plus(product(exactly(x), transposed(W)), bias)
    y = act(z, name)[0]
    y = rounded(plus(y, None if residual is None else exactly(residual)), out)
    X = exactly(x if kept is None else kept)
    z = plus(product(X, transposed(W)), bias)
    g = exactly(grad)
    if name is None:
        dz = rounded(g, dt) if grad.dtype == torch.float32 else g
    else:
        dz = rounded(times(g, act(z, name)[1]), dt)
    return y, rounded(product(dz, W), dt), rounded(product(transposed(dz), X), dt), rounded(column_sum(dz), dt)


def column_sum(q):
    v, e = q
    return v.sum(0), e.sum(0) + (v.shape[0] + 2) * STEP * (v.abs() + e).sum(0)


def gated(x, wg, wu, wd, bg, bu, bd, name, residual, grad, kept=None, plus_x=False):
    """Pairs of y and the gradients of x, the three weights and the three biases."""
    dt = x.dtype
    out = dt if residual is None or plus_x else residual.dtype
    G, U, D = exactly(wg), exactly(wu), exactly(wd)
    bias = [None if b is None else exactly(b) for b in (bg, bu, bd)]

    def hidden(v):
        X = exactly(v)
        a, slope = act(plus(product(X, transposed(G)), bias[0]), name)
        return X, a, slope, plus(product(X, transposed(U)), bias[1])

    _, a, _, up = hidden(x)
    h = rounded(times(a, up), dt)
    y = plus(product(h, transposed(D)), bias[2])
    y = rounded(plus(y, exactly(x) if plus_x else None if residual is None else exactly(residual)), out)
    X, a, slope, up = hidden(x if kept is None else kept)
    h = rounded(times(a, up), dt)
    g = exactly(grad)
    if grad.dtype == torch.float32:
        g = rounded(g, dt)
    through = product(g, D)
    dg, du = rounded(times(times(through, up), slope), dt), rounded(times(through, a), dt)
    gx = plus(product(dg, G), product(du, U))
    if plus_x:
        gx = plus(gx, g)
    grads = [gx, product(transposed(dg), X), product(transposed(du), X), product(transposed(g), h), column_sum(dg), column_sum(du),
             column_sum(g)]
    return [y] + [rounded(q, dt) for q in grads]


def near(name, got, q):
    """`got` is finite where the value is and within its bound; NaN and infinities are in the same places."""
    v, e = (t.cpu() for t in q)
    got = got.detach().cpu().double()
    assert got.shape == v.shape, f"{name}: {tuple(got.shape)} vs {tuple(v.shape)}"
    assert torch.isfinite(got).all(), f"{name}: {int((~torch.isfinite(got)).sum())} values are no numbers"
    assert_within(name, got, v, e)


def stands_for(x, fmt):
    """What the 8-bit checkpoint of x (rows, cols) stands for, in 64 bits, before it is rounded to x's type."""
    x = wide(x)
    out = torch.empty_like(x)
    most = 127.0 if fmt == "int8" else 448.0
    for c in range(0, x.shape[1], 32):
        part = x[:, c:c + 32]
        top = part.abs().amax(1, keepdim=True)
        m, ex = torch.frexp(top / most)                       # top / most = m 2^ex with m in [1/2, 1)
        e = torch.where(m == 0.5, ex - 1, ex).clamp(min=-127)
        e = torch.where(top == 0, torch.full_like(e, -127), e)
        e = torch.where(most * torch.exp2(e.double() - 1) >= top, e - 1, e).clamp(min=-127).double()
        unit = torch.exp2(e)
        assert ((most * unit >= top) | ~torch.isfinite(top)).all() and ((most * unit / 2 < top) | (e == -127)).all()
        if fmt == "e4m3":
            size = (part / unit).abs().clamp(min=2.0 ** -6)
            unit = unit * torch.exp2(torch.floor(torch.log2(size)) - 3)
        out[:, c:c + 32] = torch.round(part / unit) * unit
        out[:, c:c + 32] = torch.where(torch.isfinite(top), out[:, c:c + 32], torch.full_like(part, float("nan")))
    return out
