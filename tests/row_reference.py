"""Row operators by their definitions in 64 bits, on the CPU, and how far a 32-bit computation may be from them.

`U` is the rounding of one 32-bit operation, 2^-24 relative.  A sum of n terms in any order is off by at most (n - 1) U times the sum
of their magnitudes (to first order); the kernels' sums have chains far shorter than n, but the bound holds whatever the order.
`half_step(dtype)` is the rounding of a result to its storage type."""
import numpy as np
import torch

U = 2.0 ** -24
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the smallest subnormal: what a result near 0 is off by at least."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def philox_words(n, seed, site):
    """Words 0 ... n-1 of Philox4x32-7 as (n,) uint64."""
    m = np.uint64(0xFFFFFFFF)
    s32 = np.uint64(32)
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [block & m, block >> s32, np.full_like(block, site), np.zeros_like(block)]
    key = seed & (2 ** 64 - 1)
    k = [key & 0xFFFFFFFF, key >> 32]
    for _ in range(7):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s32) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> s32) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[:n]


def kept(shape, p, seed, site):
    n = int(np.prod(shape))
    return torch.from_numpy(philox_words(n, seed, site) >= np.uint64(int(p * 2.0 ** 32 + 0.5))).view(shape)


def dropout(x, p, seed, site, activation=None, residual=None):
    """y and dy/dx in float64."""
    x = x.detach().cpu().double()
    keep = kept(x.shape, p, seed, site)
    scale = 1.0 / (1.0 - p) if p < 1 else 0.0
    zero = torch.zeros_like(x)
    y = torch.where(x <= 0, zero, x) if activation else x
    y = torch.where(keep, y * scale, zero)
    slope = torch.where(keep & ~(x <= 0) if activation else keep, zero + scale, zero)
    if residual is not None:
        y = y + residual.detach().cpu().double()
    return y, slope


def assert_within(name, got, ref, tol):
    got, ref = got.detach().cpu().double(), ref.double()
    assert got.shape == ref.shape, f"{name}: {tuple(got.shape)} vs {tuple(ref.shape)}"
    err = (got - ref).abs()
    bad = ~(err <= tol)
    if bad.any():
        i = int(torch.argmax(torch.where(bad, err - tol, torch.full_like(err, -1))))
        tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(err)
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of tolerance; element {i}: got {got.flatten()[i]!r} "
                             f"ref {ref.flatten()[i]!r} err {err.flatten()[i]:.3e} tol {tol.flatten()[i]:.3e}")


# ------------------------------------------------------------------------------------------------
def norm_forward(x, residual, w, b, p, seed, site, eps):
    """A dict of float64 tensors of LayerNorm(residual + dropout(x)), rows in the last dimension."""
    d, slope = dropout(x, p, seed, site)
    s = residual.detach().cpu().double() + d
    w, b = w.detach().cpu().double(), b.detach().cpu().double()
    mean = s.mean(-1, keepdim=True)
    var = ((s - mean) ** 2).mean(-1, keepdim=True)
    rstd = (var + eps) ** -0.5
    hat = (s - mean) * rstd
    return dict(y=hat * w + b, hat=hat, rstd=rstd, s=s, w=w, slope=slope)


def hat_error(f):
    """How far the normalised value of a 32-bit computation may be off: the sum's own three roundings and those of the mean (a sum of
    E) times rstd, and rstd's, whose sum of E squares is off by (E + 4) U relative, plus the squares' error from the mean's."""
    E = f["s"].shape[-1]
    size = f["s"].abs().amax(-1, keepdim=True)
    shift = (E + 8) * U * size * f["rstd"]
    return shift + f["hat"].abs() * ((E + 8) * U + 2 * shift)


def norm_backward(f, g):
    g = g.detach().cpu().double()
    d = g * f["w"]
    hat = f["hat"]
    gr = f["rstd"] * (d - d.mean(-1, keepdim=True) - hat * (d * hat).mean(-1, keepdim=True))
    lead = tuple(range(g.dim() - 1))
    E = g.shape[-1]
    dh = hat_error(f)
    size, mh = d.abs(), (d * hat).abs().mean(-1, keepdim=True)
    # d is rounded once, the means are sums of E, hat is off by dh
    tol = f["rstd"] * (4 * U * size + (E + 8) * U * (size.mean(-1, keepdim=True) + hat.abs() * mh) + dh * mh
                       + hat.abs() * (size * dh).mean(-1, keepdim=True)) + (E + 8) * U * gr.abs() \
        + 2 * gr.abs() * dh.amax(-1, keepdim=True)
    rows = g.numel() // E
    return dict(gx=gr * f["slope"], gr=gr, gw=(g * hat).sum(lead), gb=g.sum(lead), tol=tol,
                tol_w=(rows + 4) * U * (g * hat).abs().sum(lead) + (g.abs() * dh).sum(lead),
                tol_b=(rows + 4) * U * g.abs().sum(lead))


# ------------------------------------------------------------------------------------------------
def act(z, activation):
    if activation == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z)
    if activation == "silu":
        return z / (1 + torch.exp(-z))
    return z


def act_slope(z, activation):
    if activation == "relu":
        return (~(z <= 0)).double()
    if activation == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def group_norm(x, w, b, G, eps, activation, segments, grad=None):
    """y, and with grad the gradients, of x (B, N, C) float64 on the CPU; segments: (first, last) row of every level.  Each result comes
    with a tolerance: `tol` entries hold what 32-bit arithmetic may be off by."""
    x = x.detach().cpu().double()
    B, N, C = x.shape
    w, b = w.detach().cpu().double(), b.detach().cpu().double()
    out = dict(y=torch.zeros_like(x), tol_y=torch.zeros_like(x), gx=torch.zeros_like(x), tol_gx=torch.zeros_like(x),
               gw=torch.zeros_like(w), gb=torch.zeros_like(b), tol_w=torch.zeros_like(w), tol_b=torch.zeros_like(b))
    g = None if grad is None else grad.detach().cpu().double()
    for l, (lo, hi) in enumerate(segments):
        if hi <= lo:
            continue
        at = l if w.dim() == 2 else slice(None)
        n = (hi - lo) * (C // G)
        v = x[:, lo:hi].view(B, hi - lo, G, C // G)
        mean = v.mean((1, 3), keepdim=True)
        rstd = (((v - mean) ** 2).mean((1, 3), keepdim=True) + eps) ** -0.5
        spread = lambda t: t.expand(B, hi - lo, G, C // G).reshape(B, hi - lo, C)
        hat = spread((v - mean) * rstd)
        # The kernels sum a thread's eight rows, the thread's blocks of eight, lanes, CTAs, in chains below `chain`.  The mean
        # of values of magnitude `size` is off by chain U size, times rstd; the sum of squares is relative to itself.
        chain = min(n, 64 + (hi - lo) / 64.0 + (C // G))
        shift = spread(chain * U * v.abs().amax((1, 3), keepdim=True) * rstd)
        dh = shift + hat.abs() * ((chain + 8) * U + 2 * shift)
        z = hat * w[at] + b[at]
        slope = act_slope(z, activation)
        zt = dh * w[at].abs() + 4 * U * (z.abs() + b[at].abs())
        out["y"][:, lo:hi] = act(z, activation)
        # SiLU's slope is below 1.1; its exponential and division are good to a few units
        out["tol_y"][:, lo:hi] = 1.1 * zt + 8 * U * z.abs()
        if g is None:
            continue
        gl = g[:, lo:hi]
        dz = gl * slope
        # slope of SiLU: changes by at most 0.5 a unit of z
        dzt = gl.abs() * (0.5 * zt + 16 * U) if activation == "silu" else gl.abs() * U
        d = dz * w[at]
        dt = dzt * w[at].abs() + U * d.abs()
        by = lambda t: t.reshape(B, hi - lo, G, C // G)
        m1, m2 = by(d).mean((1, 3), keepdim=True), by(d * hat).mean((1, 3), keepdim=True)
        e1 = by(dt + chain * U * d.abs()).mean((1, 3), keepdim=True)
        e2 = by(dt * hat.abs() + d.abs() * dh + chain * U * (d * hat).abs()).mean((1, 3), keepdim=True)
        rs = spread(rstd)
        gx = rs * (d - spread(m1) - hat * spread(m2))
        out["gx"][:, lo:hi] = gx
        out["tol_gx"][:, lo:hi] = rs * (dt + spread(e1) + hat.abs() * spread(e2) + dh * spread(m2).abs() + 4 * U * (
            d.abs() + spread(m1).abs() + (hat * spread(m2)).abs())) + gx.abs() * (dh.amax() + (chain + 8) * U)
        terms = chain + B * 80
        out["gw"][at] += (dz * hat).sum((0, 1))
        out["gb"][at] += dz.sum((0, 1))
        out["tol_w"][at] += (dzt * hat.abs() + dz.abs() * dh + terms * U * (dz * hat).abs()).sum((0, 1))
        out["tol_b"][at] += (dzt + terms * U * dz.abs()).sum((0, 1))
    return out
