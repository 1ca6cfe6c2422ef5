"""How far the row operators' 32-bit arithmetic may be from the definition, step by step.

Two comparisons instead of one.  The statistics that a forward keeps are compared with the definition's; results and gradients are
compared with the definition at the statistics that were kept.  A mean's rounding then counts where it happens and not once more, for every
row with the same sign, in a sum over rows, so that the bounds stay far below what they bound even where the mean is large
against the spread.

`U` = 2^-24 is the rounding of one operation relative to its result.  A chain of c additions is off by c U times the sum of the
magnitudes, whatever their order; c is the longest way of a term through registers, lanes, CTAs and the last sum."""
import torch

import row_reference as R
from row_reference import U


def assert_refutes(name, wrong, ref, tol, share=0.9):
    """The bound is worth something: `wrong` (a result that lost what is tested) is outside of it in `share` of the elements."""
    out = ((wrong - ref).abs() > tol).double().mean()
    assert out >= share, f"{name}: only {float(out):.2f} of a lost result would be noticed"


# ------------------------------------------------------------------------------------------------
# LayerNorm(residual + dropout(x)), rows in the last of two dimensions
# ------------------------------------------------------------------------------------------------
def norm_stats(f, eps):
    """mean, rstd of a forward of row_reference.norm_forward, and how far 32 bits may be off: mean absolutely, rstd relatively."""
    s, d = f["s"], f["dropped"]
    E = s.shape[-1]
    # a lane adds at most 36 elements (9 words of 4), then at most 5 additions over lanes
    c = min(E, 36) + 5
    # x / (1 - p): the factor is rounded, then the sum with the residual
    e = U * (d.abs() + s.abs())
    mean = s.mean(-1)
    off = e.mean(-1) + (c + 2) * U * s.abs().mean(-1)               # 1 / E rounded, the product with it
    rstd = f["rstd"].squeeze(-1)
    # Squares around a mean that is off by `off` are too large by off^2; elements off by e move their mean by at most
    # 2 rms(e) sigma (Cauchy-Schwarz), and sigma <= 1 / rstd.  The difference, its square, c additions, 1 / E, + eps: (c + 6) U.
    var = (c + 6) * U + (off * rstd) ** 2 + 2 * (e * e).mean(-1).sqrt() * rstd
    rho = 0.5 * var * (1 + 2 * var) + 6 * U                         # rsqrtf: 2 ulp = 4 U
    return mean, off, rstd, rho


def norm_given(f, stats, w, b, g, turns):
    """Results at given (mean, rstd) (rows, fp32), each with what 32 bits may add; `turns` = rows that a lane group takes."""
    s, d, slope = f["s"], f["dropped"], f["slope"]
    mean, rstd = (t.detach().cpu().double().unsqueeze(-1) for t in stats)
    w, b, g = (t.detach().cpu().double() for t in (w, b, g))
    E = s.shape[-1]
    c = min(E, 36) + 5
    hat = (s - mean) * rstd
    dh = U * (d.abs() + s.abs()) * rstd + 2 * U * hat.abs()          # the sum; the difference and the product
    y = hat * w + b
    out = dict(hat=hat, y=(y, w.abs() * dh + U * y.abs()))
    dd = g * w
    m1, m2 = dd.mean(-1, keepdim=True), (dd * hat).mean(-1, keepdim=True)
    e1 = (c + 4) * U * dd.abs().mean(-1, keepdim=True)              # product with gamma, sum, 1 / E, rstd
    e2 = (c + 4) * U * (dd * hat).abs().mean(-1, keepdim=True) + (dd.abs() * dh).mean(-1, keepdim=True)
    gr = rstd * (dd - m1 - hat * m2)
    tol = rstd * (3 * U * dd.abs() + e1 + 3 * U * m1.abs() + hat.abs() * (e2 + 4 * U * m2.abs()) + dh * m2.abs()) + 2 * U * gr.abs()
    out["gr"] = (gr, tol)
    out["gx"] = (gr * slope, tol * slope + 2 * U * (gr * slope).abs())
    # rows of a lane group, up to 32 lane groups of a CTA, 296 CTAs by 32 lanes, those lanes
    rows = turns + 32 + 10 + 32
    gh = g * hat
    out["gw"] = (gh.sum(0), rows * U * gh.abs().sum(0) + (g.abs() * dh).sum(0))
    out["gb"] = (g.sum(0), rows * U * g.abs().sum(0))
    return out


def norm_forward(x, residual, w, b, p, seed, site, eps):
    f = R.norm_forward(x, residual, w, b, p, seed, site, eps)
    f["dropped"] = f["s"] - residual.detach().cpu().double()
    return f


# ------------------------------------------------------------------------------------------------
# group norm
# ------------------------------------------------------------------------------------------------
def _chains(B, N, C, G, L):
    """Rows that a thread takes, and row lanes of a CTA: a CTA reads 1024 channels at a time (256 threads of 4, 512 of 2, 1024 of 1), a call
    has at least 148 CTAs or one an image, and a thread four rows where there are as many."""
    tiles = max(1, 148 // B)
    lanes = max(1, 1024 // C)
    return N // (tiles * lanes) + 36, lanes


def group_stats(x, G, eps, segments):
    """mean, rstd (B, L, G) and their bounds."""
    x = x.detach().cpu().double()
    B, N, C = x.shape
    rows, lanes = _chains(B, N, C, G, len(segments))
    # Eight rows (7 additions, 1 / 8 or a division of 2 ulp), merges of them, V channels, a group's entries by 8 lanes (at most
    # 1024 / G of them), 1 / n; then tiles, 444 at most, by 32 lanes, and those, or 8 CTAs of a cluster.
    chain = 12 + rows / 8 + 4 + 128 / G + 12 + 14 + 5
    mean, off, rstd, rho = (torch.zeros(B, len(segments), G, dtype=torch.float64) for _ in range(4))
    for l, (lo, hi) in enumerate(segments):
        if hi <= lo:
            continue
        v = x[:, lo:hi].reshape(B, hi - lo, G, C // G)
        m = v.mean((1, 3))
        centred = v - m[:, None, :, None]
        size, spread = v.abs().amax((1, 3)), centred.abs().amax((1, 3))
        # a step rounds the mean, and a difference of means (at most twice the spread) with its factor (2 ulp)
        o = chain * U * (size + 12 * spread)
        r = ((centred ** 2).mean((1, 3)) + eps) ** -0.5
        # means of parts off by at most o move the squares' mean by at most 2 o sigma + o^2
        var = (chain + 20) * U + 2 * o * r + (o * r) ** 2
        mean[:, l], off[:, l], rstd[:, l], rho[:, l] = m, o, r, 0.5 * var * (1 + 2 * var) + 6 * U
    return mean, off, rstd, rho


def group_given(x, w, b, G, activation, segments, stats, g):
    """Results at given (mean, rstd) (B, L, G), each with what 32 bits may add.  activation: None or "silu"."""
    x, w, b, g = (t.detach().cpu().double() for t in (x, w, b, g))
    means, rstds = (t.detach().cpu().double() for t in stats)
    B, N, C = x.shape
    rows, lanes = _chains(B, N, C, G, len(segments))
    per = C // G
    zero = lambda t: (torch.zeros_like(t), torch.zeros_like(t))
    out = dict(y=zero(x), gx=zero(x), gw=zero(w), gb=zero(w), norm=torch.zeros_like(x))
    for l, (lo, hi) in enumerate(segments):
        if hi <= lo:
            continue
        at = l if w.dim() == 2 else slice(None)
        wl, bl = w[at], b[at]
        spread = lambda t: t.repeat_interleave(per, -1)[:, None, :]
        by = lambda t: t.reshape(B, hi - lo, G, per)
        r = spread(rstds[:, l])
        hat = (x[:, lo:hi] - spread(means[:, l])) * r
        z = hat * wl + bl
        zt = 3 * U * (hat * wl).abs() + U * z.abs()                 # difference, factor, sum
        if activation == "silu":
            s = 1 / (1 + torch.exp(-z))
            # __expf: 2 + 1.173 |z| ulp; the division 2 ulp and the sum under it
            st = s * ((1 - s) * (4 + 2.4 * z.abs()) + 6) * U
            y, yt = z * s, 1.1 * zt + z.abs() * st + U * (z * s).abs()
            slope = s * (1 + z * (1 - s))
            # the slope's derivative is at most 0.5
            slopet = st * (1 + z.abs()) + 4 * U * s * (1 + z.abs()) + 0.5 * zt
        else:
            y, yt, slope, slopet = z, zt, torch.ones_like(z), torch.zeros_like(z)
        out["y"][0][:, lo:hi], out["y"][1][:, lo:hi] = y, yt
        out["norm"][:, lo:hi] = bl
        gl = g[:, lo:hi]
        dz = gl * slope
        dzt = gl.abs() * slopet + U * dz.abs()
        d = dz * wl
        # a thread's rows, row lanes, a group's channels by 8 lanes, tiles by 32 lanes, those; gamma and 1 / n
        chain = rows + lanes + per / 8 + 3 + 14 + 5 + 8
        m1, m2 = by(d).mean((1, 3)), by(d * hat).mean((1, 3))
        e1 = by(dzt * wl.abs() + chain * U * d.abs()).mean((1, 3))
        e2 = by(dzt * (wl * hat).abs() + (chain + 2) * U * (d * hat).abs()).mean((1, 3))
        gx = r * (d - spread(m1) - hat * spread(m2))
        out["gx"][0][:, lo:hi] = gx
        out["gx"][1][:, lo:hi] = r * (dzt * wl.abs() + 3 * U * d.abs() + spread(e1) + 3 * U * spread(m1).abs()
                                      + hat.abs() * (spread(e2) + 8 * U * spread(m2).abs())) + 2 * U * gx.abs()
        # a thread's rows, row lanes, tiles by 8 warps (444 / 8) and those, images and levels
        terms = rows + lanes + 56 + 8 + B * len(segments) + 8
        out["gw"][0][at] += (dz * hat).sum((0, 1))
        out["gw"][1][at] += (dzt * hat.abs() + (terms + 3) * U * (dz * hat).abs()).sum((0, 1))
        out["gb"][0][at] += dz.sum((0, 1))
        out["gb"][1][at] += (dzt + terms * U * dz.abs()).sum((0, 1))
    return out
