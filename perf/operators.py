"""Row operators around the attention, as cases that can be timed and checked: dropout from a counter-based generator,
LayerNorm(residual + dropout(x)), and channels-last group norm with an activation over the levels of a feature pyramid.

A case is a plain dict.  `listed()` gives the fixed ones, `draw(rng)` one more of the same ranges, `prepare(case, seed)` what a
program holds before the call, `run(state)` one pass, `work(case)` the bytes and operations that a pass cannot do without,
`exact(case, seed)` what `run` returns by the definition in 64 bits.  `own` picks the package's operators; without it `run`
computes the same in elementary torch operations.

The mask of a dropout is a function of (seed, site, element): element i of the tensor in row-major order takes word i mod 4 of
Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) at counter
(i div 4 low, i div 4 high, site, 0) under the key (seed low, seed high), and is kept where that word is >= p * 2^32.
"""
import math
import os
import sys

import torch

own = False

BASE = "116x200 58x100 29x50 15x25"      # 928 x 1600 images at strides 8 / 16 / 32 / 64
SMALL = "23x40"                          # 736 x 1280 images at stride 32
EPS = 1e-5


def _drop(**kw):
    c = dict(kind="dropout", rows=1, E=256, dtype="fp32", p=0.1, site=1, activation="none", residual=False, train=True)
    c.update(kw)
    return c


def _norm(**kw):
    c = dict(kind="norm", rows=1, E=256, dtype="fp32", p=0.1, site=2, train=True)
    c.update(kw)
    return c


def _group(**kw):
    c = dict(kind="group", B=6, levels=BASE, C=256, G=32, dtype="fp32", activation="none", per_level=False, train=True)
    c.update(kw)
    return c


def listed():
    return [
        # the decoder's attention adds dropout(output) to its 900 object queries: the smallest call of a training step
        _drop(name="dropout_decoder_train", rows=900, residual=True),
        # hidden rows of the feed-forward block of a 200 x 200 BEV: ReLU and dropout
        _drop(name="dropout_ffn_train", rows=40000, E=512, activation="relu"),
        # image features of six cameras at four levels in bf16: the largest tensor that is dropped out
        _drop(name="dropout_features_bf16", rows=184950, dtype="bf16", train=False),
        # sizes that divide nothing: a number of elements that is odd, half storage, another rate
        _drop(name="dropout_odd_fp16_train", rows=3777, E=59, dtype="fp16", p=0.25, residual=True),
        # end of a decoder block
        _norm(name="norm_decoder_train", rows=900),
        # end of each block of the base encoder layer, one frame
        _norm(name="norm_bev_train", rows=40000),
        # the same with two frames in bf16
        _norm(name="norm_bev_bf16_train", rows=80000, dtype="bf16"),
        # rows whose width is no multiple of four, so that most begin off the 16-byte grid; forward only
        _norm(name="norm_odd_fp16", rows=7001, E=202, dtype="fp16", p=0.3, train=False),
        # projected features of the small detector: six cameras, one level
        _group(name="group_small_train", levels=SMALL, activation="silu"),
        # projected features of the base detector: six cameras, four levels
        _group(name="group_base_train"),
        # the same served in bf16, with an activation and weights of their own for each level
        _group(name="group_base_bf16_infer", dtype="bf16", activation="relu", per_level=True, train=False),
        # odd levels, 15 channels a group, half storage
        _group(name="group_odd_fp16_train", B=3, levels="57x101 29x51 15x25", C=90, G=6, dtype="fp16", activation="silu",
               per_level=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("dropout", "norm", "norm", "group", "group"))
    dtype = rng.choice(("fp32", "fp32", "bf16", "fp16"))
    train = rng.random() < 0.7
    if kind == "group":
        h = _log_int(rng, 8, 116)
        w = max(2, int(round(h * rng.uniform(0.8, 1.9))))
        levels = []
        for _ in range(rng.randint(1, 4)):
            levels.append("%dx%d" % (h, w))
            h, w = (h + 1) // 2, (w + 1) // 2
        G = rng.choice((1, 4, 6, 8, 16, 32, 32))
        C = G * max(1, rng.randint(32, 256) // G)
        act = rng.choice(("none", "silu")) if train else rng.choice(("none", "silu", "relu"))
        return _group(B=rng.randint(1, 6), levels=" ".join(levels), C=C, G=G, dtype=dtype, activation=act,
                      per_level=rng.random() < 0.5, train=train)
    rows, p, site = _log_int(rng, 1, 80000), round(rng.uniform(0.02, 0.6), 3), rng.randint(0, 40)
    E = rng.choice((64, 128, 256, 256, 384, 512, rng.randint(1, 600)))
    rows = min(rows, 20 * 1000 * 1000 // E)
    if kind == "norm":
        return _norm(rows=rows, E=max(E, 8), dtype=dtype, p=p, site=site, train=train)
    return _drop(rows=rows, E=E, dtype=dtype, p=p, site=site, activation=rng.choice(("none", "relu")),
                 residual=rng.random() < 0.5, train=train)


# ------------------------------------------------------------------------------------------------
_DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _levels(case):
    return [tuple(int(x) for x in l.split("x")) for l in case["levels"].split()]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPE[case["dtype"]]
    normal = lambda *size: torch.randn(*size, generator=g, device="cuda")
    s = dict(case=case)
    if case["kind"] == "group":
        levels = _levels(case)
        B, N, C, L = case["B"], sum(h * w for h, w in levels), case["C"], len(levels)
        # features as a projection leaves them: each channel with a mean and a spread of its own
        s["x"] = (normal(B, N, C) * (0.5 + normal(C).abs()) + normal(C)).to(dt)
        wsize = (L, C) if case["per_level"] else (C,)
        s["weight"], s["bias"] = 1 + 0.3 * normal(*wsize), 0.3 * normal(*wsize)
        s["grad"] = normal(B, N, C).to(dt)
        shapes = torch.tensor(levels, dtype=torch.int64)
        hw = shapes[:, 0] * shapes[:, 1]
        s["shapes"], s["lsi"] = shapes.cuda(), torch.cat([hw.new_zeros(1), hw.cumsum(0)[:-1]]).cuda()
        s["rows"] = [h * w for h, w in levels]
        leaves = ("x", "weight", "bias")
    else:
        rows, E = case["rows"], case["E"]
        s["x"] = normal(rows, E).to(dt)
        s["seed"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), generator=g, device="cuda")
        s["grad"] = normal(rows, E).to(dt)
        s["residual"] = normal(rows, E).to(dt) if case.get("residual", True) else None
        leaves = ("x", "residual") if s["residual"] is not None else ("x",)
        if case["kind"] == "norm":
            s["weight"], s["bias"] = 1 + 0.3 * normal(E), 0.3 * normal(E)
            leaves += ("weight", "bias")
    if case["train"]:
        s["leaves"] = [s[k].requires_grad_(True) for k in leaves]
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _keep(n, p, seed, site):
    """Which of n elements are kept."""
    m = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device=seed.device, dtype=torch.int64)
    c0, c1, c2, c3 = block & m, block >> 32, torch.full_like(block, site), torch.zeros_like(block)
    k0, k1 = seed & m, (seed >> 32) & m
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # 64-bit products; >> keeps the sign, & drops it
        c0, c1, c2, c3 = ((b >> 32) & m) ^ c1 ^ k0, b & m, ((a >> 32) & m) ^ c3 ^ k1, a & m
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    words = torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]
    return words >= int(p * 4294967296.0 + 0.5)


def _plain_dropout(s):
    case, x = s["case"], s["x"].detach().float()
    keep = _keep(x.numel(), case["p"], s["seed"], case["site"]).view(x.shape)
    scale = 1.0 / (1.0 - case["p"])
    y = x
    if case["activation"] == "relu":
        y = y.clamp(min=0.0)
        live = keep & (x > 0)
    else:
        live = keep
    y = torch.where(keep, y * scale, torch.zeros_like(y))
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    y = y.to(s["x"].dtype)
    if not case["train"]:
        return y
    gx = torch.where(live, s["grad"].float() * scale, torch.zeros_like(x)).to(s["x"].dtype)
    return (y, gx) + ((s["grad"],) if s["residual"] is not None else ())


def _plain_norm(s):
    case, dt = s["case"], s["x"].dtype
    x, r, w = s["x"].detach().float(), s["residual"].detach().float(), s["weight"].detach()
    keep = _keep(x.numel(), case["p"], s["seed"], case["site"]).view(x.shape)
    scale = 1.0 / (1.0 - case["p"])
    total = r + torch.where(keep, x * scale, torch.zeros_like(x))
    centred = total - total.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    hat = centred * rstd
    y = (hat * w + s["bias"].detach()).to(dt)
    if not case["train"]:
        return y
    g = s["grad"].float()
    d = g * w
    gr = rstd * (d - d.mean(-1, keepdim=True) - hat * (d * hat).mean(-1, keepdim=True))
    gx = torch.where(keep, gr * scale, torch.zeros_like(gr))
    return y, gx.to(dt), gr.to(dt), (g * hat).sum(0), g.sum(0)


def _plain_group(s):
    case, dt, G = s["case"], s["x"].dtype, s["case"]["G"]
    x, w, b = s["x"].detach().float(), s["weight"].detach(), s["bias"].detach()
    g = s["grad"].float()
    B, _, C = x.shape
    ys, gxs, gws, gbs, at = [], [], [], [], 0
    for l, n in enumerate(s["rows"]):
        wl, bl = (w[l], b[l]) if case["per_level"] else (w, b)
        v = x[:, at:at + n].reshape(B, n, G, C // G)
        centred = v - v.mean((1, 3), keepdim=True)
        rstd = torch.rsqrt((centred * centred).mean((1, 3), keepdim=True) + EPS)
        hat = (centred * rstd).view(B, n, C)
        z = hat * wl + bl
        sig = torch.sigmoid(z) if case["activation"] == "silu" else None
        ys.append(z if case["activation"] == "none" else z.clamp(min=0.0) if case["activation"] == "relu" else z * sig)
        if case["train"]:
            dz = g[:, at:at + n]
            if case["activation"] == "relu":
                dz = dz * (z > 0)
            elif case["activation"] == "silu":
                dz = dz * sig * (1 + z * (1 - sig))
            gws.append((dz * hat).sum((0, 1)))
            gbs.append(dz.sum((0, 1)))
            d, h4 = (dz * wl).view(B, n, G, C // G), hat.view(B, n, G, C // G)
            gx = rstd * (d - d.mean((1, 3), keepdim=True) - h4 * (d * h4).mean((1, 3), keepdim=True))
            gxs.append(gx.view(B, n, C))
        at += n
    y = torch.cat(ys, 1).to(dt)
    if not case["train"]:
        return y
    join = torch.stack if case["per_level"] else (lambda t: sum(t[1:], t[0]))
    return y, torch.cat(gxs, 1).to(dt), join(gws), join(gbs)


# ------------------------------------------------------------------------------------------------
# the package's operators
# ------------------------------------------------------------------------------------------------
def _package():
    path = os.path.join(os.getcwd(), "3d-deformable-attention_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import dfa3d_b200
    return dfa3d_b200


def _own_call(s):
    case, M = s["case"], _package()
    if case["kind"] == "dropout":
        act = None if case["activation"] == "none" else case["activation"]
        return M.dropout(s["x"], case["p"], s["seed"], case["site"], activation=act, residual=s["residual"])
    if case["kind"] == "norm":
        return M.dropout_add_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], case["p"], s["seed"], case["site"],
                                        eps=EPS)
    act = None if case["activation"] == "none" else case["activation"]
    return M.group_norm(s["x"], case["G"], s["weight"], s["bias"], eps=EPS, activation=act, spatial_shapes=s["shapes"],
                        level_start_index=s["lsi"])


def run(state):
    if not own:
        with torch.no_grad():
            return {"dropout": _plain_dropout, "norm": _plain_norm, "group": _plain_group}[state["case"]["kind"]](state)
    if not state["case"]["train"]:
        with torch.no_grad():
            return _own_call(state)
    y = _own_call(state)
    return (y,) + torch.autograd.grad(y, state["leaves"], state["grad"])


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def _mul_hi_lo(a, const):
    """High and low 32 bits of a * const from 16-bit halves."""
    al, ah, bl, bh = a & 0xFFFF, a >> 16, const & 0xFFFF, const >> 16
    low = al * bl
    mid = ah * bl + (low >> 16)
    mid2 = al * bh + (mid & 0xFFFF)
    return ah * bh + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | (low & 0xFFFF)


def _uniform_words(n, seed, site):
    key = int(seed) & (2 ** 64 - 1)
    key = [key & 0xFFFFFFFF, key >> 32]
    i = torch.arange(-(-n // 4), device="cuda")
    ctr = [i % 2 ** 32, i // 2 ** 32, torch.zeros_like(i) + site, torch.zeros_like(i)]
    for r in range(7):
        k = [(key[0] + r * 0x9E3779B9) % 2 ** 32, (key[1] + r * 0xBB67AE85) % 2 ** 32]
        h0, l0 = _mul_hi_lo(ctr[0], 0xD2511F53)
        h1, l1 = _mul_hi_lo(ctr[2], 0xCD9E8D57)
        ctr = [h1 ^ ctr[1] ^ k[0], l1, h0 ^ ctr[3] ^ k[1], l0]
    return torch.stack(ctr, -1).flatten()[:n]


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach().double()
    if case["kind"] == "group":
        B, N, C = x.shape
        G, act = case["G"], case["activation"]
        w, b = s["weight"].detach().double(), s["bias"].detach().double()
        y, gx = torch.empty_like(x), torch.empty_like(x)
        gw, gb = torch.zeros_like(w), torch.zeros_like(b)
        first = 0
        for l, (h, wd) in enumerate(_levels(case)):
            rows = slice(first, first + h * wd)
            first += h * wd
            at = l if case["per_level"] else slice(None)
            for i in range(B):
                v = x[i, rows]
                by_group = v.t().reshape(G, -1)
                var, mean = torch.var_mean(by_group, 1, correction=0)
                inv = (var + EPS).rsqrt()
                spread = lambda t: t.repeat_interleave(C // G)
                hat = (v - spread(mean)) * spread(inv)
                z = hat * w[at] + b[at]
                if act == "silu":
                    y[i, rows] = z / (1 + torch.exp(-z))
                else:
                    y[i, rows] = torch.maximum(z, torch.zeros_like(z)) if act == "relu" else z
                if not case["train"]:
                    continue
                dz = s["grad"][i, rows].double()
                if act == "relu":
                    dz = torch.where(z > 0, dz, torch.zeros_like(dz))
                elif act == "silu":
                    sg = 1 / (1 + torch.exp(-z))
                    dz = dz * (sg + z * sg * (1 - sg))
                gw[at] += (dz * hat).sum(0)
                gb[at] += dz.sum(0)
                d = dz * w[at]
                m1 = spread(d.t().reshape(G, -1).mean(1))
                m2 = spread((d * hat).t().reshape(G, -1).mean(1))
                gx[i, rows] = spread(inv) * (d - m1 - hat * m2)
        return (y, gx, gw, gb) if case["train"] else y
    rows, E = x.shape
    kept = (_uniform_words(rows * E, s["seed"].item(), case["site"]) >= math.floor(case["p"] * 2 ** 32 + 0.5)).view(rows, E)
    factor = kept.double() / (1 - case["p"])
    g = s["grad"].double()
    if case["kind"] == "dropout":
        active = (x > 0).double() if case["activation"] == "relu" else torch.ones_like(x)
        y = x * active * factor
        out = (y if s["residual"] is None else y + s["residual"].detach().double(), g * active * factor)
        if s["residual"] is not None:
            out += (g,)
        return out if case["train"] else out[0]
    total = s["residual"].detach().double() + x * factor
    var, mean = torch.var_mean(total, 1, correction=0, keepdim=True)
    hat = (total - mean) / (var + EPS).sqrt()
    w = s["weight"].detach().double()
    y = hat * w + s["bias"].detach().double()
    if not case["train"]:
        return y
    gr = g * w
    gr = (gr - gr.mean(1, keepdim=True) - hat * (gr * hat).mean(1, keepdim=True)) / (var + EPS).sqrt()
    return y, gr * factor, gr, (g * hat).sum(0), g.sum(0)


# ------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "group":
        levels = _levels(case)
        n = case["B"] * sum(h * w for h, w in levels) * case["C"]
        params = 4 * 2 * case["C"] * (len(levels) if case["per_level"] else 1)
        if case["train"]:                # x and grad read, y and grad_x written, weights read and their gradients written
            return {"bytes": 4 * n * e + 2 * params, "flops": 24 * n}
        return {"bytes": 2 * n * e + params, "flops": 8 * n}
    n = case["rows"] * case["E"]
    if case["kind"] == "dropout":
        passes = 2 + (1 if case["residual"] else 0) + (2 if case["train"] else 0)
        return {"bytes": passes * n * e + 8, "flops": (3 if case["train"] else 2) * n}
    params = 4 * 2 * case["E"]
    if case["train"]:                    # x, residual, grad read; y, grad_x, grad_residual written
        return {"bytes": 6 * n * e + 2 * params + 8, "flops": 24 * n}
    return {"bytes": 3 * n * e + params + 8, "flops": 10 * n}
