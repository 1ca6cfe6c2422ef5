"""Operators of the feed-forward block, as cases that can be timed and checked: a matrix product with bias, activation and residual
in its epilogue, a gated feed-forward block, and activation checkpoints in 8 bits with their use in the backward of both.

A case is a plain dict.  `listed()` gives the fixed ones, `draw(rng)` one more of the same ranges, `prepare(case, seed)` what a
program holds before the call, `run(state)` one pass, `work(case)` the bytes and operations that a pass cannot do without,
`exact(case, seed)` what `run` returns by the definition in 64 bits.  `own` picks the package's operators; without it `run`
computes the same in elementary torch operations.

An 8-bit checkpoint holds blocks of 32 neighbours of a row under one power of two 2^e, the smallest for which no element is beyond
the format's largest number (127 for int8, 448 for e4m3); an element is x / 2^e rounded to nearest even and stands for that times
2^e.  An operator with a checkpoint runs its forward on its input, and its backward on what the checkpoint of its input stands for.
"""
import math
import os
import sys

import torch

own = False


def _linear(**kw):
    c = dict(kind="linear", rows=1, K=256, N=256, dtype="bf16", act="none", bias=True, residual="none", ckpt="none", train=True)
    c.update(kw)
    return c


def _gated(**kw):
    c = dict(kind="gated", rows=1, E=256, F=512, dtype="bf16", act="silu", bias=False, residual=True, ckpt="none", train=True)
    c.update(kw)
    return c


def _pack(**kw):
    c = dict(kind="pack", rows=1, cols=256, dtype="bf16", fmt="int8")
    c.update(kw)
    return c


def listed():
    return [
        # first product of the decoder's feed-forward block, served: 900 object queries, the smallest call
        _linear(name="linear_decoder_infer", rows=900, N=512, act="relu", train=False),
        # value projection of six cameras at four levels: the longest product
        _linear(name="linear_value_infer", rows=184950, train=False),
        # first product of the feed-forward block over a 200 x 200 BEV
        _linear(name="linear_bev_train", rows=40000, N=512, act="gelu"),
        # the block's second product, added to a residual stream that is kept in 32 bits, its input kept in 8
        _linear(name="linear_bev_int8_train", rows=40000, K=512, residual="fp32", ckpt="int8"),
        # sizes that divide nothing
        _linear(name="linear_odd_fp16_train", rows=3777, K=59, N=202, dtype="fp16", act="silu", residual="same"),
        # gated block of the decoder: the smallest call of a training step
        _gated(name="gated_decoder_train", rows=900, bias=True),
        # gated block of the base encoder layer, served
        _gated(name="gated_bev_fp16_infer", rows=40000, dtype="fp16", train=False),
        # the same trained
        _gated(name="gated_bev_train", rows=40000),
        # two frames, a wide block, its input kept in 8 bits
        _gated(name="gated_wide_e4m3_train", rows=80000, F=1024, act="gelu", bias=True, ckpt="e4m3"),
        # sizes that divide nothing
        _gated(name="gated_odd_fp16_train", rows=7001, E=90, F=250, dtype="fp16", bias=True, ckpt="int8"),
        # hidden rows of the feed-forward block, kept in 8 bits until the backward
        _pack(name="pack_hidden_fp32", rows=40000, cols=512, dtype="fp32"),
        # image features of six cameras at four levels
        _pack(name="pack_features_e4m3", rows=184950, fmt="e4m3"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "gated", "gated", "pack"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    ckpt = rng.choice(("none", "none", "int8", "e4m3"))
    train = rng.random() < 0.7
    width = lambda: rng.choice((64, 128, 256, 256, 512, rng.randint(8, 600)))
    if kind == "pack":
        cols = width()
        return _pack(rows=min(_log_int(rng, 1, 184950), 40 * 1000 * 1000 // cols), cols=cols, dtype=rng.choice(("fp32", dtype)),
                     fmt=rng.choice(("int8", "e4m3")))
    rows = _log_int(rng, 1, 184950)
    if kind == "linear":
        K, N = width(), rng.choice((width(), 1024))
        return _linear(rows=min(rows, 6 * 10 ** 9 // (K * N), 60 * 10 ** 6 // max(K, N)), K=K, N=N, dtype=dtype,
                       act=rng.choice(("none", "relu", "silu", "gelu")), bias=rng.random() < 0.8,
                       residual=rng.choice(("none", "same", "fp32")), ckpt=ckpt if train else "none", train=train)
    E, F = width(), rng.choice((width(), 1024))
    return _gated(rows=min(rows, 10 ** 10 // (E * F), 40 * 10 ** 6 // max(E, F)), E=E, F=F, dtype=dtype,
                  act=rng.choice(("relu", "silu", "silu", "gelu")), bias=rng.random() < 0.5, residual=rng.random() < 0.7,
                  ckpt=ckpt if train else "none", train=train)


# ------------------------------------------------------------------------------------------------
_DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BIASES = ("b_gate", "b_up", "b_down")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPE[case["dtype"]]
    normal = lambda *size: torch.randn(*size, generator=g, device="cuda")
    s = dict(case=case)
    # rows as a norm leaves them: columns with a scale and a mean of their own
    rows_of = lambda n, cols: (normal(n, cols) * (1 + 0.3 * normal(cols)) + 0.3 * normal(cols)).to(dt)
    weight = lambda n, k: (normal(n, k) / math.sqrt(k)).to(dt)
    if case["kind"] == "pack":
        # hidden rows as an activation leaves them, columns of very different size
        s["x"] = (normal(case["rows"], case["cols"]) * torch.exp(normal(case["cols"]))).to(dt)
        return s
    if case["kind"] == "linear":
        rows, K, N = case["rows"], case["K"], case["N"]
        s["x"], s["weight"] = rows_of(rows, K), weight(N, K)
        s["bias"] = (0.3 * normal(N)).to(dt) if case["bias"] else None
        out = torch.float32 if case["residual"] == "fp32" else dt
        s["residual"] = normal(rows, N).to(out) if case["residual"] != "none" else None
        s["grad"] = normal(rows, N).to(out)
        leaves = ("x", "weight", "bias", "residual")
    else:
        rows, E, F = case["rows"], case["E"], case["F"]
        s["x"], s["w_gate"], s["w_up"], s["w_down"] = rows_of(rows, E), weight(F, E), weight(F, E), weight(E, F)
        for name, n in zip(_BIASES, (F, F, E)):
            s[name] = (0.3 * normal(n)).to(dt) if case["bias"] else None
        s["grad"] = normal(rows, E).to(dt)
        leaves = ("x", "w_gate", "w_up", "w_down") + _BIASES
    if case["train"]:
        s["leaves"] = [s[k].requires_grad_(True) for k in leaves if s[k] is not None]
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _stands_for(x, fmt):
    """What the 8-bit checkpoint of x (rows, cols) stands for, in 32 bits."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -cols % 32)).view(rows, -1, 32)
    m, ex = torch.frexp(v.abs().amax(-1, keepdim=True))                  # amax = m 2^ex, m in [1/2, 1)
    top, shift = (127 / 128, 7) if fmt == "int8" else (448 / 512, 9)     # largest number = top 2^shift
    e = torch.where(m > 0, ex - shift + (m > top), torch.full_like(ex, -127)).clamp(min=-127)
    q = torch.ldexp(v, -e)
    q = torch.round(q) if fmt == "int8" else q.to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, e).view(rows, -1)[:, :cols]


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "silu":
        sg = torch.sigmoid(z)
        return sg * (1 + z * (1 - sg))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _wide(t):
    return None if t is None else t.detach().float()


def _product(x, w, b):
    z = x @ w.t()
    return z if b is None else z + b


def _plain_linear(s):
    case, dt = s["case"], s["x"].dtype
    x, w, b, r, g = (_wide(s[k]) for k in ("x", "weight", "bias", "residual", "grad"))
    y = _act(_product(x, w, b), case["act"])
    y = (y if r is None else y + r).to(s["grad"].dtype)
    if not case["train"]:
        return y
    if case["ckpt"] != "none":
        x = _stands_for(s["x"].detach(), case["ckpt"])
    dz = g * _slope(_product(x, w, b), case["act"])
    grads = [(dz @ w).to(dt), (dz.t() @ x).to(dt)]
    if b is not None:
        grads.append(dz.sum(0).to(dt))
    if r is not None:
        grads.append(s["grad"])
    return (y, *grads)


def _plain_gated(s):
    case, dt, act = s["case"], s["x"].dtype, s["case"]["act"]
    x, wg, wu, wd, bg, bu, bd, g = (_wide(s[k]) for k in ("x", "w_gate", "w_up", "w_down") + _BIASES + ("grad",))
    y = _product(_act(_product(x, wg, bg), act) * _product(x, wu, bu), wd, bd)
    y = (y + x if case["residual"] else y).to(dt)
    if not case["train"]:
        return y
    if case["ckpt"] != "none":
        x = _stands_for(s["x"].detach(), case["ckpt"])
    gate, up = _product(x, wg, bg), _product(x, wu, bu)
    opened = _act(gate, act)
    dh = g @ wd
    dg, du = dh * up * _slope(gate, act), dh * opened
    gx = dg @ wg + du @ wu
    grads = [(gx + g if case["residual"] else gx).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt), (g.t() @ (opened * up)).to(dt)]
    if bg is not None:
        grads += [dg.sum(0).to(dt), du.sum(0).to(dt), g.sum(0).to(dt)]
    return (y, *grads)


def _plain_pack(s):
    return _stands_for(s["x"], s["case"]["fmt"]).to(s["x"].dtype)


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
    if case["kind"] == "pack":
        return M.decompress8(M.compress8(s["x"], case["fmt"]))
    ckpt = None if case["ckpt"] == "none" else case["ckpt"]
    if case["kind"] == "linear":
        act = None if case["act"] == "none" else case["act"]
        return M.linear_act(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"], checkpoint=ckpt)
    return M.gated_feed_forward(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["b_gate"], s["b_up"], s["b_down"],
                                activation=case["act"], residual=s["x"] if case["residual"] else None, checkpoint=ckpt)


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return {"linear": _plain_linear, "gated": _plain_gated, "pack": _plain_pack}[case["kind"]](state)
    if not case.get("train"):
        with torch.no_grad():
            return _own_call(state)
    y = _own_call(state)
    return (y,) + torch.autograd.grad(y, state["leaves"], state["grad"])


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def _checkpoint_exact(x, fmt):
    x = x.double()
    out = torch.empty_like(x)
    largest = 127.0 if fmt == "int8" else 448.0
    for first in range(0, x.shape[1], 32):
        part = x[:, first:first + 32]
        top = part.abs().max(1, keepdim=True).values
        e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -149) / largest))
        e = torch.where(largest * torch.exp2(e) < top, e + 1, e)                  # where the logarithm was rounded
        e = torch.where(largest * torch.exp2(e - 1) >= top, e - 1, e).clamp(min=-127.0)
        unit = torch.exp2(e)
        if fmt == "e4m3":       # three bits behind the leading one, down to 2^-6, and the same spacing below
            size = (part / unit).abs().clamp(min=2.0 ** -6)
            unit = unit * torch.exp2(torch.floor(torch.log2(size)) - 3)
        out[:, first:first + 32] = torch.round(part / unit) * unit
    return out


def _act_exact(z, act):
    """The activation and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.maximum(z, torch.zeros_like(z)), torch.where(z > 0, 1.0, 0.0).double()
    if act == "silu":
        e = torch.exp(-z)
        return z / (1 + e), (1 + e + z * e) / (1 + e) ** 2
    half = 0.5 * torch.special.erfc(-z / 2 ** 0.5)
    return z * half, half + z * (2 * math.pi) ** -0.5 * torch.exp(-(z ** 2) / 2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "pack":
        return _checkpoint_exact(s["x"], case["fmt"])
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v)}
    x, g, act = d["x"], d["grad"], case["act"]
    affine = lambda v, w, b: torch.addmm(d[b], v, d[w].t()) if b in d else torch.mm(v, d[w].t())
    again = x if case["ckpt"] == "none" else _checkpoint_exact(s["x"].detach(), case["ckpt"])
    if case["kind"] == "linear":
        y = _act_exact(affine(x, "weight", "bias"), act)[0]
        if "residual" in d:
            y = y + d["residual"]
        if not case["train"]:
            return y
        dz = g * _act_exact(affine(again, "weight", "bias"), act)[1]
        out = [y, torch.mm(dz, d["weight"]), torch.mm(dz.t(), again)]
        return tuple(out + ([dz.sum(0)] if "bias" in d else []) + ([g] if "residual" in d else []))
    hidden = lambda v: _act_exact(affine(v, "w_gate", "b_gate"), act) + (affine(v, "w_up", "b_up"),)
    a, _, up = hidden(x)
    y = affine(a * up, "w_down", "b_down")
    if case["residual"]:
        y = y + x
    if not case["train"]:
        return y
    a, slope, up = hidden(again)
    through = torch.mm(g, d["w_down"])
    du, dg = through * a, through * slope * up
    gx = torch.mm(dg, d["w_gate"]) + torch.mm(du, d["w_up"])
    out = [y, gx + g if case["residual"] else gx, torch.mm(dg.t(), again), torch.mm(du.t(), again), torch.mm(g.t(), a * up)]
    return tuple(out + ([dg.sum(0), du.sum(0), g.sum(0)] if "b_gate" in d else []))


# ------------------------------------------------------------------------------------------------
def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    rows = case["rows"]
    if case["kind"] == "pack":
        # the codes and their scales are written, and read when they are taken out again
        n = rows * case["cols"]
        codes = n + rows * -(-case["cols"] // 32)
        return {"bytes": 2 * n * size + 2 * codes, "flops": 4 * n}
    if case["kind"] == "linear":
        K, N = case["K"], case["N"]
        out = 4 if case["residual"] == "fp32" else size
        bytes_ = rows * K * size + (N * K + (N if case["bias"] else 0)) * size + rows * N * out
        if case["residual"] != "none":
            bytes_ += rows * N * out
        flops = 2 * rows * N * K
        if case["train"]:       # the gradient of the result in, those of the input and the parameters out
            bytes_ += rows * N * out + rows * K * size + (N * K + (N if case["bias"] else 0)) * size
            flops *= 3
        return {"bytes": bytes_, "flops": flops}
    E, F = case["E"], case["F"]
    params = (3 * E * F + ((2 * F + E) if case["bias"] else 0)) * size
    bytes_, flops = 2 * rows * E * size + params, 6 * rows * E * F
    if case["train"]:
        bytes_ += 2 * rows * E * size + params
        flops *= 3
    return {"bytes": bytes_, "flops": flops}
