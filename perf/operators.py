"""Workloads of the network operators of ``rune_b200.ops``: normalisation, linear layer, gated layer.

Each case is one pass of one operator, forward alone (serving) or forward and backward
(training), on data of the distributions that the Möbius networks see: hidden states of unit
scale with a few loud channels, weights of scale 1 / sqrt(inputs), unit output gradients.

``run`` computes the plain form in float32 (elementary torch operations, one rounding at the
end) where ``own`` is false, and calls ``rune_b200.ops`` where it is true. ``exact`` evaluates
the definitions in float64 by automatic differentiation, apart from both.
"""

import math

import torch

own = False

EPS = 1.0e-8  # the Möbius networks' norm_eps
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


# ----------------------------------------------------------------------------------- the cases
def norm(name, dtype, rows, width, residual, train=False, out="same"):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "width": width,
            "residual": residual, "train": train, "out": out}


def linear(name, dtype, rows, inputs, outputs, act, bias, residual, train=False):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "in": inputs,
            "out": outputs, "act": act, "bias": bias, "residual": residual, "train": train}


def gated(name, dtype, rows, inputs, outputs, act, bias, train=False):
    return {"name": name, "op": "gated", "dtype": dtype, "rows": rows, "in": inputs,
            "out": outputs, "act": act, "bias": bias, "train": train}


def listed():
    return [
        # one new row before a wide layer: launch latency is everything
        norm("norm_one_row", "bf16", 1, 4096, residual=True),
        # training over the per-atom states of a 36x36x36 rocksalt box at the EQ hidden width
        norm("norm_atoms_train", "bf16", 373248, 256, residual=True, train=True),
        # float32 states with an odd number of odd rows
        norm("norm_odd_fp32_train", "fp32", 4099, 1001, residual=False, train=True),
        # a long prompt's rows, left in 8 bits with a scale per row for an 8-bit product
        norm("norm_to_8bit", "bf16", 16384, 4096, residual=True, out="e4m3"),
        # one new row through a wide layer: the weights are read once
        linear("linear_one_row", "bf16", 1, 4096, 8192, "silu", bias=True, residual=False),
        # an 8-bit product of a prompt of ordinary length
        linear("linear_8bit", "e4m3", 2048, 4096, 8192, "gelu", bias=True, residual=False),
        # the largest training step: matrix products bound it
        linear("linear_train", "bf16", 8192, 4096, 4096, "gelu", bias=True, residual=True,
               train=True),
        # odd sizes throughout: no row of any matrix starts on 16 bytes
        linear("linear_odd_train", "fp16", 777, 515, 1001, "tanh", bias=True, residual=True,
               train=True),
        # a handful of sequences decoding together
        gated("gated_five_rows", "fp16", 5, 4096, 8192, "silu", bias=False),
        # training over the atoms of a 24x24x24 rocksalt box, EQ hidden and feed-forward widths
        gated("gated_atoms_train", "bf16", 110592, 256, 512, "silu", bias=True, train=True),
        # a prompt through a wide gated layer
        gated("gated_prompt", "bf16", 4096, 4096, 8192, "gelu", bias=False),
        # a ragged training batch of middling width
        gated("gated_ragged_train", "fp16", 4001, 2048, 2816, "silu", bias=False, train=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width spread over its logarithm: a multiple of 8 three times out of four, else any."""
    n = _spread(rng, low, high)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(["norm", "linear", "gated"])
    if op == "norm":
        out = rng.choice(["same", "same", "e4m3"])
        width = _width(rng, 64, 8192)
        rows = min(_spread(rng, 1, 400000), max(1, (1 << 26) // width))
        return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "rows": rows,
                "width": width, "residual": rng.random() < 0.5,
                "train": out == "same" and rng.random() < 0.5, "out": out}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "e4m3"])
    inputs, outputs = _width(rng, 96, 8192), _width(rng, 96, 8192)
    train = dtype != "e4m3" and rng.random() < 0.5
    both = 2 if op == "gated" else 1
    rows = min(_spread(rng, 1, 120000),
               max(1, (1 << (36 if train else 37)) // (inputs * outputs * both)),
               (1 << 28) // (inputs + 3 * both * outputs))
    case = {"op": op, "dtype": dtype, "rows": rows, "in": inputs, "out": outputs,
            "act": rng.choice(["silu", "gelu", "tanh"]), "bias": rng.random() < 0.5,
            "train": train}
    if op == "linear":
        case["act"] = rng.choice(["none", "silu", "gelu", "tanh"])
        case["residual"] = rng.random() < 0.5
    return case


# ------------------------------------------------------------------------------------ the data
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": case}
    rows = case["rows"]
    if case["op"] == "norm":
        dt, width = DTYPES[case["dtype"]], case["width"]
        loud = 1.0 + 7.0 * (torch.rand(width, generator=gen, device="cuda") < 0.02)
        s["x"] = (normal(rows, width) * loud).to(dt)
        s["weight"] = (1.0 + 0.1 * normal(width)).to(dt)
        if case["residual"]:
            s["residual"] = normal(rows, width).to(dt)
        if case["train"]:
            s["dy"] = normal(rows, width).to(dt)
            if case["residual"]:
                s["dh"] = normal(rows, width).to(dt)
    else:
        inputs, outputs = case["in"], case["out"]
        n = 2 * outputs if case["op"] == "gated" else outputs
        x, w = normal(rows, inputs), normal(n, inputs) / math.sqrt(inputs)
        if case["dtype"] == "e4m3":
            for key, t in (("x", x), ("weight", w)):
                scale = t.abs().amax(1, keepdim=True) / E4M3_MAX
                s[key] = (t / scale).to(torch.float8_e4m3fn)
                s[key + "_scale"] = scale.reshape(-1)
            dt = torch.bfloat16
        else:
            dt = DTYPES[case["dtype"]]
            s["x"], s["weight"] = x.to(dt), w.to(dt)
        if case["bias"]:
            s["bias"] = (0.1 * normal(n)).to(dt)
        if case.get("residual"):
            s["residual"] = normal(rows, outputs).to(dt)
        if case["train"]:
            s["dy"] = normal(rows, outputs).to(dt)
    if case["train"]:
        for key in ("x", "weight", "bias", "residual"):
            if key in s:
                s[key].requires_grad_(True)
    return s


def work(case):
    rows, dt = case["rows"], case["dtype"]
    if case["op"] == "norm":
        n, width = rows * case["width"], case["width"]
        b = BYTES[dt]
        if case["out"] == "e4m3":
            moved = n * (b * (3 if case["residual"] else 1) + 1) + 4 * rows + b * width
        else:
            moved = n * b * (4 if case["residual"] else 2) + b * width
        if case["train"]:  # dy, dh and the saved states in; dx out; dweight
            moved += n * b * (4 if case["residual"] else 3) + b * width
        return {"bytes": moved, "flops": n * (12 if case["train"] else 5)}
    n = case["out"] * (2 if case["op"] == "gated" else 1)
    b, ob = BYTES[dt], 2
    moved = b * (rows * case["in"] + n * case["in"]) + ob * rows * case["out"]
    moved += ob * n if case["bias"] else 0
    moved += ob * rows * case["out"] if case.get("residual") else 0
    moved += 4 * (rows + n) if dt == "e4m3" else 0
    flops = 2 * rows * n * case["in"]
    if case["train"]:  # dy, x and the weights in; dx, dweight and dbias out
        moved += ob * rows * case["out"] + 2 * b * (rows * case["in"] + n * case["in"])
        moved += ob * n if case["bias"] else 0
        flops *= 3
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------------- plain forms
def _act(kind, z):
    """(value, derivative) of the activation at z, elementwise."""
    if kind == "tanh":
        t = torch.tanh(z)
        return t, 1.0 - t * t
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if kind == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    return z, torch.ones_like(z)


def _plain_norm(s, case):
    dt = s["x"].dtype
    w = s["weight"].float()
    h = s["x"].float()
    if case["residual"]:
        h = h + s["residual"].float()
    r = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    y = h * r * w
    if case["out"] == "e4m3":
        amax = y.abs().amax(1, keepdim=True)
        scale = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
        out = {"q": (y / scale).to(torch.float8_e4m3fn), "scale": scale.reshape(-1)}
    else:
        out = {"y": y.to(dt)}
    if case["residual"]:
        out["h"] = h.to(dt)
    if case["train"]:
        g = s["dy"].float()
        n = h * r
        gw = g * w
        dx = r * (gw - n * (gw * n).mean(1, keepdim=True))
        if case["residual"]:
            dx = dx + s["dh"].float()
            out["dresidual"] = dx.to(dt)
        out["dx"] = dx.to(dt)
        out["dweight"] = (g * n).sum(0).to(dt)
    return out


def _plain_product(s):
    z = s["x"].float() @ s["weight"].float().t()
    if "x_scale" in s:
        z = z * s["x_scale"][:, None] * s["weight_scale"][None, :]
    return z + s["bias"].float() if "bias" in s else z


def _plain_linear(s, case):
    z = _plain_product(s)
    dt = torch.bfloat16 if case["dtype"] == "e4m3" else s["x"].dtype
    a, da = _act(case["act"], z)
    y = a + s["residual"].float() if case["residual"] else a
    out = {"y": y.to(dt)}
    if case["train"]:
        _plain_gradients(out, s, s["dy"].float() * da, dt)
        if case["residual"]:
            out["dresidual"] = s["dy"]
    return out


def _plain_gated(s, case):
    gate, up = _plain_product(s).chunk(2, dim=1)
    dt = torch.bfloat16 if case["dtype"] == "e4m3" else s["x"].dtype
    a, da = _act(case["act"], gate)
    out = {"y": (a * up).to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        _plain_gradients(out, s, torch.cat([dy * up * da, dy * a], dim=1), dt)
    return out


def _plain_gradients(out, s, dz, dt):
    out["dx"] = (dz @ s["weight"].float()).to(dt)
    out["dweight"] = (dz.t() @ s["x"].float()).to(dt)
    if "bias" in s:
        out["dbias"] = dz.sum(0).to(dt)


# ------------------------------------------------------------------------------ the framework's
def _own_forward(s, case):
    from rune_b200 import ops

    if case["op"] == "norm":
        call = ops.rms_norm_fp8 if case["out"] == "e4m3" else ops.rms_norm
        got = call(s["x"], s["weight"], residual=s.get("residual"), eps=EPS)
        names = ("q", "scale", "h") if case["out"] == "e4m3" else ("y", "h")
        return dict(zip(names, got if isinstance(got, tuple) else (got,)))
    more = {"x_scale": s["x_scale"], "weight_scale": s["weight_scale"]} if "x_scale" in s else {}
    if case["op"] == "linear":
        act = None if case["act"] == "none" else case["act"]
        return {"y": ops.linear(s["x"], s["weight"], bias=s.get("bias"), activation=act,
                                residual=s.get("residual"), **more)}
    return {"y": ops.gated_linear(s["x"], s["weight"], bias=s.get("bias"),
                                  activation=case["act"], **more)}


def _gradients(s, out):
    """out with the gradients of its results for dy (and dh) by automatic differentiation."""
    results, given = [out["y"]], [s["dy"]]
    if "dh" in s:
        results.append(out["h"])
        given.append(s["dh"])
    keys = [k for k in ("x", "weight", "bias", "residual") if k in s]
    found = torch.autograd.grad(results, [s[k] for k in keys], given)
    return {**{k: v.detach() for k, v in out.items()},
            **{"d" + k: g for k, g in zip(keys, found)}}


def run(state):
    case = state["case"]
    if own:
        out = _own_forward(state, case)
        return _gradients(state, out) if case["train"] else out
    with torch.no_grad():
        plain = {"norm": _plain_norm, "linear": _plain_linear, "gated": _plain_gated}
        return plain[case["op"]](state, case)


# --------------------------------------------------------------------------------- the 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach().double().requires_grad_(v.requires_grad) if torch.is_tensor(v) else v
         for k, v in s.items()}
    fn = torch.nn.functional
    acts = {"none": lambda z: z, "tanh": torch.tanh, "silu": fn.silu, "gelu": fn.gelu}
    out = {}
    if case["op"] == "norm":
        h = s["x"] + s["residual"] if case["residual"] else s["x"]
        y = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + EPS) * s["weight"]
        if case["out"] == "e4m3":  # the values before their rounding to 8 bits
            scale = y.abs().amax(-1) / E4M3_MAX
            out = {"q": y / scale[:, None], "scale": scale}
        else:
            out = {"y": y}
        if case["residual"]:
            out["h"] = h
    else:
        x, w = s["x"], s["weight"]
        if "x_scale" in s:
            x, w = x * s["x_scale"][:, None], w * s["weight_scale"][:, None]
        z = fn.linear(x, w, s.get("bias"))
        if case["op"] == "gated":
            n = case["out"]
            out["y"] = acts[case["act"]](z[:, :n]) * z[:, n:]
        else:
            out["y"] = acts[case["act"]](z)
            if case["residual"]:
                out["y"] = out["y"] + s["residual"]
    return _gradients(s, out) if case["train"] else out
