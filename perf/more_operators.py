"""Workloads of the operators of ``rune_b200.ops`` whose weights depend on the row, and of the
optimiser's update: routing rows to experts, sorting rows by group and back, the groups' linear
and gated layers, orthogonalised updates.

Each case is one pass of one operator, forward alone (serving) or forward and backward
(training). Rows choose their groups as elements or experts are met: some groups many times more
often than others, some not at all, and some rows in none.

``run`` computes the plain form in float32 (elementary torch operations, one rounding at the
end) where ``own`` is false, and calls ``rune_b200.ops`` where it is true. ``exact`` evaluates
the definitions in float64 by automatic differentiation, apart from both.
"""

import math

import torch

own = False

EPS = 1.0e-7
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ----------------------------------------------------------------------------------- the cases
def route(name, dtype, rows, groups, k, train=False):
    return {"name": name, "op": "route", "dtype": dtype, "rows": rows, "groups": groups, "k": k,
            "train": train}


def sort(name, dtype, rows, width, groups, k, dropped=0.0, train=False):
    return {"name": name, "op": "sort", "dtype": dtype, "rows": rows, "width": width,
            "groups": groups, "k": k, "dropped": dropped, "train": train}


def grouped(name, dtype, rows, inputs, outputs, groups, act, gated, bias, dropped=0.0, train=False):
    return {"name": name, "op": "grouped", "dtype": dtype, "rows": rows, "in": inputs,
            "out": outputs, "groups": groups, "act": act, "gated": gated, "bias": bias,
            "dropped": dropped, "train": train}


def orthogonal(name, dtype, batch, m, n, steps=5):
    return {"name": name, "op": "orthogonal", "dtype": dtype, "batch": batch, "m": m, "n": n,
            "steps": steps}


def listed():
    return [
        # one new row's choice among the experts: launch latency is everything
        route("route_one_row", "bf16", 1, 64, 2),
        # a training batch's rows among many experts, with the router's gradient
        route("route_train", "fp32", 16384, 256, 8, train=True),
        # a handful of rows to their experts and back
        sort("sort_five_rows", "bf16", 5, 4096, 64, 2),
        # training: the atoms of a 24x24x24 rocksalt box at the EQ hidden width, two experts each
        sort("sort_atoms_train", "bf16", 110592, 256, 8, 2, train=True),
        # float32 states by element, 89 of them, odd width, some rows without a network
        sort("sort_elements_train", "fp32", 32001, 515, 89, 1, dropped=0.1, train=True),
        # a handful of rows through their experts' gated layers: the weights are read once
        grouped("experts_ten_rows", "fp16", 10, 4096, 2048, 16, "silu", gated=True, bias=False),
        # NEP's per-element networks on the descriptors of a 20x20x20 ternary alloy
        grouped("elements_train", "bf16", 32000, 35, 30, 3, "tanh", gated=False, bias=True, train=True),
        # the experts' gated layers over the atoms of a 24x24x24 rocksalt box, two experts each
        grouped("experts_atoms_train", "bf16", 221184, 256, 512, 8, "silu", gated=True, bias=True,
                train=True),
        # a long prompt's rows through many wide experts
        grouped("experts_prompt", "bf16", 32768, 2048, 4096, 64, "gelu", gated=False, bias=False),
        # a ragged training batch, more groups than the rows fill, some rows in none
        grouped("experts_ragged_train", "fp16", 8001, 1024, 1408, 61, "silu", gated=True, bias=False,
                dropped=0.05, train=True),
        # the hidden matrices of a small network, one update
        orthogonal("update_small", "fp32", 8, 256, 512),
        # a wide layer's update
        orthogonal("update_wide", "bf16", 1, 4096, 4096),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width spread over its logarithm: a multiple of 8 three times out of four, else any."""
    n = _spread(rng, low, high)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(["route", "sort", "grouped", "grouped", "grouped", "orthogonal"])
    train, groups = rng.random() < 0.5, _spread(rng, 2, 256)
    if op == "route":
        rows = _spread(rng, 1, 131072)
        return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "rows": rows,
                "groups": groups, "k": min(groups, _spread(rng, 1, 8)), "train": train}
    dropped = rng.choice([0.0, 0.0, 0.1])
    if op == "sort":
        width, k = _width(rng, 32, 8192), min(groups, _spread(rng, 1, 8))
        rows = min(_spread(rng, 1, 131072), max(1, (1 << 25) // (width * k)))
        return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "rows": rows,
                "width": width, "groups": groups, "k": k, "dropped": dropped, "train": train}
    if op == "grouped":
        inputs, outputs, gated = _width(rng, 32, 4096), _width(rng, 16, 4096), rng.random() < 0.5
        both = 2 if gated else 1
        groups = min(groups, max(2, (1 << 28) // (inputs * outputs * both)))
        rows = min(_spread(rng, 1, 200000),
                   max(1, (1 << (35 if train else 36)) // (inputs * outputs * both)),
                   (1 << 27) // (inputs + 3 * both * outputs))
        act = rng.choice(["silu", "gelu", "tanh"] if gated else ["none", "silu", "gelu", "tanh"])
        return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "rows": rows, "in": inputs,
                "out": outputs, "groups": groups, "act": act, "gated": gated,
                "bias": rng.random() < 0.5, "dropped": dropped, "train": train}
    m, n = _width(rng, 64, 4096), _width(rng, 64, 4096)
    batch = min(_spread(rng, 1, 32), max(1, (1 << 36) // (m * n * min(m, n))))
    return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "batch": batch, "m": m,
            "n": n, "steps": rng.choice([3, 5, 5, 6])}


# ------------------------------------------------------------------------------------ the data
def _popularity(groups, gen):
    """Logits of the groups' shares: a few times as many rows for some as for others."""
    return torch.randn(groups, generator=gen, device="cuda")


def _choice(case, gen, k):
    """[rows, k] different groups of each row, int32; -1 where a row has none."""
    rows, groups = case["rows"], case["groups"]
    u = torch.rand(rows, groups, generator=gen, device="cuda").clamp_(1.0e-9, 1.0 - 1.0e-7)
    score = _popularity(groups, gen) - torch.log(-torch.log(u))
    index = score.topk(k, dim=1).indices.to(torch.int32)
    if case["dropped"]:
        index[torch.rand(rows, k, generator=gen, device="cuda") < case["dropped"]] = -1
    return index


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s, op, dt = {"case": case}, case["op"], DTYPES[case["dtype"]]
    leaves = ()
    if op == "route":
        rows, groups, k = case["rows"], case["groups"], case["k"]
        s["logits"] = (normal(rows, groups) + _popularity(groups, gen)).to(dt)
        if case["train"]:
            s["dweights"] = normal(rows, k)
            leaves = ("logits",)
    elif op == "sort":
        rows, width, k = case["rows"], case["width"], case["k"]
        s["index"] = _choice(case, gen, k)
        s["x"], s["y"] = normal(rows, width).to(dt), normal(rows * k, width).to(dt)
        s["weights"] = torch.softmax(normal(rows, k), 1)
        if case["train"]:
            s["dxs"], s["dout"] = normal(rows * k, width).to(dt), normal(rows, width).to(dt)
            leaves = ("x", "y", "weights")
    elif op == "grouped":
        rows, inputs, groups = case["rows"], case["in"], case["groups"]
        n = case["out"] * (2 if case["gated"] else 1)
        index = _choice(case, gen, 1).reshape(-1)
        key = torch.where(index < 0, groups, index)
        order = torch.argsort(key, stable=True).to(torch.int32)
        place = torch.empty_like(order)
        place[order.long()] = torch.arange(rows, device="cuda", dtype=torch.int32)
        offsets = torch.searchsorted(key[order.long()].contiguous(),
                                     torch.arange(groups + 1, device="cuda", dtype=torch.int32))
        s["offsets"], s["order"] = offsets.to(torch.int32), order
        s["place"] = torch.where(index < 0, -1, place)
        s["order"][int(offsets[-1]):] = -1
        s["bounds"] = offsets.tolist()
        s["x"] = normal(rows, inputs).to(dt)
        s["weight"] = (normal(groups, n, inputs) / math.sqrt(inputs)).to(dt)
        if case["bias"]:
            s["bias"] = (0.1 * normal(groups, n)).to(dt)
        if case["train"]:
            s["dy"] = normal(rows, case["out"]).to(dt)
            leaves = ("x", "weight", "bias")
    else:
        # a gradient: noise, and a few directions in which it is louder
        b, m, n = case["batch"], case["m"], case["n"]
        x = normal(b, m, n)
        r = min(4, m, n)
        x = x + normal(b, m, r) @ normal(b, r, n) / math.sqrt(r)
        s["x"] = (1.0e-3 * x).to(dt)
    for key in leaves:
        if key in s:
            s[key].requires_grad_(True)
    return s


def work(case):
    op, b = case["op"], BYTES[case["dtype"]]
    if op == "route":
        n, chosen = case["rows"] * case["groups"], case["rows"] * case["k"]
        moved = n * b + 8 * chosen
        if case["train"]:  # the weights' gradients and the choices in, the logits' gradients out
            moved += n * b + 12 * chosen
        return {"bytes": moved, "flops": n * case["k"]}
    if op == "sort":
        n, slots = case["rows"] * case["width"], case["rows"] * case["k"]
        wide = slots * case["width"]
        moved = b * (2 * n + 2 * wide) + 16 * slots + 4 * case["groups"]
        if case["train"]:  # dxs, dout and y in, dx, dy and dweights out
            moved += b * (2 * n + 3 * wide) + 8 * slots
        return {"bytes": moved, "flops": wide * (7 if case["train"] else 2)}
    if op == "grouped":
        n = case["out"] * (2 if case["gated"] else 1)
        met = min(case["groups"], case["rows"])  # groups whose weights have to be read
        weights = n * case["in"] * b
        moved = b * case["rows"] * (case["in"] + case["out"]) + met * weights
        moved += met * n * b if case["bias"] else 0
        flops = 2 * case["rows"] * n * case["in"]
        if case["train"]:  # dy, x and the weights in; dx, dweight and dbias out
            moved += b * case["rows"] * (2 * case["in"] + case["out"])
            moved += (met + case["groups"]) * weights
            moved += case["groups"] * n * b if case["bias"] else 0
            flops *= 3
        return {"bytes": moved, "flops": flops}
    small, large = sorted((case["m"], case["n"]))
    size = case["batch"] * small * large
    # of the two symmetric products half the values are needed
    return {"bytes": size * (b + 2),
            "flops": case["steps"] * case["batch"] * (3 * small * small * large + small ** 3)}


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


def _plain_route(s, case):
    logits, k = s["logits"].float(), case["k"]
    value, index = torch.sort(logits, dim=1, descending=True, stable=True)
    value, index = value[:, :k], index[:, :k]
    e = torch.exp(value - value[:, :1])
    w = e / e.sum(1, keepdim=True)
    out = {"index": index.to(torch.int32), "weights": w}
    if case["train"]:
        g = s["dweights"]
        d = w * (g - (w * g).sum(1, keepdim=True))
        out["dlogits"] = torch.zeros_like(logits).scatter(1, index, d).to(s["logits"].dtype)
    return out


def _plain_sort(s, case):
    index, groups, k, dt = s["index"], case["groups"], case["k"], s["x"].dtype
    flat = index.reshape(-1)
    key = torch.where((flat >= 0) & (flat < groups), flat, groups)
    order = torch.argsort(key, stable=True)
    slots = torch.arange(flat.numel(), device=flat.device)
    offsets = torch.searchsorted(key[order], torch.arange(groups + 1, device=flat.device,
                                                          dtype=key.dtype))
    held = slots < offsets[-1]
    place = torch.empty_like(order)
    place[order] = torch.where(held, slots, -1)
    rows, inside = order // k, (place >= 0)[:, None]
    xs = torch.where(held[:, None], s["x"][rows], 0)
    w = torch.where(inside, s["weights"].reshape(-1, 1), 0)
    back = torch.where(inside, s["y"].float()[place.clamp(min=0)], 0)
    out = {"offsets": offsets.to(torch.int32),
           "order": torch.where(held, order, -1).to(torch.int32),
           "place": place.reshape(index.shape).to(torch.int32), "xs": xs,
           "out": (back * w).reshape(*index.shape, -1).sum(1).to(dt)}
    if case["train"]:
        dxs = torch.where(inside, s["dxs"].float()[place.clamp(min=0)], 0)
        out["dx"] = dxs.reshape(*index.shape, -1).sum(1).to(dt)
        dout = s["dout"].float()
        out["dy"] = torch.where(held[:, None], dout[rows] * w[order], 0).to(dt)
        out["dweights"] = (dout[slots // k] * back).sum(1).reshape(index.shape)
    return out


def _plain_grouped(s, case):
    x, weight, dt = s["x"].float(), s["weight"].float(), s["x"].dtype
    bias = s["bias"].float() if "bias" in s else None
    n, train = case["out"], case["train"]
    y = x.new_zeros(case["rows"], n)
    if train:
        dx, dw = torch.zeros_like(x), torch.zeros_like(weight)
        db = torch.zeros_like(bias) if bias is not None else None
        dy = s["dy"].float()
    for g, (a, b) in enumerate(zip(s["bounds"], s["bounds"][1:])):
        if a == b:
            continue
        z = x[a:b] @ weight[g].t()
        if bias is not None:
            z = z + bias[g]
        if case["gated"]:
            gate, up = z[:, :n], z[:, n:]
            v, d = _act(case["act"], gate)
            y[a:b] = v * up
            dz = torch.cat([dy[a:b] * up * d, dy[a:b] * v], dim=1) if train else None
        else:
            y[a:b], d = _act(case["act"], z)
            dz = dy[a:b] * d if train else None
        if train:
            dx[a:b], dw[g] = dz @ weight[g], dz.t() @ x[a:b]
            if bias is not None:
                db[g] = dz.sum(0)
    out = {"y": y.to(dt)}
    if train:
        out["dx"], out["dweight"] = dx.to(dt), dw.to(dt)
        if bias is not None:
            out["dbias"] = db.to(dt)
    return out


def _plain_orthogonal(s, case):
    x = s["x"].float()
    a, b, c = COEFFICIENTS
    x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + EPS)
    turned = x.size(1) > x.size(2)
    if turned:
        x = x.transpose(1, 2)
    for _ in range(case["steps"]):
        g = x @ x.transpose(1, 2)
        x = a * x + (b * g + c * (g @ g)) @ x
    return {"update": (x.transpose(1, 2) if turned else x).to(torch.bfloat16)}


# ------------------------------------------------------------------------------ the framework's
def _own(s, case):
    from rune_b200 import ops

    if case["op"] == "route":
        index, weights = ops.route(s["logits"], case["k"])
        return {"index": index, "weights": weights}
    if case["op"] == "sort":
        groups = ops.row_groups(s["index"], case["groups"])
        return {"offsets": groups.offsets, "order": groups.order, "place": groups.place,
                "xs": ops.to_groups(s["x"], groups),
                "out": ops.from_groups(s["y"], groups, s["weights"])}
    if case["op"] == "grouped":
        groups = ops.RowGroups(s["offsets"], s["order"], s["place"])
        call = ops.grouped_gated_linear if case["gated"] else ops.grouped_linear
        act = None if case["act"] == "none" else case["act"]
        return {"y": call(s["x"], s["weight"], groups, bias=s.get("bias"), activation=act)}
    return {"update": ops.orthogonalize(s["x"], steps=case["steps"], coefficients=COEFFICIENTS,
                                        eps=EPS)}


def _gradients(s, out):
    """out with the gradients of its results for what is given of them."""
    pairs = [(out[k], s["d" + k]) for k in ("weights", "xs", "out", "y") if "d" + k in s]
    keys = [k for k in ("logits", "x", "y", "weights", "weight", "bias")
            if k in s and s[k].requires_grad]
    found = torch.autograd.grad([p[0] for p in pairs], [s[k] for k in keys],
                                [p[1] for p in pairs])
    return {**{k: v.detach() for k, v in out.items()},
            **{"d" + k: g for k, g in zip(keys, found)}}


def run(state):
    case = state["case"]
    if own:
        out = _own(state, case)
        return _gradients(state, out) if case.get("train") else out
    with torch.no_grad():
        plain = {"route": _plain_route, "sort": _plain_sort, "grouped": _plain_grouped,
                 "orthogonal": _plain_orthogonal}
        return plain[case["op"]](state, case)


# --------------------------------------------------------------------------------- the 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach().double().requires_grad_(v.requires_grad)
         if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    fn = torch.nn.functional
    if case["op"] == "route":
        logits, n = s["logits"], case["groups"]
        # the rank of every logit: how many come before it
        index = torch.empty(case["rows"], case["k"], dtype=torch.int64, device="cuda")
        flat = logits.detach().clone()
        for j in range(case["k"]):
            top = flat.amax(1, keepdim=True)
            at = torch.where(flat == top, torch.arange(n, device="cuda"), n).amin(1)
            index[:, j] = at
            flat.scatter_(1, at[:, None], -math.inf)
        out = {"index": index.to(torch.int32),
               "weights": torch.softmax(logits.gather(1, index), 1)}
    elif case["op"] == "sort":
        rows, k, groups = case["rows"], case["k"], case["groups"]
        flat = s["index"].reshape(-1).long()
        member = torch.nonzero((flat >= 0) & (flat < groups)).reshape(-1)
        counts = torch.bincount(flat[member], minlength=groups)
        offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        slot = member[torch.sort(flat[member] * flat.numel() + member).indices]
        order, place = torch.full_like(flat, -1), torch.full_like(flat, -1)
        order[:slot.numel()] = slot
        place[slot] = torch.arange(slot.numel(), device="cuda")
        xs = s["x"].new_zeros(rows * k, case["width"])
        xs = torch.cat([s["x"][slot // k], xs[slot.numel():]])
        parts = s["y"][:slot.numel()] * s["weights"].reshape(-1)[slot][:, None]
        summed = torch.zeros_like(s["x"]).index_add(0, slot // k, parts)
        out = {"offsets": offsets.to(torch.int32), "order": order.to(torch.int32),
               "place": place.reshape(rows, k).to(torch.int32), "xs": xs, "out": summed}
    elif case["op"] == "grouped":
        acts = {"none": lambda z: z, "tanh": torch.tanh, "silu": fn.silu, "gelu": fn.gelu}
        parts, n = [], case["out"]
        for g in range(case["groups"]):
            rows = s["x"][s["bounds"][g]:s["bounds"][g + 1]]
            z = fn.linear(rows, s["weight"][g], s["bias"][g] if case["bias"] else None)
            a = acts[case["act"]]
            parts.append(a(z[:, :n]) * z[:, n:] if case["gated"] else a(z))
        parts.append(s["x"].new_zeros(case["rows"] - s["bounds"][-1], n))
        out = {"y": torch.cat(parts)}
    else:
        a, b, c = COEFFICIENTS
        x = s["x"] / (torch.linalg.matrix_norm(s["x"], keepdim=True) + EPS)
        for _ in range(case["steps"]):
            if case["m"] <= case["n"]:
                g = torch.bmm(x, x.mT)
                x = a * x + b * torch.bmm(g, x) + c * torch.bmm(g, torch.bmm(g, x))
            else:
                g = torch.bmm(x.mT, x)
                x = a * x + b * torch.bmm(x, g) + c * torch.bmm(torch.bmm(x, g), g)
        out = {"update": x}
    return _gradients(s, out) if case.get("train") else out
