"""Group norm with a gated activation and the gated feed-forward block on the rows of sparse tensors.

Rows are [N, C], channels last, the samples of a batch one behind the other (offsets int32 [B + 1]).  A case is a dict of
plain values; `op` selects the operator, `train` the forward pass alone or with its gradients.

  norm   groups of channel copies normalised per sample, affine parameters, activation: scalars through one
         activation, every field of order l > 0 times the activation of its gate scalar (the last channels)
  ff     y = (act(x Wg' + bg) * (x Wu' + bu)) Wo' + bo (+ residual)

`own` False computes them from elementary operations, True calls the library's operators.
"""
import math
import os
import sys

import torch
import torch.nn.functional as F

own = False

EPS = 1e-5
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one steerable layer's norm and gate on two small objects: latency of a per-object call
        {"name": "norm-small", "op": "norm", "rows": 3501, "batch": 2, "irreps": "2,2,2,2", "groups": 1, "act": "gate",
         "dtype": "fp32", "train": False, "spread": 0.2},
        # norm and gate of a steerable block in training, voxels of eight objects
        {"name": "norm-irreps-train", "op": "norm", "rows": 96011, "batch": 8, "irreps": "4,4,4,4", "groups": 2, "act": "gate",
         "dtype": "fp32", "train": True, "spread": 0.3},
        # per-point features of a training batch of 64 objects with 1024 points, 32 groups
        {"name": "norm-scalars-train", "op": "norm", "rows": 65536, "batch": 64, "irreps": "256", "groups": 32, "act": "silu",
         "dtype": "fp32", "train": True, "spread": 0.0},
        # one large scene: a single sample, all rows share their statistics
        {"name": "norm-scene", "op": "norm", "rows": 203437, "batch": 1, "irreps": "64", "groups": 8, "act": "relu",
         "dtype": "fp32", "train": False, "spread": 0.0},
        # stored 16-bit features of a large batch, more than the L2 cache holds
        {"name": "norm-large-bf16", "op": "norm", "rows": 786432, "batch": 256, "irreps": "128", "groups": 16, "act": "silu",
         "dtype": "bf16", "train": False, "spread": 0.4},
        # ragged samples, an empty one, channel counts that no vector width divides
        {"name": "norm-ragged-fp16-train", "op": "norm", "rows": 50021, "batch": 37, "irreps": "9,3,3", "groups": 3, "act": "gate",
         "dtype": "fp16", "train": True, "spread": 0.9},
        # the head on the pooled feature of a single object
        {"name": "ff-token", "op": "ff", "rows": 1, "c": 256, "hidden": 1024, "out": 256, "act": "silu", "bias": False,
         "residual": True, "dtype": "bf16", "train": False},
        # the same on the pooled features of a batch, full precision
        {"name": "ff-batch", "op": "ff", "rows": 64, "c": 256, "hidden": 512, "out": 128, "act": "gelu", "bias": True,
         "residual": False, "dtype": "fp32", "train": False},
        # per-point block in full precision, training
        {"name": "ff-points-train", "op": "ff", "rows": 16384, "c": 128, "hidden": 512, "out": 128, "act": "silu", "bias": False,
         "residual": True, "dtype": "fp32", "train": True},
        # per-point block of a training batch of 64 objects with 1024 points in 16 bits
        {"name": "ff-points-train-bf16", "op": "ff", "rows": 65536, "c": 256, "hidden": 1024, "out": 256, "act": "silu",
         "bias": False, "residual": True, "dtype": "bf16", "train": True},
        # inference on the points of a large batch, wide rows
        {"name": "ff-large-bf16", "op": "ff", "rows": 131072, "c": 512, "hidden": 2048, "out": 512, "act": "silu", "bias": False,
         "residual": True, "dtype": "bf16", "train": False},
        # widths that are no multiple of a tile, biases, another output width
        {"name": "ff-odd-fp16-train", "op": "ff", "rows": 10007, "c": 100, "hidden": 300, "out": 76, "act": "gelu", "bias": True,
         "residual": False, "dtype": "fp16", "train": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype, train = rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.5
    if rng.random() < 0.5:
        if rng.random() < 0.5:
            groups = rng.choice([1, 2, 4, 8, 16, 32])
            irreps, act = str(groups * _log_int(rng, 1, max(1, 256 // groups))), rng.choice(["silu", "gelu", "relu", "none"])
        else:
            groups = rng.choice([1, 1, 2, 3])
            irreps = ",".join(str(groups * rng.randint(1, 6)) for _ in range(rng.randint(2, 4)))
            act = "gate"
        c = sum(int(m) * (2 * l + 1) for l, m in enumerate(irreps.split(",")))
        rows = _log_int(rng, 1000, min(500000, 30_000_000 // c))
        return {"op": "norm", "rows": rows, "batch": _log_int(rng, 1, 256), "irreps": irreps, "groups": groups, "act": act,
                "dtype": dtype, "train": train, "spread": round(rng.random() * 0.9, 2)}
    c, hidden = _log_int(rng, 16, 512), _log_int(rng, 32, 2048)
    if rng.random() < 0.6:
        c, hidden = max(16, c // 16 * 16), max(32, hidden // 32 * 32)
    out = c if rng.random() < 0.5 else _log_int(rng, 16, 512)
    residual = out == c and rng.random() < 0.7
    most = int(1.2e11 / (c + out) / hidden / (3 if train else 1))
    return {"op": "ff", "rows": _log_int(rng, 1, max(2, min(131072, most))), "c": c, "hidden": hidden, "out": out,
            "act": rng.choice(["silu", "gelu", "relu"]), "bias": rng.random() < 0.5, "residual": residual, "dtype": dtype, "train": train}


# ------------------------------------------------------------------------------------- inputs
def _layout(case):
    """Rs of the input rows [(copies, order), ...]; a gated norm's last entry holds one scalar for each field of order l > 0."""
    Rs = [(int(m), l) for l, m in enumerate(case["irreps"].split(","))]
    gates = sum(m for m, l in Rs if l > 0) if case["act"] == "gate" else 0
    # (the gates are as many as the fields, and those of every order are a multiple of the groups)
    return Rs + ([(gates, 0)] if gates else []), gates


def _lengths(case, seed):
    """Rows of each sample: `spread` 0 gives samples of one size, near 1 very different ones, the second of them empty."""
    b, n = case["batch"], case["rows"]
    g = torch.Generator().manual_seed(seed + 7)
    share = 1.0 - case["spread"] * torch.rand(b, generator=g, dtype=torch.float64)
    if b > 1 and case["spread"] > 0.5:
        share[1] = 0.0
    ends = torch.round(share.cumsum(0) / share.sum() * n).long()
    ends[-1] = n
    return torch.cat([torch.zeros(1, dtype=torch.long), ends])


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def leaf(v, kind=t):
        return v.to(kind).requires_grad_(case["train"])

    n, state = case["rows"], {"case": case}
    if case["op"] == "norm":
        Rs, gates = _layout(case)
        c, fields, scalars = sum(m * (2 * l + 1) for m, l in Rs), sum(m for m, l in Rs), sum(m for m, l in Rs if l == 0)
        # what a convolution leaves: channels of different sizes, scalars off centre
        state["x"] = leaf(normal(n, c) * (0.5 + torch.rand(c, generator=g, device="cuda")) + 0.8 * normal(c))
        state["offsets"] = _lengths(case, seed).int().cuda()
        state["weight"], state["bias"] = leaf(1 + 0.2 * normal(fields), torch.float32), leaf(0.2 * normal(scalars), torch.float32)
        state["gy"] = normal(n, c - gates).to(t) if case["train"] else None
        return state
    c, h, o = case["c"], case["hidden"], case["out"]
    state["x"] = leaf(normal(n, c))
    state["w_in"], state["w_out"] = leaf(normal(2, h, c) / math.sqrt(c)), leaf(normal(o, h) / math.sqrt(h))
    state["b_in"] = leaf(0.2 * normal(2, h)) if case["bias"] else None
    state["b_out"] = leaf(0.2 * normal(o)) if case["bias"] else None
    state["residual"] = normal(n, o).to(t) if case["residual"] else None
    state["gy"] = normal(n, o).to(t) if case["train"] else None
    return state


# ------------------------------------------------------------------------------------- the library's operators
_ACT = {"none": None, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gate": (F.relu, torch.sigmoid)}


def _library():
    path = os.path.join(os.getcwd(), "ss-conv_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from ss_conv.feedforward import gated_feedforward
    from ss_conv.groupnorm import group_norm
    return group_norm, gated_feedforward


def _own(s):
    case = s["case"]
    group_norm, gated_feedforward = _library()
    if case["op"] == "norm":
        y = group_norm(s["x"], s["offsets"], _layout(case)[0], case["groups"], s["weight"], s["bias"], EPS, _ACT[case["act"]])
        wanted = ["x", "weight", "bias"]
    else:
        y = gated_feedforward(s["x"], s["w_in"], s["w_out"], s["b_in"], s["b_out"], _ACT[case["act"]], s["residual"])
        wanted = ["x", "w_in", "w_out"] + (["b_in", "b_out"] if case["bias"] else [])
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [s[k] for k in wanted], s["gy"])
    return {"y": y.detach(), **{"g_" + k: v for k, v in zip(wanted, grads)}}


# ------------------------------------------------------------------------------------- plain forms
def _value(act, z):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _slope(act, z):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 - s)
    return torch.ones_like(z)


def _tables(Rs, groups, device):
    """Per channel: group, field, scalar slot (-1 for l > 0); per group: copies in it."""
    group, field, scalar, copies = [], [], [], []
    f = s = 0
    for m, l in Rs:
        each = m // groups
        for k in range(m):
            group += [len(copies) + k // each] * (2 * l + 1)
            field += [f + k] * (2 * l + 1)
            scalar += [s + k if l == 0 else -1] * (2 * l + 1)
        copies += [each] * groups
        f, s = f + m, s + (m if l == 0 else 0)
    return [torch.tensor(v, device=device) for v in (group, field, scalar, copies)]


def _per_sample(v, offsets):
    """Sums of rows v [N, k] over each sample, in 64 bits."""
    # (one running sum down the columns, one column behind the other)
    run = torch.zeros(v.numel() + 1, dtype=torch.float64, device=v.device)
    torch.cumsum(v.t().reshape(-1), 0, dtype=torch.float64, out=run[1:])
    at = torch.arange(v.shape[1], device=v.device) * v.shape[0]
    return run[offsets[1:, None] + at] - run[offsets[:-1, None] + at]


def _plain_norm(s):
    case = s["case"]
    x, offsets = s["x"].detach().float(), s["offsets"].long()
    Rs, gates = _layout(case)
    group, field, scalar, copies = _tables(Rs, case["groups"], x.device)
    centred = scalar >= 0
    is_mean = torch.zeros(copies.numel(), dtype=torch.bool, device=x.device).index_put_((group,), centred)
    member = (group[:, None] == torch.arange(copies.numel(), device=x.device)).float()        # [C, groups]
    count = ((offsets[1:] - offsets[:-1])[:, None] * copies).clamp(min=1).double()
    row = torch.bucketize(torch.arange(x.shape[0], device=x.device), offsets[1:], right=True)
    w, b = s["weight"].detach()[field], torch.where(centred, s["bias"].detach()[scalar.clamp(min=0)], torch.zeros(()).cuda())
    mu = torch.where(is_mean, _per_sample(x @ member, offsets) / count, torch.zeros((), dtype=torch.float64, device=x.device)).float()
    d = x - mu[row][:, group]
    r = (1 / torch.sqrt(_per_sample((d * d) @ member, offsets) / count + EPS)).float()[row][:, group]
    hat = d * r
    z = hat * w + b
    act = case["act"]
    if act == "gate":
        m0, body = Rs[0][0], z.shape[1] - gates
        gate = (field[m0:body] - m0)                                                         # of each channel with l > 0
        sig = _value("sigmoid", z[:, body:])
        y = torch.cat([_value("relu", z[:, :m0]), z[:, m0:body] * sig[:, gate]], 1)
    else:
        y = _value(act, z)
    t = s["x"].dtype
    if not case["train"]:
        return {"y": y.to(t)}
    gy = s["gy"].float()
    if act == "gate":
        by_gate = (gate[:, None] == torch.arange(gates, device=x.device)).float()
        dz = torch.cat([gy[:, :m0] * _slope("relu", z[:, :m0]), gy[:, m0:] * sig[:, gate],
                        ((gy[:, m0:] * z[:, m0:body]) @ by_gate) * _slope("sigmoid", z[:, body:])], 1)
    else:
        dz = gy * _slope(act, z)
    a = dz * w
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    s1 = torch.where(is_mean, _per_sample(a @ member, offsets) / count, zero).float()[row][:, group]
    s2 = (_per_sample((a * hat) @ member, offsets) / count).float()[row][:, group]
    gx = r * (a - s1 - hat * s2)
    gw = torch.zeros_like(s["weight"], dtype=torch.float64).index_add_(0, field, (dz * hat).sum(0, dtype=torch.float64))
    gb = dz.sum(0, dtype=torch.float64)[centred]
    return {"y": y.to(t), "g_x": gx.to(t), "g_weight": gw.float(), "g_bias": gb.float()}


def _plain_ff(s):
    case, t = s["case"], s["x"].dtype
    x, wg, wu, wo = s["x"].detach().float(), s["w_in"][0].detach().float(), s["w_in"][1].detach().float(), s["w_out"].detach().float()
    g, u = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        g, u = g + s["b_in"][0].detach().float(), u + s["b_in"][1].detach().float()
    a = _value(case["act"], g)
    h = a * u
    y = h @ wo.t()
    if case["bias"]:
        y = y + s["b_out"].detach().float()
    if case["residual"]:
        y = y + s["residual"].float()
    if not case["train"]:
        return {"y": y.to(t)}
    gy = s["gy"].float()
    dh = gy @ wo
    du, dg = dh * a, dh * u * _slope(case["act"], g)
    out = {"y": y.to(t), "g_x": (dg @ wg + du @ wu).to(t), "g_w_in": torch.stack([dg.t() @ x, du.t() @ x]).to(t),
           "g_w_out": (gy.t() @ h).to(t)}
    if case["bias"]:
        out["g_b_in"] = torch.stack([dg.sum(0, dtype=torch.float64), du.sum(0, dtype=torch.float64)]).to(t)
        out["g_b_out"] = gy.sum(0, dtype=torch.float64).to(t)
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_norm(state) if state["case"]["op"] == "norm" else _plain_ff(state)


def work(case):
    n, size = case["rows"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        Rs, gates = _layout(case)
        c = sum(m * (2 * l + 1) for m, l in Rs)
        cells = n * (2 * c - gates)
        return {"bytes": size * cells * (2 if case["train"] else 1), "flops": (25 if case["train"] else 10) * n * c}
    c, h, o = case["c"], case["hidden"], case["out"]
    rows, weights = n * (c + o), 2 * h * c + h * o
    flops = 2 * n * weights
    if case["train"]:
        return {"bytes": size * (2 * rows + 2 * weights + (n * o if case["residual"] else 0)), "flops": 3 * flops}
    return {"bytes": size * (rows + weights + (n * o if case["residual"] else 0)), "flops": flops}


# ------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_activation(act, z):
    return {"none": lambda v: v, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}[act](z)


def _exact_norm(case, x, weight, bias, bounds):
    Rs, gates = _layout(case)
    body = x.shape[1] - gates
    parts = []
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        if hi == lo:
            continue
        fields, ch, f, sc = [], 0, 0, 0
        for m, l in Rs:
            d = 2 * l + 1
            v = x[lo:hi, ch:ch + m * d].reshape(hi - lo, case["groups"], -1, d)
            if l == 0:
                v = v - v.mean(dim=(0, 2, 3), keepdim=True)
            v = v / torch.sqrt((v * v).sum(3, keepdim=True).mean(dim=(0, 2), keepdim=True) + EPS)
            v = v.reshape(hi - lo, m, d) * weight[f:f + m, None]
            if l == 0:
                v = v + bias[sc:sc + m, None]
                sc += m
            fields.append(v)
            ch, f = ch + m * d, f + m
        if case["act"] != "gate":
            parts.append(_exact_activation(case["act"], fields[0].reshape(hi - lo, -1)))
            continue
        gate, used, rows = torch.sigmoid(fields.pop()), 0, []
        for k, v in enumerate(fields):
            if k == 0:
                v = F.relu(v)
            else:
                v, used = v * gate[:, used:used + v.shape[1]], used + v.shape[1]
            rows.append(v.reshape(hi - lo, -1))
        parts.append(torch.cat(rows, 1))
    return torch.cat(parts) if parts else x.new_zeros(0, body)


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: (v.detach().double().requires_grad_(v.requires_grad) if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in s.items()}
    if case["op"] == "norm":
        y = _exact_norm(case, d["x"], d["weight"], d["bias"], s["offsets"].tolist())
        wanted = ["x", "weight", "bias"]
    else:
        both = torch.einsum("nc,khc->knh", d["x"], d["w_in"])
        if case["bias"]:
            both = both + d["b_in"][:, None]
        y = F.linear(_exact_activation(case["act"], both[0]) * both[1], d["w_out"], d["b_out"])
        if case["residual"]:
            y = y + d["residual"]
        wanted = ["x", "w_in", "w_out"] + (["b_in", "b_out"] if case["bias"] else [])
    if not case["train"]:
        return {"y": y.detach()}
    grads = torch.autograd.grad(y, [d[k] for k in wanted], d["gy"])
    return {"y": y.detach(), **{"g_" + k: v for k, v in zip(wanted, grads)}}
