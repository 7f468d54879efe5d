"""Definitions of the row operators in 64 bits, value by value with the terms that each value is made of: a result in float32 may be off by so
many half steps (2^-24) of those, whatever cancels."""
import torch
import torch.nn.functional as F

HALF = 2.0 ** -24


def activation(act, z):
    """(value, slope), neither of them rounded."""
    z = z.detach().requires_grad_(True)
    v = z * 1 if act is None else act(z)
    return v.detach(), torch.autograd.grad(v.sum(), [z])[0]


def group_norm(x, offsets, Rs, groups, w, b, eps, act, gy):
    """Group norm of the samples with its gradients for gy (None: none): {"y", "x", "weight", "bias"} -> (value, terms); parameters' terms are the
    root of the sum of the squares of what they are summed from, their errors go either way.  "gy" is gy with zeros where ReLU's slope
    may fall on either side.

    A normalised value is off by half steps of (|x| + mean |x|) r, what the activation makes of it by its slope or that of the slope, both
    below 1.13."""
    scalar, gate = act if isinstance(act, tuple) else (act, act)
    layout = [(m, l) for m, l in Rs if m > 0]
    n_gate = sum(m for m, l in layout if l > 0) if gate is not None else 0
    c_out = x.shape[1] - n_gate
    fields, first, ch = [], [], 0                # (order, group) of each field, its first channel
    for e, (m, l) in enumerate(layout):
        for k in range(m):
            fields.append((l, e * groups + k // (m // groups)))
            first.append(ch)
            ch += 2 * l + 1
    field = torch.tensor([i for i, (l, _) in enumerate(fields) for _ in range(2 * l + 1)])
    is_scalar = torch.tensor([fields[i][0] == 0 for i in field.tolist()])
    group = torch.tensor([fields[i][1] for i in field.tolist()])
    n_group = int(group.max()) + 1
    copies = torch.tensor([sum(1 for l, k in fields if k == g) for g in range(n_group)], dtype=torch.float64)
    member = (group[:, None] == torch.arange(n_group)).double()
    slot = torch.cumsum(torch.tensor([l == 0 for l, _ in fields]).long(), 0) - 1
    weight = torch.ones(len(fields), dtype=torch.float64) if w is None else w
    wc = weight[field]
    bc = torch.where(is_scalar, b[slot[field].clamp(min=0)], 0.0) if b is not None else torch.zeros(x.shape[1], dtype=torch.float64)
    mean_of = torch.tensor([any(l == 0 and k == g for l, k in fields) for g in range(n_group)])
    vectors = [i for i, (l, _) in enumerate(fields) if l > 0]
    gate_field = torch.arange(len(fields) - n_gate, len(fields))
    out = {k: [torch.zeros(x.shape[0], c), torch.zeros(x.shape[0], c)] for k, c in (("y", c_out), ("x", x.shape[1]))}
    out = {k: [t.double() for t in v] for k, v in out.items()}
    sums = {"weight": [torch.zeros(len(fields), dtype=torch.float64) for _ in range(2)],
            "bias": [torch.zeros(sum(1 for l, _ in fields if l == 0), dtype=torch.float64) for _ in range(2)]}
    found = {"gy": None if gy is None else gy.clone()}
    for lo, hi in zip(offsets[:-1], offsets[1:]):
        if hi <= lo:
            continue
        v, rows = x[lo:hi], hi - lo
        count = rows * copies
        mu = torch.where(mean_of, (v @ member).sum(0) / count, 0.0)[group]
        size = ((v.abs() @ member).sum(0) / count)[group]
        d = v - mu
        r = 1 / torch.sqrt(((d * d) @ member).sum(0) / count + eps)[group]
        hat, far = d * r, (v.abs() + size) * r
        z, zt = hat * wc + bc, far * wc.abs() + bc.abs()
        body, gz = z[:, :c_out], z[:, c_out:]
        val, slope = activation(scalar, body)
        plain = is_scalar[:c_out]
        y, yt = torch.where(plain, val, body), torch.where(plain, val.abs() + 1.13 * zt[:, :c_out] * (scalar is not None) + zt[:, :c_out] * (scalar is None), zt[:, :c_out])
        if n_gate:
            gv, gs = activation(gate, gz)
            gt = zt[:, c_out:]
            at = torch.full((len(fields),), -1)
            at[vectors] = torch.arange(n_gate)
            mine = at[field[:c_out]].clamp(min=0)
            y = torch.where(plain, y, body * gv[:, mine])
            yt = torch.where(plain, yt, zt[:, :c_out] * gv[:, mine].abs() + body.abs() * gt[:, mine] + y.abs())
        out["y"][0][lo:hi], out["y"][1][lo:hi] = y, yt
        if gy is None:
            continue
        g = gy[lo:hi]
        curved = 0.0 if scalar in (None, torch.relu, F.relu) else 1.13
        if scalar in (torch.relu, F.relu):
            g = found["gy"][lo:hi] = torch.where(plain & (body.abs() < 2.0 ** -12 * zt[:, :c_out]), 0.0, g)
        dz = torch.where(plain, g * slope, g)
        dt = torch.where(plain, g.abs() * (slope.abs() + curved * zt[:, :c_out]), g.abs())
        if n_gate:
            pick = (at[field[:c_out]][:, None] == torch.arange(n_gate)).double()
            into = (g * body) @ pick
            intot = (g.abs() * (body.abs() + zt[:, :c_out])) @ pick
            dt = torch.where(plain, dt, g.abs() * (gv[:, mine].abs() + gt[:, mine]))
            dz = torch.where(plain, dz, g * gv[:, mine])
            dz, dt = torch.cat([dz, into * gs], 1), torch.cat([dt, intot * (gs.abs() + gt)], 1)
        a, at_ = dz * wc, dt * wc.abs()
        s1 = torch.where(mean_of, (a @ member).sum(0) / count, 0.0)[group]
        s2 = (((a * hat) @ member).sum(0) / count)[group]
        t1 = torch.where(mean_of, (at_ @ member).sum(0) / count, 0.0)[group]
        t2 = (((at_ * far) @ member).sum(0) / count)[group]
        out["x"][0][lo:hi] = r * (a - s1 - hat * s2)
        out["x"][1][lo:hi] = r * (at_ + t1 + far * t2)
        by_field = (field[:, None] == torch.arange(len(fields))).double()
        sums["weight"][0] += ((dz * hat).sum(0)) @ by_field
        sums["weight"][1] += ((dt * far) ** 2).sum(0) @ by_field
        sums["bias"][0] += dz.sum(0)[is_scalar]
        sums["bias"][1] += (dt ** 2).sum(0)[is_scalar]
    found["y"] = tuple(out["y"])
    if gy is not None:
        found["x"] = tuple(out["x"])
        for k, (value, squares) in sums.items():
            found[k] = (value, squares.sqrt())
    return found



def feedforward(t, act, gy):
    """The gated feed-forward block and its gradients: name -> (value, size, rounded, stages).  t: x, w_in, w_out, b_in, b_out, residual (the last
    three may be None) in 64 bits.

    What errors that go either way are measured by: size, of sums in float32, is the root of the sum of the squares of the terms, with those of
    the sums that the terms come from; rounded is the root of the sum of the squares of the terms that 16-bit rows round on the way.  stages:
    products one behind the other."""
    x, (wg, wu), wo = t["x"], t["w_in"], t["w_out"]
    g, u = x @ wg.t(), x @ wu.t()
    if t["b_in"] is not None:
        g, u = g + t["b_in"][0], u + t["b_in"][1]
    a, slope = activation(act, g)
    h = a * u
    y = h @ wo.t()
    if t["b_out"] is not None:
        y = y + t["b_out"]
    if t["residual"] is not None:
        y = y + t["residual"]
    dh = gy @ wo
    dg, du = dh * u * slope, dh * a
    sq = lambda *v: [k * k for k in v]  # noqa: E731
    x2, wg2, wu2, wo2, gy2 = sq(x, wg, wu, wo, gy)
    # an error of g or u, steps of the root of its sum, goes on into h, dg and du; so does one of dh
    g2, u2, dh2 = x2 @ wg2.t() + g * g, x2 @ wu2.t() + u * u, gy2 @ wo2 + dh * dh
    h2 = g2 * u2 + h * h
    dg2, du2 = dh2 * u2 + dg * dg, dh2 * g2 + du * du
    out = {"y": (y, h2 @ wo2.t(), (h * h) @ wo2.t(), 2),
           "x": (dg @ wg + du @ wu, dg2 @ wg2 + du2 @ wu2, (dg * dg) @ wg2 + (du * du) @ wu2, 3),
           "w_in": (torch.stack([dg.t() @ x, du.t() @ x]), torch.stack([dg2.t() @ x2, du2.t() @ x2]), torch.stack([(dg * dg).t() @ x2, (du * du).t() @ x2]), 3),
           "w_out": (gy.t() @ h, gy2.t() @ h2, gy2.t() @ (h * h), 2),
           "b_in": (torch.stack([dg.sum(0), du.sum(0)]), torch.stack([dg2.sum(0), du2.sum(0)]), torch.stack([(dg * dg).sum(0), (du * du).sum(0)]), 2),
           "b_out": (gy.sum(0), gy2.sum(0), torch.zeros_like(gy.sum(0)), 1)}
    out = {k: (v, (squares + v * v).sqrt(), rounded.sqrt(), stages) for k, (v, squares, rounded, stages) in out.items()}
    out["kink"] = (g.abs() / g2.sqrt()).min()           # how near a gate comes to zero
    return out
