"""The routed-experts operators of ``nersemble_amd.experts`` as a set of measured calls.

Four operators that are used one after another by a routed network (``nersemble_amd.tcnn.RoutedNetwork``):

``route``    scores of the experts for every row (softmax or sigmoid), choice of the best ``top_k`` (with a balancing bias
             and a choice of expert groups in front where asked for), their weights; forward, and the gradient of the logits
``plan``     the (row, choice) entries ordered by expert: segment offsets, source entry of every ordered row, place of every
             entry
``linear``   every ordered row times the weight matrix of its expert; forward, and the gradients of inputs and weights
``combine``  the weighted sum of a row's ``top_k`` expert outputs; forward, and the gradients of outputs and weights

Each is given twice: as a user calls it (``own``), and in elementary torch operations.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

_DT = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _route(name, tokens, experts, top_k, scores, dtype, train, groups=1, top_groups=1, group_top=1, bias=False, scale=1.0,
           renorm=True):
    return dict(name=name, op="route", tokens=tokens, experts=experts, top_k=top_k, scores=scores, dtype=dtype, train=train,
                groups=groups, top_groups=top_groups, group_top=group_top, bias=bias, scale=scale, renorm=renorm)


def _plan(name, tokens, experts, top_k, masked):
    return dict(name=name, op="plan", tokens=tokens, experts=experts, top_k=top_k, masked=masked)


def _linear(name, tokens, experts, top_k, n_in, n_out, dtype, train, gather, relu, master, masked):
    return dict(name=name, op="linear", tokens=tokens, experts=experts, top_k=top_k, n_in=n_in, n_out=n_out, dtype=dtype,
                train=train, gather=gather, relu=relu, master=master, masked=masked)


def _combine(name, tokens, experts, top_k, n_out, dtype, train, masked):
    return dict(name=name, op="combine", tokens=tokens, experts=experts, top_k=top_k, n_out=n_out, dtype=dtype, train=train,
                masked=masked)


def listed():
    return [
        # one row alone (a single token that is served): latency of one small call
        _route("route one row", 1, 64, 6, "softmax", "float32", False),
        # the samples of one training step (2^20) routed to as many experts as an ensemble has grids (32)
        _route("route samples train", 1 << 20, 32, 2, "softmax", "float32", True),
        # many experts in groups, balanced by a bias that only the choice sees; 16-bit logits, an odd number of rows
        _route("route groups train", 30011, 256, 8, "sigmoid", "bfloat16", True, 8, 4, 2, True, 2.5),
        # a batch of rays (4096), two choices each
        _plan("plan rays", 4096, 16, 2, 0.0),
        # a step's samples, a part of which lies outside the scene box and is not routed; an odd number of experts
        _plan("plan samples masked", (1 << 20) - 3, 61, 2, 0.25),
        # four tokens that are served: most weights are read for one row
        _linear("linear single tokens", 4, 64, 8, 1024, 1024, "float16", False, True, False, False, 0.0),
        # first layer of small networks (32 -> 64, ReLU) over a quarter of a step's samples
        _linear("linear samples train", 1 << 18, 16, 2, 32, 64, "float16", True, True, True, False, 0.0),
        # wide layers, long batches: bound by the matrix units
        _linear("linear wide train", 16384, 16, 2, 1024, 2048, "bfloat16", True, True, False, False, 0.0),
        # odd counts and widths, rows already in the experts' order, 32-bit weights whose gradient stays in 32 bits
        _linear("linear odd train", 5003, 23, 3, 176, 136, "float16", True, False, False, True, 0.1),
        # outputs of four served tokens joined
        _combine("combine single tokens", 4, 64, 8, 1024, "float16", False, 0.0),
        # outputs of small networks (16 wide) joined over a step's samples, a part of which was not routed
        _combine("combine samples train", (1 << 19) + 1, 32, 2, 16, "float16", True, 0.25),
        # wide rows, many choices
        _combine("combine wide train", 8192, 64, 8, 1024, "bfloat16", True, 0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["route", "plan", "linear", "linear", "combine"])
    while True:
        tokens = _log_int(rng, 1, 1 << 20)
        experts = _log_int(rng, 2, 256)
        top_k = rng.randint(1, min(8, experts))
        dtype = rng.choice(["float16", "bfloat16"])
        masked = rng.choice([0.0, 0.0, 0.1, 0.3])
        train = rng.random() < 0.6
        if op == "route":
            if tokens * experts > (1 << 25):
                continue
            c = _route("", tokens, experts, top_k, rng.choice(["softmax", "sigmoid"]), rng.choice(["float32", dtype]), train,
                       bias=rng.random() < 0.5, scale=rng.choice([1.0, 2.5]), renorm=rng.random() < 0.7)
            if rng.random() < 0.4:
                groups = rng.choice([2, 3, 4, 5, 8])
                per = -(-experts // groups)
                c["experts"], c["groups"], c["top_groups"] = per * groups, groups, rng.randint(1, groups)
                c["group_top"] = rng.choice([1, 2]) if per > 1 else 1
                c["top_k"] = min(top_k, c["top_groups"] * per)
                if c["experts"] > 256 or tokens * c["experts"] > (1 << 25):
                    continue
            # (a single renormalised weight is a constant: it has no gradient to compare)
            c["renorm"] = c["renorm"] and c["top_k"] > 1
        elif op == "plan":
            if tokens * top_k > (1 << 21):
                continue
            c = _plan("", tokens, experts, top_k, masked)
        elif op == "linear":
            hi = 256 if rng.random() < 0.5 else 2048
            n_in, n_out = 8 * _log_int(rng, 2, hi // 8), 8 * _log_int(rng, 2, hi // 8)
            rows = tokens * top_k
            if rows * n_in * n_out > 32768 * 1024 * 2048 or rows * (n_in + n_out) > 32768 * 2048 \
                    or experts * n_in * n_out > 64 * 1024 * 1024:
                continue
            # (32-bit weights' gradients are compared in 32 bits, where the sign of a value next to zero would show: no ReLU)
            relu = rng.random() < 0.5
            c = _linear("", tokens, experts, top_k, n_in, n_out, dtype, train, rng.random() < 0.6, relu,
                        (not relu) and rng.random() < 0.5, masked)
        else:
            n_out = 8 * _log_int(rng, 1, 256)
            if tokens * top_k * n_out > 8192 * 8 * 1024:
                continue
            c = _combine("", tokens, experts, top_k, n_out, dtype, train, masked)
        del c["name"]
        return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _logits(case, g):
    """Unequal popularity of the experts, as a router that is being trained has."""
    return _randn(g, case["tokens"], case["experts"]) * 1.5 + _randn(g, case["experts"]) * 0.5


def _chosen(case, g):
    """[tokens, top_k] int32: distinct experts of every row, -1 throughout for the rows that are masked."""
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    out = torch.empty((T, k), dtype=torch.int32, device="cuda")
    tilt = _randn(g, E) * 0.5
    step = max(1, (1 << 26) // E)
    for t in range(0, T, step):
        n = min(step, T - t)
        out[t:t + n] = (_randn(g, n, E) * 1.5 + tilt).topk(k, dim=1).indices.to(torch.int32)
    if case["masked"] > 0:
        out[torch.rand((T,), generator=g, device="cuda") < case["masked"]] = -1
    return out


def _ordered(chosen, n_experts):
    """(offsets, rows, positions) of a plan, by a stable sort."""
    flat = chosen.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < n_experts), flat, n_experts)
    order = torch.sort(key, stable=True).indices
    counts = torch.zeros(n_experts + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([counts.new_zeros(1), counts[:n_experts].cumsum(0)])
    place = torch.arange(flat.numel(), device=flat.device)
    valid = place < offsets[-1]
    rows = torch.where(valid, order, -1)
    positions = torch.empty_like(flat).scatter_(0, order, torch.where(valid, place, -1))
    return offsets.to(torch.int32), rows.to(torch.int32), positions.to(torch.int32).reshape(chosen.shape)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=case)
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    if case["op"] == "route":
        s["logits"] = _logits(case, g).to(_DT[case["dtype"]])
        s["bias"] = _randn(g, E) * 0.1 if case["bias"] else None
        s["grad"] = _randn(g, T, k)
        s["logits"].requires_grad_(case["train"])
    elif case["op"] == "plan":
        s["chosen"] = _chosen(case, g)
    else:
        dt = _DT[case["dtype"]]
        s["offsets"], s["rows"], s["positions"] = _ordered(_chosen(case, g), E)
        # rows that a program with a fixed room for each expert would keep free: the plain form's padded layout
        s["room"] = max(1, int((s["offsets"][1:] - s["offsets"][:-1]).max()))
        if case["op"] == "linear":
            x = _randn(g, T if case["gather"] else T * k, case["n_in"]).to(dt)
            w = _randn(g, E, case["n_out"], case["n_in"]) / math.sqrt(case["n_in"])
            s["grad"] = _randn(g, T * k, case["n_out"]).to(dt)
            s["x"] = x.requires_grad_(case["train"])
            s["w16"] = w.to(dt) if case["master"] else None
            s["w"] = (w if case["master"] else w.to(dt)).requires_grad_(case["train"])
        else:
            s["y"] = _randn(g, T * k, case["n_out"]).to(dt).requires_grad_(case["train"])
            s["weights"] = torch.softmax(_randn(g, T, k), dim=1).requires_grad_(case["train"])
            s["grad"] = _randn(g, T, case["n_out"]).to(dt)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from nersemble_amd import experts as X
    case = s["case"]
    op, train = case["op"], case["train"] if "train" in case else False
    if op == "plan":
        plan = X.expert_plan(s["chosen"], case["experts"])
        return {"offsets": plan.offsets, "rows": plan.rows, "positions": plan.positions}
    if op == "route":
        weights, chosen = X.route_experts(s["logits"], case["top_k"], scores=case["scores"], bias=s["bias"],
                                          n_groups=case["groups"], top_groups=case["top_groups"],
                                          group_top=case["group_top"], renormalise=case["renorm"], scale=case["scale"])
        if not train:
            return {"weights": weights, "chosen": chosen}
        (d,) = torch.autograd.grad(weights, [s["logits"]], s["grad"])
        return {"weights": weights, "chosen": chosen, "dlogits": d}
    plan = X.ExpertPlan(s["offsets"], s["rows"], s["positions"])
    if op == "linear":
        y = X.expert_linear(s["x"], s["w"], plan, gather=case["gather"], relu=case["relu"], w16=s["w16"])
        if not train:
            return {"y": y}
        dx, dw = torch.autograd.grad(y, [s["x"], s["w"]], s["grad"])
        return {"y": y, "dx": dx, "dw": dw}
    out = X.expert_combine(s["y"], s["weights"], plan)
    if not train:
        return {"out": out}
    dy, dweights = torch.autograd.grad(out, [s["y"], s["weights"]], s["grad"])
    return {"out": out, "dy": dy, "dweights": dweights}


def _run_plain(s):
    with torch.no_grad():
        return {"route": _plain_route, "plan": _plain_plan, "linear": _plain_linear, "combine": _plain_combine}[
            s["case"]["op"]](s, s["case"])


def _plain_route(s, case):
    """The choice is made in 64 bits: two scores next to each other must not change places."""
    x = s["logits"].detach()
    T, E, k, G = case["tokens"], case["experts"], case["top_k"], case["groups"]
    xd = x.double()
    if case["scores"] == "softmax":
        e = torch.exp(xd - xd.amax(dim=1, keepdim=True))
        score = e / e.sum(dim=1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-xd))
    choice = score if s["bias"] is None else score + s["bias"].double()
    if G > 1:
        by_group = torch.sort(choice.view(T, G, E // G), dim=2, descending=True).values[..., :case["group_top"]].sum(dim=2)
        kept = torch.sort(by_group, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        on = torch.zeros((T, G), dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        choice = choice.view(T, G, E // G).masked_fill(~on[..., None], -math.inf).view(T, E)
    chosen = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :k]
    score = score.float()
    u = score.gather(1, chosen)
    total = u.sum(dim=1, keepdim=True)
    w = (u / total if case["renorm"] else u) * case["scale"]
    out = {"weights": w, "chosen": chosen.to(torch.int32)}
    if case["train"]:
        g = s["grad"] * case["scale"]
        du = (g - (g * u).sum(dim=1, keepdim=True) / total) / total if case["renorm"] else g
        if case["scores"] == "softmax":
            ds = torch.zeros_like(score).scatter_(1, chosen, du)
            d = score * (ds - (du * u).sum(dim=1, keepdim=True))
        else:
            d = torch.zeros_like(score).scatter_(1, chosen, du * u * (1.0 - u))
        out["dlogits"] = d.to(x.dtype)
    return out


def _plain_plan(s, case):
    offsets, rows, positions = _ordered(s["chosen"], case["experts"])
    return {"offsets": offsets, "rows": rows, "positions": positions}


def _plain_linear(s, case):
    """Every expert's rows in a room of its own of the same size, and products over the batch of experts in 32 bits."""
    T, E, k, K, N, C = case["tokens"], case["experts"], case["top_k"], case["n_in"], case["n_out"], s["room"]
    x, w = s["x"].detach(), (s["w"] if s["w16"] is None else s["w16"]).detach()
    R = T * k
    offsets = s["offsets"].long()
    place = torch.arange(R, device=x.device)
    valid = place < offsets[-1]
    expert = torch.searchsorted(offsets[1:].contiguous(), place, right=True).clamp(max=E - 1)
    slot = torch.where(valid, expert * C + place - offsets[expert], E * C)
    source = torch.where(valid, s["rows"].long() // k, T) if case["gather"] else place
    pad = x.new_zeros((1, K), dtype=torch.float32)
    xs = torch.cat([x.float(), pad])[source] if case["gather"] else x.float()
    xp = torch.zeros((E * C + 1, K), dtype=torch.float32, device=x.device).index_copy_(0, slot, xs)[:-1].view(E, C, K)
    wf = w.float()
    yp = torch.bmm(xp, wf.transpose(1, 2).contiguous())
    if case["relu"]:
        yp = yp * (yp > 0)
    y = torch.cat([yp.view(E * C, N), yp.new_zeros((1, N))])[slot]
    out = {"y": y.to(x.dtype)}
    if case["train"]:
        dyp = torch.zeros((E * C + 1, N), dtype=torch.float32, device=x.device).index_copy_(0, slot, s["grad"].float())
        dyp = dyp[:-1].view(E, C, N)
        if case["relu"]:
            dyp = dyp * (yp > 0)
        dxp = torch.cat([torch.bmm(dyp, wf).view(E * C, K), pad])[slot]
        if case["gather"]:
            # the place of every choice of a row; row R of what is gathered stands for a choice that is not there
            pos = torch.where(s["positions"] >= 0, s["positions"].long(), R)
            dxp = torch.cat([dxp, pad])[pos].sum(dim=1)
        out["dx"] = dxp.to(x.dtype)
        out["dw"] = torch.bmm(dyp.transpose(1, 2).contiguous(), xp).to(s["w"].dtype)
    return out


def _plain_combine(s, case):
    R = case["tokens"] * case["top_k"]
    y, w = s["y"].detach(), s["weights"].detach()
    there = s["positions"] >= 0
    pos = torch.where(there, s["positions"].long(), R)
    ys = torch.cat([y.float(), y.new_zeros((1, y.shape[1]), dtype=torch.float32)])[pos]
    out = {"out": (w[..., None] * ys).sum(dim=1).to(y.dtype)}
    if case["train"]:
        g = s["grad"].float()
        dy = torch.zeros((R + 1, y.shape[1]), dtype=torch.float32, device=y.device)
        dy.index_copy_(0, pos.view(-1), (w[..., None] * g[:, None, :]).view(R, -1))
        out["dy"] = dy[:R].to(y.dtype)
        out["dweights"] = (g[:, None, :] * ys).sum(dim=2)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    R = T * k
    if case["op"] == "plan":
        return {"bytes": 4 * (3 * R + E + 1), "flops": R}
    e = _SIZE[case["dtype"]]
    if case["op"] == "route":
        # forward: logits in, weights and choices out; backward: the weights' gradient in, the logits' gradient out
        return {"bytes": T * (E * e + 8 * k) + (T * (4 * k + E * e) if case["train"] else 0),
                "flops": T * E * (8 if case["train"] else 4)}
    live = max(1, int(round(R * (1.0 - case["masked"]))))
    N = case["n_out"]
    if case["op"] == "combine":
        moved = live * N * e + T * N * e + 8 * R
        if case["train"]:
            moved += T * N * e + R * N * e + 4 * R
        return {"bytes": moved, "flops": (2 + 3 * case["train"]) * live * N}
    K = case["n_in"]
    read_x = (T if case["gather"] else live) * K * e
    weights = min(E, live) * N * K * e
    moved = read_x + weights + R * N * e + 4 * R
    if case["train"]:
        moved += live * N * e + (T if case["gather"] else R) * K * e + E * N * K * (4 if case["master"] else e)
    return {"bytes": moved, "flops": (6 if case["train"] else 2) * live * N * K}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    E, k = case["experts"], case["top_k"]
    if case["op"] == "route":
        return _exact_route(s, case)
    if case["op"] == "plan":
        flat = s["chosen"].view(-1)
        offsets = torch.zeros(E + 1, dtype=torch.int32, device=flat.device)
        rows, positions = torch.full_like(flat, -1), torch.full_like(flat, -1)
        filled = 0
        for e in range(E):
            mine = torch.nonzero(flat == e).view(-1)
            rows[filled:filled + mine.numel()] = mine.to(torch.int32)
            positions[mine] = torch.arange(filled, filled + mine.numel(), dtype=torch.int32, device=flat.device)
            filled += mine.numel()
            offsets[e + 1] = filled
        return {"offsets": offsets, "rows": rows, "positions": positions.view_as(s["chosen"])}
    if case["op"] == "combine":
        y, w, g, pos = s["y"].detach().double(), s["weights"].detach().double(), s["grad"].double(), s["positions"].long()
        out = torch.zeros_like(g)
        dy, dw = torch.zeros_like(y), torch.zeros_like(w)
        for j in range(k):
            at = torch.nonzero(pos[:, j] >= 0).view(-1)
            p = pos[at, j]
            out[at] += w[at, j, None] * y[p]
            dy[p] = w[at, j, None] * g[at]
            dw[at, j] = (g[at] * y[p]).sum(dim=1)
        return {"out": out, "dy": dy, "dweights": dw} if case["train"] else {"out": out}
    x, g = s["x"].detach().double(), s["grad"].double()
    w = (s["w"] if s["w16"] is None else s["w16"]).detach().double()
    y, dx, dw = torch.zeros_like(g), torch.zeros_like(x), torch.zeros_like(w)
    bounds = s["offsets"].tolist()
    for e in range(E):
        a, b = bounds[e], bounds[e + 1]
        if a == b:
            continue
        source = torch.div(s["rows"][a:b].long(), k, rounding_mode="floor") if case["gather"] else torch.arange(
            a, b, device=x.device)
        z = x[source] @ w[e].t().contiguous()
        y[a:b] = z.clamp(min=0) if case["relu"] else z
        if case["train"]:
            dz = g[a:b].where(z > 0, torch.zeros_like(z)) if case["relu"] else g[a:b]
            dx.index_add_(0, source, dz @ w[e])
            dw[e] = dz.t().contiguous() @ x[source]
    return {"y": y, "dx": dx, "dw": dw} if case["train"] else {"y": y}


def _exact_route(s, case):
    x = s["logits"].detach().double()
    T, E = x.shape
    k, G = case["top_k"], case["groups"]
    score = torch.softmax(x, dim=1) if case["scores"] == "softmax" else torch.sigmoid(x)
    choice = score.clone() if s["bias"] is None else score + s["bias"].double()

    def best(v):
        """The place of the largest value of every row, the lowest such place where several are as large."""
        top = v.max(dim=1, keepdim=True).values
        return torch.where(v == top, torch.arange(v.shape[1], device=v.device), v.shape[1]).min(dim=1).indices

    if G > 1:
        rest = choice.view(T, G, E // G).clone()
        total = torch.zeros((T, G), dtype=torch.float64, device=x.device)
        for _ in range(case["group_top"]):
            m = rest.max(dim=2)
            total += m.values
            rest.scatter_(2, m.indices[..., None], -math.inf)
        on = torch.zeros((T, G), dtype=torch.bool, device=x.device)
        for _ in range(case["top_groups"]):
            at = best(total)[:, None]
            on.scatter_(1, at, True)
            total.scatter_(1, at, -math.inf)
        choice[~on.repeat_interleave(E // G, dim=1)] = -math.inf
    chosen = torch.empty((T, k), dtype=torch.int64, device=x.device)
    for j in range(k):
        chosen[:, j] = best(choice)
        choice.scatter_(1, chosen[:, j:j + 1], -math.inf)
    on = torch.zeros((T, E), dtype=torch.bool, device=x.device).scatter_(1, chosen, True)
    mine = torch.gather(score, 1, chosen)
    norm = mine.sum(dim=1, keepdim=True) if case["renorm"] else torch.ones((T, 1), dtype=torch.float64, device=x.device)
    weights = case["scale"] * mine / norm
    out = {"weights": weights, "chosen": chosen.to(torch.int32)}
    if case["train"]:
        # through the weights w = scale * s / norm, then through the score, written for all experts at once
        g = torch.zeros((T, E), dtype=torch.float64, device=x.device).scatter_(1, chosen, s["grad"].double())
        ds = case["scale"] / norm * g
        if case["renorm"]:
            ds = torch.where(on, ds - ((g * score).sum(dim=1, keepdim=True) * case["scale"] / norm ** 2), torch.zeros_like(ds))
        if case["scores"] == "softmax":
            out["dlogits"] = score * ds - score * (score * ds).sum(dim=1, keepdim=True)
        else:
            out["dlogits"] = ds * score * torch.sigmoid(-x)
    return out
