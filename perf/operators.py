"""The routed-experts operators as measured cases: routing, grouping, products per expert, combination.

A token is routed to its `top_k` best experts (centers), the (token, choice) pairs are grouped by expert, each
group is multiplied with its expert's matrix, and a token's results are summed with its weights.  Every operator
has a plain form here in elementary float32 torch operations, rounded once at the end, and `exact` in float64.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
INF = float("inf")


# ---------------------------------------------------------------- cases

def _route(name, T, E, k, dtype="f32", score="softmax", bias=False, groups=1, top_groups=1, renorm=True, scale=1.0,
           masked=0, grad=False):
    return {"name": name, "op": "route", "T": T, "E": E, "k": k, "dtype": dtype, "score": score, "bias": bias,
            "groups": groups, "top_groups": top_groups, "renorm": renorm, "scale": scale, "masked": masked,
            "grad": grad}


def _group(name, T, E, k, masked=0):
    return {"name": name, "op": "group", "T": T, "E": E, "k": k, "masked": masked}


def _matmul(name, T, E, k, N, D, dtype="bf16", masked=0, gather=True, grad=False):
    return {"name": name, "op": "matmul", "T": T, "E": E, "k": k, "N": N, "D": D, "dtype": dtype, "masked": masked,
            "gather": gather, "grad": grad}


def _combine(name, T, E, k, H, dtype="bf16", masked=0, weighted=True, grad=False):
    return {"name": name, "op": "combine", "T": T, "E": E, "k": k, "H": H, "dtype": dtype, "masked": masked,
            "weighted": weighted, "grad": grad}


def listed():
    return [
        # one new token of a served model: latency alone
        _route("route_token", 1, 64, 4, "bf16"),
        # a prompt through a router with sigmoid scores, a balance bias and expert groups; some rows are padding
        _route("route_prompt_groups", 4001, 256, 8, "f32", "sigmoid", True, 8, 4, True, 2.5, 200),
        # a training batch: choices, weights and the logits' gradient, 16-bit logits (ties are common there)
        _route("route_train", 65536, 128, 8, "bf16", renorm=False, grad=True),
        # the plan of a batch of single tokens
        _group("group_batch", 24, 128, 8),
        # the plan of a long training batch with padded rows
        _group("group_train", 131072, 256, 8, 1000),
        # one new token: the chosen experts' matrices are read once, nothing else counts
        _matmul("expert_token", 1, 64, 8, 2048, 2048),
        # a batch of single tokens from several users, sizes that are no multiple of a tile
        _matmul("expert_batch", 48, 32, 4, 1000, 1336, "f16"),
        # a long prompt: many rows an expert, uneven over the experts
        _matmul("expert_prompt", 8192, 64, 8, 2048, 2048),
        # a training step's products: forward, the inputs' gradient, the matrices' gradient; padded rows
        _matmul("expert_train", 4099, 16, 4, 1536, 2048, masked=100, grad=True),
        # a small training step on odd sizes, rows already grouped
        _matmul("expert_train_odd", 777, 12, 2, 515, 333, "f16", gather=False, grad=True),
        # joining the experts' answers for a batch of single tokens
        _combine("combine_batch", 48, 32, 4, 2048),
        # joining in training, with the gradients of the experts' answers and of the weights
        _combine("combine_train", 16384, 64, 8, 2048, masked=300, grad=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _dim(rng, lo, hi):
    """A feature count: mostly multiples of 64, some of 8 only, some odd."""
    n, u = _log(rng, lo, hi), rng.random()
    return max(64, n // 64 * 64) if u < 0.5 else max(8, n // 8 * 8) if u < 0.8 else n


def draw(rng):
    op = rng.choice(["route", "route", "group", "matmul", "matmul", "matmul", "combine", "combine"])
    E = rng.choice([8, 12, 16, 32, 60, 64, 96, 128, 160, 256]) if op != "matmul" else rng.choice([4, 8, 12, 16, 32, 60, 64, 128])
    k = rng.randint(1, min(8, E // 2))
    if op == "route":
        T = _log(rng, 1, 65536)
        score = rng.choice(["softmax", "sigmoid"])
        groups = rng.choice([1, 1, 4])
        return _drop(_route("", T, E, k, rng.choice(["f32", "bf16", "f16"]), score, rng.random() < 0.5, groups,
                            1 if groups == 1 else rng.choice([2, 3]), rng.random() < 0.6, rng.choice([1.0, 2.5]),
                            rng.choice([0, T // 10]), rng.random() < 0.5))
    if op == "group":
        T = _log(rng, 1, 131072)
        return _drop(_group("", T, E, k, rng.choice([0, T // 10])))
    if op == "matmul":
        N, D, T = _dim(rng, 64, 2048), _dim(rng, 64, 2048), _log(rng, 1, 8192)
        grad = T >= 32 and rng.random() < 0.5
        T = max(1, min(T, int(5.4e11 / (2.0 * k * N * D * (3 if grad else 1)))))
        return _drop(_matmul("", T, E, k, N, D, rng.choice(["bf16", "f16"]), rng.choice([0, T // 10]),
                             rng.random() < 0.7, grad))
    T, H = _log(rng, 1, 16384), _dim(rng, 64, 2048)
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    T = T if dtype != "f32" else max(1, T // 2)
    return _drop(_combine("", T, E, k, H, dtype, rng.choice([0, T // 10]), rng.random() < 0.8, rng.random() < 0.5))


def _drop(case):
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs

def _popularity(E):
    """Experts are not equally liked: log popularity falling by about a factor of four over the experts."""
    return -0.5 * torch.log1p(torch.arange(E, dtype=torch.float32) * (15.0 / E))


def _logits(T, E, gen):
    pop = _popularity(E)[torch.randperm(E, generator=gen)].cuda()
    g = torch.Generator("cuda").manual_seed(gen.initial_seed())
    return torch.randn(T, E, generator=g, device="cuda") * 1.5 + pop, g


def _mask(case, gen):
    """Rows that are real: `masked` of them, anywhere, are padding."""
    m = torch.ones(case["T"], dtype=torch.bool)
    m[torch.randperm(case["T"], generator=gen)[:case["masked"]]] = False
    return m.cuda() if case["masked"] else None


def _ids(case, gen):
    """Distinct choices for each token, -1 for padding."""
    l, g = _logits(case["T"], case["E"], gen)
    ids = l.topk(case["k"], dim=1).indices.to(torch.int32)
    m = _mask(case, gen)
    if m is not None:
        ids[~m] = -1
    return ids, g


def _plan(ids, E):
    """offsets, rows, slot of a stable grouping by expert (ids outside [0, E) are left out)."""
    k = ids.shape[-1] if ids.ndim == 2 else 1
    flat = ids.reshape(-1).long()
    P = flat.numel()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    sorted_key, order = torch.sort(key, stable=True)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=ids.device).index_add_(0, key, torch.ones_like(key))
    ends = counts[:E].cumsum(0)
    offsets = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    kept = sorted_key < E
    rows = torch.where(kept, order // k, -1).to(torch.int32)
    at = torch.where(kept, torch.arange(P, device=ids.device), -1)
    slot = torch.empty_like(at).index_copy_(0, order, at).to(torch.int32).reshape(ids.shape)
    return offsets, rows, slot


def prepare(case, seed):
    gen = torch.Generator().manual_seed(int(seed))
    op, T, E, k = case["op"], case["T"], case["E"], case["k"]
    s = {"case": case}
    if op == "route":
        l, g = _logits(T, E, gen)
        s["logits"] = l.to(TYPES[case["dtype"]])
        s["bias"] = torch.randn(E, generator=g, device="cuda") * 0.1 if case["bias"] else None
        s["mask"] = _mask(case, gen)
        s["dweights"] = torch.randn(T, k, generator=g, device="cuda") if case["grad"] else None
        return s
    ids, g = _ids(case, gen)
    if op == "group":
        s["ids"] = ids
        return s
    dt = TYPES[case["dtype"]]
    s["offsets"], s["rows"], s["slot"] = _plan(ids, E)
    P = T * k
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)  # noqa: E731
    if op == "matmul":
        N, D = case["N"], case["D"]
        s["x"] = rand(T if case["gather"] else P, D).to(dt)
        s["w"] = (rand(E, N, D) / math.sqrt(D)).to(dt)
        s["dy"] = rand(P, N).to(dt) if case["grad"] else None
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())   # rows of the fullest expert
        return s
    H = case["H"]
    s["y"] = rand(P, H).to(dt)
    w = torch.rand(T, k, generator=g, device="cuda") + 0.05
    s["weights"] = w / w.sum(1, keepdim=True) if case["weighted"] else None
    s["dout"] = rand(T, H).to(dt) if case["grad"] else None
    return s


# ---------------------------------------------------------------- plain forms (float32)

def _keep(key, c):
    """Keys of the experts outside the best groups become -inf."""
    G, E = c["groups"], c["E"]
    if G == 1:
        return key
    best = key.reshape(-1, G, E // G).topk(min(2, E // G), dim=2).values
    gscore = torch.where(best > -INF, best, 0.0).sum(2)
    gscore = torch.where(best[:, :, 0] > -INF, gscore, -INF)
    order = torch.sort(gscore, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
    keep = torch.zeros_like(gscore, dtype=torch.bool).scatter_(1, order, True)
    return torch.where(keep.repeat_interleave(E // G, dim=1), key, -INF)


def _plain_route(s):
    c = s["case"]
    l = s["logits"].float()
    ok = l > -INF
    if s["mask"] is not None:
        ok = ok & s["mask"][:, None]
    sig = 1.0 / (1.0 + torch.exp(-l))
    key = l if c["score"] == "softmax" else sig
    if s["bias"] is not None:
        key = key + s["bias"]
    key = _keep(torch.where(ok & (key > -INF), key, -INF), c)
    sk, si = torch.sort(key, dim=1, descending=True, stable=True)
    got = sk[:, :c["k"]] > -INF
    idx = si[:, :c["k"]]
    if c["score"] == "softmax":
        over = torch.where(got, l.gather(1, idx), -INF) if c["renorm"] else torch.where(ok, l, -INF)
        m = over.amax(1, keepdim=True)
        m = torch.where(m > -INF, m, 0.0)
        total = torch.exp(over - m).sum(1, keepdim=True)
        p = torch.where(got, torch.exp(l.gather(1, idx) - m) / total, 0.0)
    else:
        p = torch.where(got, sig.gather(1, idx), 0.0)
        if c["renorm"]:
            total = p.sum(1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
    out = {"ids": torch.where(got, idx, -1).to(torch.int32), "weights": c["scale"] * p}
    if s["dweights"] is None:
        return out
    g = torch.where(got, s["dweights"], 0.0) * c["scale"]
    dot = (g * p).sum(1, keepdim=True)
    if c["score"] == "softmax":
        # dl_i = p_i ([i chosen] g_i - sum g p): over the chosen when renormalised, over all the available otherwise
        if c["renorm"]:
            dl = torch.zeros_like(l).scatter_add_(1, idx, p * (g - dot))
        else:
            full = torch.where(ok, torch.exp(l - m) / total, 0.0)
            dl = torch.where(ok, -full * dot, 0.0).scatter_add_(1, idx, p * g)
    else:
        sg = torch.where(got, sig.gather(1, idx), 0.0)
        ds = g
        if c["renorm"]:
            ds = torch.where(total > 0, (g - dot) / total, 0.0)
        dl = torch.zeros_like(l).scatter_add_(1, idx, ds * sg * (1.0 - sg))
    out["dlogits"] = dl.to(s["logits"].dtype)
    return out


def _padded(s):
    """(index [E, most] of each expert's positions, whether each is real, position of every pair in that table)."""
    off = s["offsets"].long()
    at = torch.arange(s["most"], device=off.device)
    idx = off[:-1, None] + at
    real = idx < off[1:, None]
    pos = torch.arange(s["rows"].numel(), device=off.device)
    e = (pos[:, None] >= off[None, 1:]).sum(1)
    kept = e < off.numel() - 1
    e = torch.where(kept, e, 0)
    return torch.where(real, idx, 0), real, torch.where(kept, e * s["most"] + pos - off[e], 0), kept


def _plain_matmul(s):
    c = s["case"]
    idx, real, back, kept = _padded(s)
    dt = s["x"].dtype
    w = s["w"].float()
    src = s["rows"].long()[idx] if c["gather"] else idx
    xp = torch.where(real[:, :, None], s["x"].float()[torch.where(real, src, 0)], 0.0)
    y = torch.bmm(xp, w.transpose(1, 2)).reshape(-1, c["N"])[back]
    out = {"y": torch.where(kept[:, None], y, 0.0).to(dt)}
    if s["dy"] is None:
        return out
    dyp = torch.where(real[:, :, None], s["dy"].float()[idx], 0.0)
    dx = torch.where(kept[:, None], torch.bmm(dyp, w).reshape(-1, c["D"])[back], 0.0)
    if c["gather"]:
        slot = s["slot"].long()
        dx = torch.where((slot >= 0)[:, :, None], dx[slot.clamp(min=0)], 0.0).sum(1)
    out["dx"] = dx.to(dt)
    out["dw"] = torch.bmm(dyp.transpose(1, 2), xp).to(dt)
    return out


def _plain_combine(s):
    slot = s["slot"].long()
    got = slot >= 0
    at = torch.where(got, slot, 0)
    y = s["y"].float()
    w = torch.where(got, s["weights"] if s["weights"] is not None else 1.0, 0.0)
    yg = torch.where(got[:, :, None], y[at], 0.0)
    out = {"out": (yg * w[:, :, None]).sum(1).to(s["y"].dtype)}
    if s["dout"] is None:
        return out
    do = s["dout"].float()
    dy = torch.zeros_like(y)
    dy[slot[got]] = (w[:, :, None] * do[:, None, :])[got]
    out["dy"] = dy.to(s["y"].dtype)
    if s["weights"] is not None:
        out["dweights"] = (yg * do[:, None, :]).sum(2)
    return out


def _plain_group(s):
    offsets, rows, slot = _plan(s["ids"], s["case"]["E"])
    return {"offsets": offsets, "rows": rows, "slot": slot}


# ---------------------------------------------------------------- one pass

def _own_route(s):
    from mlx_kmeans_b200 import route, route_grad
    c = s["case"]
    ids, weights = route(s["logits"], c["k"], score=c["score"], bias=s["bias"], groups=c["groups"],
                         top_groups=c["top_groups"], renormalize=c["renorm"], scale=c["scale"], mask=s["mask"])
    out = {"ids": ids, "weights": weights}
    if s["dweights"] is not None:
        out["dlogits"] = route_grad(s["dweights"], s["logits"], ids, score=c["score"], renormalize=c["renorm"],
                                    scale=c["scale"])
    return out


def _own_group(s):
    from mlx_kmeans_b200 import group_rows
    g = group_rows(s["ids"], s["case"]["E"])
    return {"offsets": g.offsets, "rows": g.rows, "slot": g.slot}


def _own_matmul(s):
    from mlx_kmeans_b200 import RowGroups, expert_matmul, expert_matmul_grad
    c = s["case"]
    g = RowGroups(s["offsets"], s["rows"], s["slot"])
    out = {"y": expert_matmul(s["x"], s["w"], g, gather=c["gather"])}
    if s["dy"] is not None:
        out["dx"], out["dw"] = expert_matmul_grad(s["dy"], s["x"], s["w"], g, gather=c["gather"])
    return out


def _own_combine(s):
    from mlx_kmeans_b200 import RowGroups, combine_rows, combine_rows_grad
    g = RowGroups(s["offsets"], s["rows"], s["slot"])
    out = {"out": combine_rows(s["y"], g, s["weights"])}
    if s["dout"] is not None:
        out["dy"], dw = combine_rows_grad(s["dout"], s["y"], g, s["weights"])
        if s["weights"] is not None:
            out["dweights"] = dw
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"route": _own_route, "group": _own_group, "matmul": _own_matmul, "combine": _own_combine}[op](state)
    return {"route": _plain_route, "group": _plain_group, "matmul": _plain_matmul, "combine": _plain_combine}[op](state)


# ---------------------------------------------------------------- what a pass cannot do without

def _active(case, rows):
    """Expected number of experts with a row, for choices drawn by popularity."""
    p = torch.softmax(_popularity(case["E"]).double(), 0)
    return float((1.0 - (1.0 - torch.clamp(p * case["k"], max=1.0)) ** rows).sum())


def work(case):
    T, E, k = case["T"], case["E"], case["k"]
    real = T - case["masked"]
    if case["op"] == "route":
        b = SIZE[case["dtype"]]
        byts = T * E * b + T * k * 8 + (T if case["masked"] else 0) + (4 * E if case["bias"] else 0)
        flops = 4.0 * T * E
        if case["grad"]:
            byts += T * E * b + T * k * 4
            flops += 4.0 * T * (E if case["score"] == "softmax" and not case["renorm"] else k)
        return {"bytes": byts, "flops": flops}
    if case["op"] == "group":
        return {"bytes": 12 * T * k + 4 * (E + 1), "flops": 0}
    b = SIZE[case["dtype"]]
    if case["op"] == "matmul":
        N, D = case["N"], case["D"]
        x = (real if case["gather"] else real * k) * D * b
        w = _active(case, real) * N * D * b
        byts = x + w + T * k * N * b + 4 * T * k
        flops = 2.0 * real * k * N * D
        if case["grad"]:
            byts += real * k * N * b + (T if case["gather"] else T * k) * D * b + E * N * D * b
            flops *= 3
        return {"bytes": byts, "flops": flops}
    H = case["H"]
    byts = real * k * H * b + T * H * b + T * k * (8 if case["weighted"] else 4)
    flops = 2.0 * real * k * H
    if case["grad"]:
        byts += real * H * b + T * k * H * b + (4 * T * k if case["weighted"] else 0)
        flops += (3.0 if case["weighted"] else 0.0) * real * k * H
    return {"bytes": byts, "flops": flops}


# ---------------------------------------------------------------- float64

def _exact_route(c, s):
    T, E, k, d = c["T"], c["E"], c["k"], torch.float64
    l = s["logits"].to(d)
    live = torch.ones(T, dtype=torch.bool, device=l.device) if s["mask"] is None else s["mask"]
    score = l if c["score"] == "softmax" else torch.special.expit(l)
    key = score if s["bias"] is None else score + s["bias"].to(d)
    if c["groups"] > 1:
        per = key.view(T, c["groups"], -1)
        rank = per.sort(2, descending=True).values[:, :, :2].sum(2)
        chosen = rank.topk(c["top_groups"], dim=1).indices
        off = torch.ones(T, c["groups"], dtype=torch.bool, device=l.device)
        off[torch.arange(T, device=l.device)[:, None], chosen] = False
        key = key.masked_fill(off[:, :, None].expand(per.shape).reshape(T, E), -INF)
    pick = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    if c["score"] == "softmax":
        base = torch.full_like(l, -INF).scatter(1, pick, l.gather(1, pick)) if c["renorm"] else l
        prob = torch.softmax(base, 1)
    else:
        prob = score
        if c["renorm"]:
            prob = score / score.gather(1, pick).sum(1, keepdim=True)
    w = prob.gather(1, pick) * c["scale"] * live[:, None]
    out = {"ids": None, "weights": w}
    if s["dweights"] is not None:
        # the Jacobian of the scores times the incoming gradient, spread over the experts first
        up = s["dweights"].to(d) * live[:, None] * c["scale"]
        spread = torch.zeros_like(l).scatter_(1, pick, up)
        if c["score"] == "softmax":
            out["dlogits"] = prob * (spread - (spread * prob).sum(1, keepdim=True))
        else:
            slope = score * torch.special.expit(-l)
            chosen = torch.zeros_like(l).scatter_(1, pick, 1.0)
            if c["renorm"]:
                total = (score * chosen).sum(1, keepdim=True)
                out["dlogits"] = chosen * slope * (spread / total - (spread * score).sum(1, keepdim=True) / total ** 2)
            else:
                out["dlogits"] = slope * spread
            out["dlogits"] = out["dlogits"] * live[:, None]
    return out


def _exact_matmul(c, s):
    d = torch.float64
    off = s["offsets"].tolist()
    P, N, D = c["T"] * c["k"], c["N"], c["D"]
    x, dev = s["x"].to(d), s["x"].device
    y = torch.zeros(P, N, dtype=d, device=dev)
    out = {"y": y}
    if s["dy"] is not None:
        dx, dw = torch.zeros_like(x), torch.zeros(c["E"], N, D, dtype=d, device=dev)
        out |= {"dx": dx, "dw": dw}
    for e in range(c["E"]):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        at = s["rows"][a:b].long() if c["gather"] else torch.arange(a, b, device=dev)
        w = s["w"][e].to(d)
        y[a:b] = x[at] @ w.T
        if s["dy"] is not None:
            g = s["dy"][a:b].to(d)
            dx.index_add_(0, at, g @ w)
            dw[e] = g.T @ x[at]
    return out


def _exact_combine(c, s):
    d = torch.float64
    T, k, H = c["T"], c["k"], c["H"]
    out = torch.zeros(T, H, dtype=d, device=s["y"].device)
    grad = s["dout"] is not None
    dy = torch.zeros(T * k, H, dtype=d, device=out.device) if grad else None
    dw = torch.zeros(T, k, dtype=d, device=out.device)
    for j in range(k):
        t = (s["slot"][:, j] >= 0).nonzero()[:, 0]
        p = s["slot"][t, j].long()
        w = s["weights"][t, j].to(d) if s["weights"] is not None else torch.ones(len(t), dtype=d, device=out.device)
        v = s["y"][p].to(d)
        out.index_add_(0, t, v * w[:, None])
        if grad:
            up = s["dout"][t].to(d)
            dy[p] = up * w[:, None]
            dw[t, j] = torch.linalg.vecdot(up, v)
    res = {"out": out}
    if grad:
        res["dy"] = dy
        if s["weights"] is not None:
            res["dweights"] = dw
    return res


def exact(case, seed):
    if case["op"] == "group":
        return None                     # whole numbers only: the plain form's are the answer
    s = prepare(case, seed)
    return {"route": _exact_route, "matmul": _exact_matmul, "combine": _exact_combine}[case["op"]](case, s)
