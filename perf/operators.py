"""Cases, plain forms and exact values of the adapter and router-training operators.

Three operators, named by a case's ``"op"``:

``adapter``  y[t] = x[t].W + s_a (x[t].A_a).B_a with a = ids[t] (< 0: no adapter): the low-rank adapters of many
             requests beside one shared projection (``latent_b200.adapter_project``).
``balance``  the load-balance and z losses of a router over packed sequences, the expert counts, and the gradient of
             the loss with respect to the logits (``latent_b200.balance_loss``).
``route``    the gradient of the routing weights of ``latent_b200.router_topk`` with respect to its scores or logits
             (``latent_b200.router_topk_grad``).

With ``own`` false ``run`` computes them in elementary torch operations in 32 bits, rounded once at the end; with
``own`` true it makes the calls a user makes.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}

# The adapter case with the most multiply-adds; a drawn case has no more.
MOST_MACS = 8192 * 4096 * 14336


def listed():
    return [
        # one request decoding alone beside a 2048-wide projection: latency is all that counts
        {"name": "adapter_one_token", "op": "adapter", "dtype": "bf16", "out": "bf16", "layout": "kn", "T": 1, "K": 2048,
         "N": 2048, "n": 8, "r": 16, "requests": 1, "bare": 0},
        # a decode batch, a request and an adapter per token, some requests on the base model only
        {"name": "adapter_decode_32", "op": "adapter", "dtype": "bf16", "out": "bf16", "layout": "nk", "T": 32, "K": 2048,
         "N": 1408, "n": 48, "r": 16, "requests": 32, "bare": 4},
        # a wide layer's up projection for 64 decoding requests that share 24 adapters of larger rank
        {"name": "adapter_decode_64_wide", "op": "adapter", "dtype": "bf16", "out": "bf16", "layout": "kn", "T": 64,
         "K": 7168, "N": 2048, "n": 24, "r": 64, "requests": 64, "bare": 8},
        # router logits of 64 decoding requests with adapted routers: few columns, fp32 results for the top-k
        {"name": "adapter_router_logits", "op": "adapter", "dtype": "bf16", "out": "f32", "layout": "nk", "T": 64, "K": 7168,
         "N": 256, "n": 16, "r": 8, "requests": 64, "bare": 0},
        # five prompts packed to an odd length, fp16, odd rank
        {"name": "adapter_prompts_2047", "op": "adapter", "dtype": "f16", "out": "f16", "layout": "nk", "T": 2047, "K": 4096,
         "N": 4096, "n": 6, "r": 33, "requests": 5, "bare": 0},
        # sixteen prompts beside the widest projection of the shipped configurations: the largest case
        {"name": "adapter_prompts_8192", "op": "adapter", "dtype": "bf16", "out": "bf16", "layout": "kn", "T": 8192,
         "K": 4096, "N": 14336, "n": 12, "r": 16, "requests": 16, "bare": 2},
        # a small calibration batch: launch latency
        {"name": "balance_64", "op": "balance", "dtype": "f32", "T": 64, "E": 64, "k": 6, "sequences": 1, "padded": 0,
         "behind": 0, "dropped": 0, "z": 0},
        # a training batch of the 256-expert layer, a loss per packed sequence, with the z loss
        {"name": "balance_16384", "op": "balance", "dtype": "f32", "T": 16384, "E": 256, "k": 8, "sequences": 8,
         "padded": 0, "behind": 0, "dropped": 1, "z": 1},
        # bf16 logits, padded rows inside sequences of odd lengths (some empty) and rows behind the last one
        {"name": "balance_ragged_9001", "op": "balance", "dtype": "bf16", "T": 9001, "E": 160, "k": 6, "sequences": 37,
         "padded": 1, "behind": 1, "dropped": 1, "z": 1},
        # router gradient of a small batch
        {"name": "route_64", "op": "route", "dtype": "f32", "T": 64, "E": 64, "k": 6, "logits": 1, "renorm": 1,
         "dropped": 0},
        # the 256-expert layer's training batch: renormalised weights of softmax logits
        {"name": "route_16384", "op": "route", "dtype": "f32", "T": 16384, "E": 256, "k": 8, "logits": 1, "renorm": 1,
         "dropped": 1},
        # raw softmax weights (a dense gradient row) of bf16 logits, odd sizes
        {"name": "route_raw_9001", "op": "route", "dtype": "bf16", "T": 9001, "E": 160, "k": 6, "logits": 1, "renorm": 0,
         "dropped": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["adapter", "adapter", "balance", "route"])
    if op == "adapter":
        dtype = rng.choice(["bf16", "f16"])
        case = {"op": op, "dtype": dtype, "out": rng.choice([dtype, dtype, "f32"]), "layout": rng.choice(["kn", "nk"]),
                "T": _log(rng, 1, 8192), "K": 8 * _log(rng, 32, 896), "N": 8 * _log(rng, 8, 1792), "r": _log(rng, 4, 64),
                "n": _log(rng, 1, 64)}
        while case["T"] * case["K"] * case["N"] > MOST_MACS:
            case["T"] = case["T"] // 2 + 1
        # a batch of single tokens is one request a row; a prompt batch packs up to 32 of them
        case["requests"] = case["T"] if case["T"] <= 256 else min(case["T"], _log(rng, 1, 32))
        case["bare"] = rng.choice([0, 0, case["requests"] // 4])
        return case
    T, E = _log(rng, 1, 16384), _log(rng, 4, 256)
    # a gradient of order 1 / T is below what fp16 holds: the losses' logits are fp32 or bf16
    case = {"op": op, "dtype": rng.choice(["f32", "bf16"] if op == "balance" else ["f32", "bf16", "f16"]), "T": T, "E": E,
            "k": rng.randint(2, min(8, E)), "dropped": rng.choice([0, 1])}
    if op == "balance":
        case.update(sequences=min(T, _log(rng, 1, 64)), padded=rng.choice([0, 1]), behind=rng.choice([0, 1]),
                    z=rng.choice([0, 1]))
    else:
        case.update(logits=rng.choice([1, 1, 0]), renorm=rng.choice([0, 1]))
        if not case["logits"]:
            case["dtype"] = "f32"
    return case


# ---------------------------------------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1_000_003 * int(seed) + 17)
    return g


def _cuts(total, parts, g):
    """parts + 1 ascending borders from 0 to total: random lengths, some of them zero when there are many."""
    inner = torch.randint(0, total + 1, (parts - 1,), generator=g, device=DEV).sort().values
    ends = torch.tensor([0, total], device=DEV)
    return torch.cat([ends[:1], inner, ends[1:]])


def _scale(i):
    return 0.5 + 0.25 * (i % 5)


def _rank(case, i):
    """Adapters have different ranks: every third one half the case's rank."""
    return max(1, case["r"] // 2) if i % 3 == 2 else case["r"]


def _prepare_adapter(case, seed):
    g, dt = _gen(seed), TYPES[case["dtype"]]
    T, K, N, n, r = (case[k] for k in ("T", "K", "N", "n", "r"))
    x = torch.randn((T, K), generator=g, device=DEV).to(dt)
    w = (torch.randn((K, N) if case["layout"] == "kn" else (N, K), generator=g, device=DEV) / math.sqrt(K)).to(dt)
    weight = w if case["layout"] == "kn" else w.t()           # a linear layer's weight, used transposed
    a = (torch.randn((n, K, r), generator=g, device=DEV) / math.sqrt(K)).to(dt)
    b = (torch.randn((n, r, N), generator=g, device=DEV) * 0.1).to(dt)
    ranks = torch.tensor([_rank(case, i) for i in range(n)], device=DEV)
    live = torch.arange(r, device=DEV)[None, :] < ranks[:, None]
    a, b = a * live[:, None, :], b * live[:, :, None]
    scales = torch.tensor([_scale(i) for i in range(n)], device=DEV)
    # requests in a random order of adapters; the last `bare` of them use the base model alone
    which = torch.randperm(case["requests"], generator=g, device=DEV) % n
    if case["bare"]:
        which[torch.randperm(case["requests"], generator=g, device=DEV)[:case["bare"]]] = -1
    if case["requests"] == T:
        ids = which
    else:
        ends = _cuts(T, case["requests"], g)
        ids = which[torch.bucketize(torch.arange(T, device=DEV), ends[1:-1].contiguous(), right=True)]
    state = {"case": case, "x": x, "weight": weight, "ids": ids.to(torch.int32).contiguous(), "a": a, "b": b,
             "scales": scales}
    if own:
        from latent_b200 import AdapterSet
        state["set"] = AdapterSet([(a[i][:, :_rank(case, i)], b[i][:_rank(case, i)], _scale(i)) for i in range(n)],
                                  device=x.device, dtype=dt)
    return state


def _router_inputs(case, g):
    """Logits of a router (a per-expert bias skews the load) and their top-k ids; with `dropped` the tail slots of some
    rows are -1, as the adaptive threshold leaves them."""
    T, E, k, dt = case["T"], case["E"], case["k"], TYPES[case["dtype"]]
    bias = torch.randn((E,), generator=g, device=DEV)
    logits = (1.5 * torch.randn((T, E), generator=g, device=DEV) + bias).to(dt)
    ids = torch.topk(logits.float() + 1e-6 * torch.rand((T, E), generator=g, device=DEV), k, dim=1).indices
    if case["dropped"]:
        kept = torch.randint(1, k + 1, (T, 1), generator=g, device=DEV)
        ids = torch.where(torch.arange(k, device=DEV)[None, :] < kept, ids, -1)
    return logits, ids.to(torch.int32).contiguous()


def _prepare_balance(case, seed):
    g = _gen(seed)
    logits, ids = _router_inputs(case, g)
    T = case["T"]
    end = T - T // 16 if case["behind"] else T
    cu = _cuts(end, case["sequences"], g).to(torch.int32)
    valid = None
    if case["padded"]:
        valid = torch.rand((T,), generator=g, device=DEV) < 0.9
    return {"case": case, "logits": logits, "ids": ids, "cu": cu, "valid": valid, "balance": 0.01,
            "z": 0.001 if case["z"] else 0.0}


def _prepare_route(case, seed):
    g = _gen(seed)
    logits, ids = _router_inputs(case, g)
    scores = logits if case["logits"] else torch.softmax(logits, dim=1)
    dw = torch.randn(ids.shape, generator=g, device=DEV)
    return {"case": case, "scores": scores, "ids": ids, "dw": dw}


def prepare(case, seed):
    return {"adapter": _prepare_adapter, "balance": _prepare_balance, "route": _prepare_route}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------------- one pass


def run(state):
    return {"adapter": _run_adapter, "balance": _run_balance, "route": _run_route}[state["case"]["op"]](state)


def _run_adapter(s):
    c = s["case"]
    out = TYPES[c["out"]]
    if own:
        from latent_b200 import adapter_project
        return adapter_project(s["x"], s["weight"], s["set"], s["ids"], out_dtype=out)
    n, r = c["n"], c["r"]
    x, ids = s["x"].float(), s["ids"].long()
    y = x @ s["weight"].float()
    t_all = x @ s["a"].float().permute(1, 0, 2).reshape(c["K"], n * r)      # every adapter's x.A ...
    t_all = t_all.view(-1, n, r) * s["scales"][None, :, None]
    mine = ids[:, None] == torch.arange(n, device=x.device)[None, :]        # ... of which a row keeps its own
    t = torch.where(mine[:, :, None], t_all, 0.0).view(-1, n * r)
    return (y + t @ s["b"].float().reshape(n * r, c["N"])).to(out)


def _segments(cu, valid, T):
    """Segment of each row (-1: behind the last sequence or masked) as a one-hot [T, S] in fp32."""
    rows = torch.arange(T, device=cu.device)
    seg = (rows[:, None] >= cu[None, :-1]) & (rows[:, None] < cu[None, 1:])
    return seg if valid is None else seg & valid[:, None]


def _run_balance(s):
    c = s["case"]
    if own:
        from latent_b200 import balance_loss
        r = balance_loss(s["logits"], s["ids"], balance_coef=s["balance"], z_coef=s["z"], valid=s["valid"],
                         cu_seqlens=s["cu"], gradient=True)
        return {"loss": r.loss, "balance": r.balance, "z": r.z, "counts": r.counts, "grad": r.grad}
    T, E = c["T"], c["E"]
    l, ids = s["logits"].float(), s["ids"].long()
    seg = _segments(s["cu"], s["valid"], T).float()
    live = seg.sum(1, keepdim=True)                                       # 1 for counted rows
    m = l.max(dim=1, keepdim=True).values
    ex = torch.exp(l - m)
    total = ex.sum(1, keepdim=True)
    p, lse = ex / total, m + torch.log(total)
    hot = (ids[:, :, None] == torch.arange(E, device=l.device)).sum(1).float()
    counts = seg.t() @ hot                                                # [S, E]
    n = seg.sum(0)                                                        # tokens per sequence
    used = (n > 0).sum().clamp(min=1).float()
    f = counts / counts.sum(1, keepdim=True).clamp(min=1)
    n1 = n.clamp(min=1)
    mean_p = (seg.t() @ p) / n1[:, None]
    balance = (E * (f * mean_p).sum()) / used
    all_n = n.sum().clamp(min=1)
    z = (live * lse * lse).sum() / all_n
    row_f = seg @ (f * (s["balance"] * E / used / n1)[:, None])           # the row's sequence, scaled
    g = p * (row_f - (row_f * p).sum(1, keepdim=True)) + live * p * lse * (2.0 * s["z"] / all_n)
    return {"loss": s["balance"] * balance + s["z"] * z, "balance": balance, "z": z, "counts": counts.to(torch.int32),
            "grad": g.to(s["logits"].dtype)}


def _run_route(s):
    c = s["case"]
    if own:
        from latent_b200 import router_topk_grad
        return router_topk_grad(s["scores"], s["ids"], s["dw"], renormalize=bool(c["renorm"]), logits=bool(c["logits"]))
    v, ids = s["scores"].float(), s["ids"].long()
    kept = ids >= 0
    at = ids.clamp(min=0)
    if c["logits"]:
        ex = torch.exp(v - v.max(dim=1, keepdim=True).values)
        p = ex / ex.sum(1, keepdim=True)
    else:
        p = v
    pk = torch.where(kept, p.gather(1, at), 0.0)
    dw = torch.where(kept, s["dw"], 0.0)
    if c["renorm"]:
        total = pk.sum(1, keepdim=True)
        w = pk / total
        gk = (dw - (w * dw).sum(1, keepdim=True)) / total                 # with respect to the kept scores
        gk = torch.where(kept, gk, 0.0)
    else:
        gk = dw
    g = torch.zeros_like(p).scatter_add_(1, at, gk)
    if c["logits"]:
        g = p * (g - (g * p).sum(1, keepdim=True))
    return g.to(s["scores"].dtype)


# ---------------------------------------------------------------------------------------------- work


def work(case):
    if case["op"] == "adapter":
        T, K, N, r = (case[k] for k in ("T", "K", "N", "r"))
        adapted = T * (case["requests"] - case["bare"]) / max(1, case["requests"])
        used = min(case["n"], case["requests"] - case["bare"])
        e = SIZE[case["dtype"]]
        return {"bytes": e * (T * K + K * N + used * r * (K + N)) + SIZE[case["out"]] * T * N + 4 * T,
                "flops": 2 * T * K * N + 2 * adapted * r * (K + N)}
    T, E, k, e = case["T"], case["E"], case["k"], SIZE[case["dtype"]]
    if case["op"] == "balance":
        return {"bytes": 2 * T * E * e + 4 * T * k + (T if case["padded"] else 0) + 4 * case["sequences"] * (E + 1),
                "flops": 12 * T * E}
    # renormalised weights of softmax logits depend on the kept logits alone; raw softmax weights need the whole row
    read = T * k * e if case["renorm"] or not case["logits"] else T * E * e
    return {"bytes": read + T * E * e + 8 * T * k, "flops": 8 * T * E}


# ---------------------------------------------------------------------------------------------- exact values


def exact(case, seed):
    s = prepare(case, seed)
    return {"adapter": _exact_adapter, "balance": _exact_balance, "route": _exact_route}[case["op"]](s)


def _exact_adapter(s):
    c = s["case"]
    x, ids = s["x"].double(), s["ids"]
    y = torch.empty((c["T"], c["N"]), dtype=torch.float64, device=x.device)
    w = s["weight"].double()
    for lo in range(0, c["T"], 1024):
        y[lo:lo + 1024] = x[lo:lo + 1024] @ w
    for i in range(c["n"]):
        rows = (ids == i).nonzero()[:, 0]
        if rows.numel():
            y[rows] += float(s["scales"][i]) * ((x[rows] @ s["a"][i].double()) @ s["b"][i].double())
    return y


def _exact_balance(s):
    c = s["case"]
    T, E = c["T"], c["E"]
    l = s["logits"].double()
    lse = torch.logsumexp(l, dim=1)
    p = torch.softmax(l, dim=1)
    valid = torch.ones(T, dtype=torch.bool, device=l.device) if s["valid"] is None else s["valid"]
    cu = s["cu"].tolist()
    counts = torch.zeros((c["sequences"], E), dtype=torch.int64, device=l.device)
    parts, coef = [], torch.zeros((T, E), dtype=torch.float64, device=l.device)
    counted = torch.zeros(T, dtype=torch.bool, device=l.device)
    for i, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
        rows = torch.arange(lo, hi, device=l.device)[valid[lo:hi]]
        if not rows.numel():
            continue
        counted[rows] = True
        e = s["ids"][rows].reshape(-1).long()
        counts[i] = torch.bincount(e[e >= 0], minlength=E)
        f = counts[i].double() / max(1, int(counts[i].sum()))
        parts.append(E * (f * p[rows].mean(0)).sum())
        coef[rows] = E * f / rows.numel()
    n, used = max(1, int(counted.sum())), max(1, len(parts))
    balance = sum(parts) / used if parts else torch.zeros((), dtype=torch.float64, device=l.device)
    z = (lse[counted] ** 2).sum() / n
    coef = coef * (s["balance"] / used)
    g = p * (coef - (coef * p).sum(1, keepdim=True)) + torch.where(counted, 2 * s["z"] * lse / n, 0.0)[:, None] * p
    return {"loss": s["balance"] * balance + s["z"] * z, "balance": balance, "z": z, "counts": counts.to(torch.int32),
            "grad": g}


def _exact_route(s):
    """By differentiating the weights in 64 bits."""
    c = s["case"]
    v = s["scores"].double().requires_grad_(True)
    p = torch.softmax(v, dim=1) if c["logits"] else v
    kept = s["ids"] >= 0
    w = p.gather(1, s["ids"].clamp(min=0).long()) * kept
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return torch.autograd.grad((w * s["dw"].double() * kept).sum(), v)[0]
