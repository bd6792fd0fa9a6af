"""Cases of the routing operators: tokens sent to experts, the experts' products, and the way back.

Each case is one call of one operator: the routing of tokens by their scores and its gradient, the plan that
sorts the routed rows by expert, the product of every row with its expert's matrix with both gradients, and the
weighted sum of a token's expert rows with its gradients.  ``own`` selects between the plain torch form and the
calls of this package.
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one new token of a served model: the call is all latency
        {"name": "route one token", "op": "route", "n": 1, "experts": 64, "top_k": 6, "dtype": "bf16", "score": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "group_score": "max", "renormalize": True, "masked": 0.0},
        # a long prompt or a training batch, balanced by a bias, experts spread over groups of devices
        {"name": "route groups bias", "op": "route", "n": 32768, "experts": 256, "top_k": 8, "dtype": "fp32", "score": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "group_score": "top2", "renormalize": True, "masked": 0.0},
        # its gradient in training, an expert count that is no power of two, some experts masked off
        {"name": "route grad", "op": "route_grad", "n": 30001, "experts": 60, "top_k": 4, "dtype": "bf16", "score": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "group_score": "max", "renormalize": True, "masked": 0.05},
        # a serving batch of many sequences, some rows dropped
        {"name": "plan batch", "op": "plan", "n": 997, "experts": 160, "top_k": 6, "dropped": 0.1, "skew": 1.0},
        # a training batch: a million routed rows
        {"name": "plan training", "op": "plan", "n": 131072, "experts": 256, "top_k": 8, "dropped": 0.0, "skew": 0.5},
        # one new token: the chosen experts' weights are read once
        {"name": "product one token", "op": "product", "n": 1, "experts": 64, "top_k": 8, "k": 2048, "width": 1536, "dtype": "bf16",
         "gather": True, "dropped": 0.0, "skew": 0.5},
        # a serving batch: a few rows for every expert
        {"name": "product batch", "op": "product", "n": 96, "experts": 64, "top_k": 6, "k": 2048, "width": 1024, "dtype": "fp16",
         "gather": True, "dropped": 0.0, "skew": 1.0},
        # a long prompt or a training batch: matrix products of ragged heights
        {"name": "product training", "op": "product", "n": 8192, "experts": 32, "top_k": 4, "k": 4096, "width": 2048, "dtype": "bf16",
         "gather": True, "dropped": 0.0, "skew": 0.5},
        # gradient with respect to the rows, few large experts, an odd number of tokens
        {"name": "product grad x", "op": "product_grad_x", "n": 6001, "experts": 8, "top_k": 2, "k": 2048, "width": 4096, "dtype": "fp16",
         "gather": False, "dropped": 0.05, "skew": 0.5},
        # gradient with respect to the weights, many small experts with uneven loads
        {"name": "product grad w", "op": "product_grad_w", "n": 8192, "experts": 64, "top_k": 4, "k": 2048, "width": 1024, "dtype": "bf16",
         "gather": True, "dropped": 0.0, "skew": 1.0},
        # the way back to token order
        {"name": "combine", "op": "combine", "n": 8192, "experts": 64, "top_k": 8, "width": 2048, "dtype": "bf16", "dropped": 0.0,
         "skew": 0.5},
        # its gradients, for the rows and for the routing weights
        {"name": "combine grad", "op": "combine_grad", "n": 5003, "experts": 16, "top_k": 4, "width": 4096, "dtype": "fp16",
         "dropped": 0.05, "skew": 0.5},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "route", "route_grad", "plan", "product", "product", "product_grad_x", "product_grad_w", "combine", "combine_grad"])
    c = {"op": op}
    if op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 2, 4, 8])
        c["n"] = _log_int(rng, 1, 32768)
        c["experts"] = groups * max(2, _log_int(rng, 8, 256) // groups)
        c["groups"] = groups
        c["top_groups"] = rng.randint(1, groups)
        c["group_score"] = rng.choice(["max", "top2"])
        c["top_k"] = rng.randint(1, min(8, c["experts"] // groups * c["top_groups"]))
        c["dtype"] = rng.choice(["fp32", "fp16", "bf16"])
        c["score"] = rng.choice(["softmax", "sigmoid"])
        c["bias"] = rng.random() < 0.5
        c["renormalize"] = rng.random() < 0.7
        c["masked"] = rng.choice([0.0, 0.0, 0.05, 0.9])
        return c
    c["dropped"] = rng.choice([0.0, 0.0, 0.1])
    c["skew"] = rng.choice([0.0, 0.5, 1.0])
    if op == "plan":
        c["n"] = _log_int(rng, 1, 131072)
        c["experts"] = _log_int(rng, 4, 256)
        c["top_k"] = rng.randint(1, min(8, c["experts"]))
        return c
    c["n"] = _log_int(rng, 1, 8192)
    c["experts"] = _log_int(rng, 4, 64)
    c["top_k"] = rng.randint(1, min(8, c["experts"]))
    c["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
    # widths are whole 16-byte rows, as weight matrices have them
    c["width"] = 8 * _log_int(rng, 8, 512)
    if op in ("combine", "combine_grad"):
        return c
    c["k"] = 8 * _log_int(rng, 8, 512)
    c["gather"] = op != "product_grad_x" and rng.random() < 0.5
    while c["n"] * c["top_k"] * c["k"] * c["width"] > 8192 * 4 * 4096 * 2048 and c["n"] > 1:
        c["n"] = (c["n"] + 1) // 2
    while c["experts"] * c["k"] * c["width"] > 32 * 4096 * 2048 and c["experts"] > c["top_k"]:
        c["experts"] = max(c["top_k"], c["experts"] // 2)
    return c


def _route_options(case):
    return {"score": case["score"], "groups": case["groups"], "top_groups": case["top_groups"],
            "group_score": case["group_score"], "renormalize": case["renormalize"], "scale": 1.0}


def _routed(case, g):
    """ids (n x top_k, -1 where a row is dropped) of tokens that prefer some experts, and what a plan holds of them:
    the offsets of the experts' rows, the routed entry of every sorted row, the sorted row of every entry."""
    n, e, k = case["n"], case["experts"], case["top_k"]
    liking = case["skew"] * torch.randn(e, generator=g, device="cuda")
    ids = (torch.randn(n, e, generator=g, device="cuda") + liking).topk(k, dim=1).indices.to(torch.int32)
    if case["dropped"]:
        ids = torch.where(torch.rand(n, k, generator=g, device="cuda") < case["dropped"], torch.full_like(ids, -1), ids)
    return ids, *_sorted_by_expert(ids, e)


def _sorted_by_expert(ids, experts):
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    key, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device=ids.device))
    rows = torch.arange(flat.numel(), device=ids.device)
    pos = torch.empty_like(rows)
    pos[order] = torch.where(key < experts, rows, -1)
    order = torch.where(key < experts, order, -1)
    return offsets.to(torch.int32), order.to(torch.int32), pos.view(ids.shape).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, n = case["op"], case["n"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(_DTYPES[case["dtype"]])

    state = {"case": case}
    if op in ("route", "route_grad"):
        e = case["experts"]
        logits = normal(n, e, scale=1.5)
        if case["masked"]:
            logits.masked_fill_(torch.rand(n, e, generator=g, device="cuda") < case["masked"], float("-inf"))
        state["logits"] = logits
        state["bias"] = 0.1 * torch.randn(e, generator=g, device="cuda") if case["bias"] else None
        if op == "route_grad":
            state["ids"] = _plain_route(logits, state["bias"], case["top_k"], **_route_options(case))[0]
            state["grad"] = torch.randn(n, case["top_k"], generator=g, device="cuda")
        return state
    state["ids"], state["offsets"], state["order"], state["pos"] = _routed(case, g)
    if op == "plan":
        return state
    m, width = n * case["top_k"], case["width"]
    if op in ("combine", "combine_grad"):
        state["y"] = normal(m, width)
        state["weights"] = torch.rand(n, case["top_k"], generator=g, device="cuda")
        if op == "combine_grad":
            state["grad"] = normal(n, width)
        return state
    k = case["k"]
    state["most"] = int((state["offsets"][1:] - state["offsets"][:-1]).max())   # rows of the fullest expert
    if op != "product_grad_x":
        state["x"] = normal(n if case["gather"] else m, k)
    if op != "product":
        state["grad"] = normal(m, width)
    if op != "product_grad_w":
        state["w"] = normal(case["experts"], width, k, scale=1.0 / math.sqrt(k))
    return state


# ---------------------------------------------------------------- plain forms


def _scores(x, score):
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(1, keepdim=True)
    return torch.where(total > 0, e / total, torch.zeros_like(e))


def _plain_route(logits, bias, top_k, score, groups, top_groups, group_score, renormalize, scale):
    x = logits.double()              # choices are compared next to their borders
    s = _scores(x, score)
    c = s if bias is None else s + bias.double()
    nothing = torch.full_like(c, float("-inf"))
    c = torch.where(torch.isinf(x) & (x < 0), nothing, c)
    if groups > 1:
        per = c.view(c.shape[0], groups, -1)
        if group_score == "max":
            of = per.amax(2)
        else:
            two = torch.sort(per, dim=2, descending=True).values[:, :, :2]
            of = torch.where(torch.isinf(two), torch.zeros_like(two), two).sum(2)
            of = torch.where(torch.isinf(two[:, :, 0]), nothing[:, :groups], of)
        best = torch.sort(of, dim=1, descending=True, stable=True).indices[:, :top_groups]
        kept = torch.zeros_like(of, dtype=torch.bool).scatter_(1, best, True)
        c = torch.where(kept[:, :, None], per, nothing.view(per.shape)).view(c.shape)
    value, ids = torch.sort(c, dim=1, descending=True, stable=True)
    value, ids = value[:, :top_k], ids[:, :top_k]
    w = torch.where(torch.isinf(value), torch.zeros_like(value), s.gather(1, ids))
    ids = torch.where(torch.isinf(value), -1, ids)
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
    return ids.to(torch.int32), (w * scale).float()


def _plain_route_grad(grad, logits, ids, score, renormalize, scale):
    s = _scores(logits.float(), score)
    there = ids >= 0
    at = ids.clamp(min=0).long()
    chosen = torch.where(there, s.gather(1, at), torch.zeros_like(grad))
    g = torch.where(there, grad * scale, torch.zeros_like(grad))
    if renormalize:
        total = chosen.sum(1, keepdim=True)
        total = torch.where(total > 0, total, torch.full_like(total, float("inf")))
        g = (g - (g * chosen).sum(1, keepdim=True) / total) / total
        g = torch.where(there, g, torch.zeros_like(g))
    ds = torch.zeros_like(s).scatter_add_(1, at, g)
    if score == "sigmoid":
        dx = ds * s * (1 - s)
    else:
        dx = s * (ds - (ds * s).sum(1, keepdim=True))
    return dx.to(logits.dtype)


def _expert_of_row(s, m):
    rows = torch.arange(m, device="cuda")
    expert = torch.searchsorted(s["offsets"][1:].long(), rows, right=True)
    return rows, expert


def _padded(s, rows):
    """rows (m x width, sorted by expert) as experts x most x width, zero behind each expert's last row."""
    e = s["case"]["experts"]
    at = s["offsets"][:-1, None].long() + torch.arange(s["most"], device="cuda")
    inside = at < s["offsets"][1:, None]
    out = rows[torch.where(inside, at, 0)]
    return torch.where(inside[:, :, None], out, torch.zeros_like(out)).view(e, s["most"], rows.shape[1])


def _rows_of(s, padded, m):
    """The inverse of _padded; rows that no expert has are zero."""
    e = s["case"]["experts"]
    rows, expert = _expert_of_row(s, m)
    some = expert < e
    expert = expert.clamp(max=e - 1)
    at = (rows - s["offsets"][expert].long()).clamp(0, s["most"] - 1)
    out = padded[expert, at]
    return torch.where(some[:, None], out, torch.zeros_like(out))


def _sorted_x(s):
    x = s["x"].float()
    if not s["case"]["gather"]:
        return x
    return x[torch.div(s["order"].clamp(min=0), s["case"]["top_k"], rounding_mode="floor").long()]


def _plain_rows_times(s, rows, w):
    """rows (m x a) times the transpose of each row's expert matrix (experts x b x a), m x b."""
    m, e = rows.shape[0], s["case"]["experts"]
    if s["most"] == 0:
        return torch.zeros(m, w.shape[1], device="cuda")
    if m <= e:                       # few rows: only their experts' matrices
        _, expert = _expert_of_row(s, m)
        out = torch.bmm(w[expert.clamp(max=e - 1)].float(), rows[:, :, None])[:, :, 0]
        return torch.where((expert < e)[:, None], out, torch.zeros_like(out))
    return _rows_of(s, torch.bmm(_padded(s, rows), w.float().transpose(1, 2)), m)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "route":
        return _plain_route(s["logits"], s["bias"], case["top_k"], **_route_options(case))
    if op == "route_grad":
        return _plain_route_grad(s["grad"], s["logits"], s["ids"], case["score"], case["renormalize"], 1.0)
    if op == "plan":
        return _sorted_by_expert(s["ids"], case["experts"])
    if op == "product":
        return _plain_rows_times(s, _sorted_x(s), s["w"]).to(s["x"].dtype)
    if op == "product_grad_x":
        return _plain_rows_times(s, s["grad"].float(), s["w"].transpose(1, 2)).to(s["grad"].dtype)
    if op == "product_grad_w":
        if s["most"] == 0:
            return torch.zeros(case["experts"], case["width"], case["k"], device="cuda", dtype=s["x"].dtype)
        return torch.bmm(_padded(s, s["grad"].float()).transpose(1, 2), _padded(s, _sorted_x(s))).to(s["x"].dtype)
    there = (s["pos"] >= 0)[:, :, None]
    y = s["y"][s["pos"].clamp(min=0).long()].float()
    if op == "combine":
        return torch.where(there, s["weights"][:, :, None] * y, torch.zeros_like(y)).sum(1).to(s["y"].dtype)
    g = s["grad"].float()
    dw = torch.where(there, g[:, None, :] * y, torch.zeros_like(y)).sum(2)
    at = s["order"].clamp(min=0).long()
    token = torch.div(at, case["top_k"], rounding_mode="floor")
    dy = s["weights"].view(-1)[at][:, None] * g[token]
    return torch.where((s["order"] >= 0)[:, None], dy, torch.zeros_like(dy)).to(s["y"].dtype), dw


def _own(s):
    import mpkmeans_b200 as M

    case = s["case"]
    op = case["op"]
    if op == "route":
        return M.route(s["logits"], case["top_k"], bias=s["bias"], **_route_options(case))
    if op == "route_grad":
        return M.route_grad(s["grad"], s["logits"], s["ids"], score=case["score"], renormalize=case["renormalize"], scale=1.0)
    if op == "plan":
        p = M.expert_plan(s["ids"], case["experts"])
        return p.offsets, p.order, p.pos
    plan = M.ExpertPlan(s["offsets"], s["order"], s["pos"])
    if op == "product":
        return M.expert_gemm(s["x"], s["w"], plan, gather=case["gather"])
    if op == "product_grad_x":
        return M.expert_gemm_grad_x(s["grad"], s["w"], plan)
    if op == "product_grad_w":
        return M.expert_gemm_grad_w(s["grad"], s["x"], plan, gather=case["gather"])
    if op == "combine":
        return M.expert_combine(s["y"], plan, s["weights"])
    return M.expert_combine_grad(s["grad"], s["y"], plan, s["weights"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    op, n, top_k, experts = case["op"], case["n"], case["top_k"], case["experts"]
    size = 4 if case.get("dtype") == "fp32" else 2
    m = n * top_k
    if op == "route":
        return {"bytes": n * experts * size + m * 8 + (4 * experts if case["bias"] else 0), "flops": 4 * n * experts}
    if op == "route_grad":
        return {"bytes": 2 * n * experts * size + m * 8, "flops": 6 * n * experts}
    if op == "plan":
        return {"bytes": 3 * 4 * m + 4 * (experts + 1), "flops": 0}
    width = case["width"]
    kept = m * (1 - case["dropped"])
    if op == "combine":
        return {"bytes": kept * width * size + n * width * size + m * 8, "flops": 2 * kept * width}
    if op == "combine_grad":
        return {"bytes": 2 * kept * width * size + n * width * size + m * 12, "flops": 3 * kept * width}
    k = case["k"]
    used = experts * (1 - (1 - 1 / experts) ** m)      # experts that some row goes to, for an even routing
    x = (n if case["gather"] else kept) * k * size
    matrices = (experts if op == "product_grad_w" else used) * width * k * size
    rows = kept * (k if op == "product_grad_x" else 0) * size
    return {"bytes": (rows if op == "product_grad_x" else x) + matrices + kept * width * size, "flops": 2 * kept * k * width}


# ------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op, n, top_k, experts = case["op"], case["n"], case["top_k"], case["experts"]
    if op == "plan":
        return None
    if op in ("route", "route_grad"):
        x = s["logits"].double()
        if case["score"] == "softmax":
            p = torch.nan_to_num(torch.exp(x - torch.logsumexp(x, 1, keepdim=True)), nan=0.0)
        else:
            p = torch.special.expit(x)
        if op == "route":
            # the choice is a whole number: held to the plain form's; the weights follow from it
            ids = _plain_route(s["logits"], s["bias"], top_k, **_route_options(case))[0].long()
            w = torch.gather(p, 1, ids.clamp(min=0)) * (ids >= 0)
            if case["renormalize"]:
                w = torch.nan_to_num(w / w.sum(1, keepdim=True), nan=0.0)
            return None, w
        ids = s["ids"].long()
        x = torch.where(torch.isinf(x), torch.full_like(x, -1e4), x).requires_grad_(True)
        p = torch.softmax(x, 1) if case["score"] == "softmax" else torch.sigmoid(x)
        w = torch.gather(p, 1, ids.clamp(min=0)) * (ids >= 0)
        if case["renormalize"]:
            w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
        (w * s["grad"].double()).sum().backward()
        some = (ids >= 0).any(1, keepdim=True)
        return x.grad * some
    order, bounds = s["order"].long(), s["offsets"].tolist()
    token = order.clamp(min=0) // top_k
    if op in ("combine", "combine_grad"):
        width = case["width"]
        kept = bounds[-1]
        out = torch.zeros(n, width, dtype=torch.float64, device="cuda")
        wr = s["weights"].double().view(-1)[order[:kept]]
        y = s["y"][:kept].double()
        if op == "combine":
            return out.index_add_(0, token[:kept], wr[:, None] * y)
        g = s["grad"].double()[token[:kept]]
        dy = torch.zeros(n * top_k, width, dtype=torch.float64, device="cuda")
        dy[:kept] = wr[:, None] * g
        dw = torch.zeros(n * top_k, dtype=torch.float64, device="cuda")
        dw[order[:kept]] = torch.linalg.vecdot(g, y)
        return dy, dw.view(n, top_k)
    k, width, m = case["k"], case["width"], n * top_k
    if op == "product_grad_w":
        out = torch.zeros(experts, width, k, dtype=torch.float64, device="cuda")
    else:
        out = torch.zeros(m, width if op == "product" else k, dtype=torch.float64, device="cuda")
    for e in range(experts):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        if op != "product_grad_x":
            x = s["x"][token[lo:hi] if case["gather"] else slice(lo, hi)].double()
        if op == "product":
            out[lo:hi] = x @ s["w"][e].double().T
        elif op == "product_grad_x":
            out[lo:hi] = s["grad"][lo:hi].double() @ s["w"][e].double()
        else:
            out[e] = s["grad"][lo:hi].double().T @ x
    return out
