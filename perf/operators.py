"""The grouped operators of this package as measured work: products grouped by expert, low-rank adapters, the router.

`run` computes one pass in plain torch (`own` false) or through the package's public entry points (`own` true).
"""
import math

import torch

own = False

BF16, FP16, FP32 = "bfloat16", "float16", "float32"


def listed():
    return [
        # the router: one token being decoded, a large prompt batch, a training step with the gradient of the scores
        {"name": "route one token", "op": "route", "tokens": 1, "experts": 128, "k": 8, "dtype": BF16, "renormalize": True, "train": False},
        {"name": "route prompts", "op": "route", "tokens": 16384, "experts": 128, "k": 8, "dtype": BF16, "renormalize": True, "train": False},
        {"name": "route training", "op": "route", "tokens": 5001, "experts": 60, "k": 4, "dtype": FP32, "renormalize": False, "train": True},
        # the experts' up projection: one token being decoded, a decode batch, prompts
        {"name": "experts one token", "op": "experts", "tokens": 1, "experts": 128, "k": 8, "K": 2048, "N": 1536, "dtype": BF16, "tree": False, "train": False},
        {"name": "experts decode batch", "op": "experts", "tokens": 64, "experts": 128, "k": 8, "K": 2048, "N": 1536, "dtype": BF16, "tree": False, "train": False},
        {"name": "experts prompts", "op": "experts", "tokens": 4096, "experts": 64, "k": 8, "K": 2048, "N": 1536, "dtype": BF16, "tree": False, "train": False},
        # the row-split down projection: K summed in the tree that tensor-parallel shards share
        {"name": "experts down, row-split", "op": "experts", "tokens": 2048, "experts": 64, "k": 8, "K": 1536, "N": 2048, "dtype": FP16, "tree": True, "train": False},
        # training: output and both gradients, a full step and an odd one
        {"name": "experts training", "op": "experts", "tokens": 8192, "experts": 32, "k": 2, "K": 2048, "N": 2048, "dtype": BF16, "tree": False, "train": True},
        {"name": "experts training, odd", "op": "experts", "tokens": 1003, "experts": 7, "k": 3, "K": 520, "N": 1000, "dtype": BF16, "tree": False, "train": True},
        # adapters beside o_proj of the benchmark's layer: one token, a decode batch of many requests, prompts
        {"name": "adapters one token", "op": "adapters", "tokens": 1, "requests": 1, "adapters": 16, "rank": 16, "K": 4096, "N": 4096, "dtype": BF16},
        {"name": "adapters decode batch", "op": "adapters", "tokens": 96, "requests": 96, "adapters": 48, "rank": 16, "K": 12288, "N": 4096, "dtype": BF16},
        {"name": "adapters prompts", "op": "adapters", "tokens": 8192, "requests": 24, "adapters": 16, "rank": 32, "K": 4096, "N": 4096, "dtype": BF16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "adapters", "adapters"])
    if op == "route":
        experts = _log(rng, 2, 512)
        return {"op": op, "tokens": _log(rng, 1, 16384), "experts": experts, "k": rng.randint(1, min(experts, 16)),
                "dtype": rng.choice([BF16, FP16, FP32]), "renormalize": rng.random() < 0.5, "train": rng.random() < 0.5}
    while True:
        if op == "experts":
            experts, tree, train = _log(rng, 2, 128), rng.random() < 0.3, rng.random() < 0.4
            k_step = 512 if tree else 8
            case = {"op": op, "tokens": _log(rng, 1, 8192), "experts": experts, "k": rng.randint(1, min(experts, 8)),
                    "K": k_step * _log(rng, max(1, 64 // k_step), 4096 // k_step), "N": 8 * _log(rng, 8, 512),
                    "dtype": rng.choice([BF16, BF16, FP16]), "tree": tree, "train": train and not tree}
            flops = 2 * case["tokens"] * case["k"] * case["K"] * case["N"] * (3 if case["train"] else 1)
            if flops <= 2.0e11 and experts * case["K"] * case["N"] <= 4.0e8:
                return case
        else:
            tokens = _log(rng, 1, 8192)
            case = {"op": op, "tokens": tokens, "requests": min(tokens, _log(rng, 1, 96)), "adapters": _log(rng, 1, 64),
                    "rank": 8 * rng.randint(1, 8), "K": 8 * _log(rng, 32, 1536), "N": 8 * _log(rng, 32, 1536),
                    "dtype": rng.choice([BF16, BF16, FP16])}
            if 2 * tokens * (case["K"] + case["N"]) * case["adapters"] * case["rank"] <= 1.0e11 and tokens * (case["K"] + case["N"]) <= 7.0e7:
                return case


def _type(case):
    return getattr(torch, case["dtype"])


def _grouping(ids, groups):
    """(order, position, offsets) of rows sorted by group; ids below zero belong to none and come last."""
    key = torch.where(ids < 0, groups, ids)
    order = torch.sort(key, stable=True).indices
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=ids.device)
    offsets = torch.zeros(groups + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.cumsum(torch.bincount(key, minlength=groups + 1)[:groups], 0)
    return order.to(torch.int32), position.to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype or _type(case))

    s = {"case": case}
    T = case["tokens"]
    if case["op"] == "route":
        E = case["experts"]
        # some experts are liked more than others
        s["logits"] = normal(T, E) + normal(E, scale=0.5)
        if case["train"]:
            s["logits"].requires_grad_(True)
            s["dw"] = normal(T, case["k"], dtype=torch.float32)
    elif case["op"] == "experts":
        E, K, N = case["experts"], case["K"], case["N"]
        scores = normal(T, E, dtype=torch.float32) + normal(E, scale=0.5, dtype=torch.float32)
        ids = torch.topk(scores, case["k"]).indices.flatten()
        s["offsets"] = _grouping(ids, E)[2]
        s["longest"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())  # the plain form pads every group to it
        s["x"] = normal(T * case["k"], K)
        s["w"] = torch.empty(E, N, K, device="cuda", dtype=_type(case)).normal_(0.0, 0.02, generator=g)
        if case["train"]:
            s["x"].requires_grad_(True)
            s["w"].requires_grad_(True)
            s["dy"] = normal(T * case["k"], N, scale=0.1)
    else:
        L, R, K, N = case["adapters"], case["rank"], case["K"], case["N"]
        # requests of uneven lengths, each with one adapter; about one in eight has none
        request = torch.sort(torch.cat([torch.arange(case["requests"], device="cuda"),
                                        torch.randint(case["requests"], (T - case["requests"],), generator=g, device="cuda")])).values
        chosen = torch.randint(L, (case["requests"],), generator=g, device="cuda")
        none = torch.rand(case["requests"], generator=g, device="cuda") < 0.125
        none[0] = False
        s["ids"] = torch.where(none, -1, chosen)[request].to(torch.int32)
        # the grouping of the batch's rows is made once a step and serves every layer of the model
        s["groups"] = _grouping(s["ids"].long(), L)
        s["x"], s["y"] = normal(T, K), normal(T, N)
        s["a"] = normal(L, R, K, scale=1.0 / math.sqrt(K))
        s["b"] = normal(L, N, R, scale=0.3)
        s["scales"] = torch.rand(L, generator=g, device="cuda") + 0.5
    return s


def run(state):
    return {"route": _route, "experts": _experts, "adapters": _adapters}[state["case"]["op"]](state)


def _route(s):
    case, logits = s["case"], s["logits"]
    k, E = case["k"], case["experts"]
    if own:
        if case["train"]:
            from llm_reproducibility_b200.tbik.autograd import tree_route_topk
            r = tree_route_topk(logits, k, renormalize=case["renormalize"])
            out = {"dlogits": torch.autograd.grad(r.weights, logits, s["dw"])[0]}
        else:
            from llm_reproducibility_b200.tbik.row_groups import route_topk
            r, out = route_topk(logits, k, renormalize=case["renormalize"]), {}
        return {"weights": r.weights.detach(), "ids": r.ids, "order": r.groups.order, "position": r.groups.position,
                "offsets": r.groups.offsets, **out}
    x = logits.detach().float()
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]  # equal scores: the lowest index first
    top = torch.gather(x, 1, ids)
    over = top if case["renormalize"] else x
    peak = over.amax(1, keepdim=True)
    total = torch.exp(over - peak).sum(1, keepdim=True)
    weights = torch.exp(top - peak) / total
    order, position, offsets = _grouping(ids.flatten(), E)
    out = {"weights": weights, "ids": ids.to(torch.int32), "order": order, "position": position, "offsets": offsets}
    if case["train"]:
        inner = (weights * s["dw"]).sum(1, keepdim=True)
        if case["renormalize"]:
            d = torch.zeros_like(x).scatter_(1, ids, weights * (s["dw"] - inner))
        else:
            d = torch.exp(x - peak) / total * (torch.zeros_like(x).scatter_(1, ids, s["dw"]) - inner)
        out["dlogits"] = d.to(logits.dtype)
    return out


def _experts(s):
    case, x, w, offsets = s["case"], s["x"], s["w"], s["offsets"]
    if own:
        if case["train"]:
            from llm_reproducibility_b200.tbik.autograd import tree_grouped_linear
            y = tree_grouped_linear(x, w, offsets)
            dx, dw = torch.autograd.grad(y, (x, w), s["dy"])
            return {"y": y.detach(), "dx": dx, "dw": dw}
        from llm_reproducibility_b200.tbik.grouped_matmul import grouped_matmul_tp_persistent
        return {"y": grouped_matmul_tp_persistent(x, w, offsets, leaf=case["K"] // 8 if case["tree"] else None)}
    x, w = x.detach(), w.detach()
    M, E, longest = x.shape[0], case["experts"], s["longest"]
    # every group padded to the longest: row r of group e sits in slot e * longest + r
    start = offsets[:-1].long()
    rows = torch.arange(M, device=x.device)
    group = torch.searchsorted(offsets[1:].long(), rows, right=True)
    slot = group * longest + rows - start[group]

    def padded(t):
        return torch.zeros(E * longest, t.shape[1], device=t.device).index_copy_(0, slot, t.float()).view(E, longest, -1)

    wf, xp = w.float(), padded(x)
    out = {"y": torch.bmm(xp, wf.transpose(1, 2)).flatten(0, 1)[slot].to(x.dtype)}
    if case["train"]:
        gp = padded(s["dy"])
        out["dx"] = torch.bmm(gp, wf).flatten(0, 1)[slot].to(x.dtype)
        out["dw"] = torch.bmm(gp.transpose(1, 2), xp).to(w.dtype)
    return out


def _adapters(s):
    x, y, a, b, scales = s["x"], s["y"], s["a"], s["b"], s["scales"]
    if own:
        from llm_reproducibility_b200.tbik.adapters import lora_add
        from llm_reproducibility_b200.tbik.row_groups import RowGroups
        return {"y": lora_add(y, x, a, b, RowGroups(*s["groups"]), scales)}
    L, R = a.shape[0], a.shape[1]
    # every row through every adapter, then only its own is kept
    h = (x.float() @ a.float().flatten(0, 1).t()).view(-1, L, R)
    mine = s["ids"][:, None] == torch.arange(L, device=x.device)[None, :]
    h = torch.where(mine[:, :, None], h * scales[None, :, None], 0.0)
    return {"y": (y.float() + h.flatten(1) @ b.float().transpose(1, 2).flatten(0, 1)).to(y.dtype)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        x = s["logits"].detach().double()
        ids = torch.argsort(-x, dim=1, stable=True)[:, : case["k"]]
        p = torch.softmax(x, 1)
        w = p.gather(1, ids)
        if case["renormalize"]:
            w = w / w.sum(1, keepdim=True)
        out = {"weights": w, "ids": None, "order": None, "position": None, "offsets": None}
        if case["train"]:
            # the Jacobian of a softmax over the set S that it runs over: dx = p * (dp - <p, dp>)
            dp = torch.zeros_like(x).scatter_(1, ids, s["dw"].double())
            q = torch.zeros_like(x).scatter_(1, ids, w) if case["renormalize"] else p
            out["dlogits"] = q * (dp - (q * dp).sum(1, keepdim=True))
        return out
    if case["op"] == "experts":
        x, w, at = s["x"].detach(), s["w"].detach(), s["offsets"].tolist()
        y = torch.zeros(x.shape[0], case["N"], dtype=torch.float64, device=x.device)
        dx, dw = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros(w.shape, dtype=torch.float64, device=x.device)
        for e, (lo, hi) in enumerate(zip(at, at[1:])):
            we, xe = w[e].double(), x[lo:hi].double()
            y[lo:hi] = xe @ we.t()
            if case["train"]:
                ge = s["dy"][lo:hi].double()
                dx[lo:hi], dw[e] = ge @ we, ge.t() @ xe
        return {"y": y, "dx": dx, "dw": dw} if case["train"] else {"y": y}
    y, ids = s["y"].double(), s["ids"].long()
    for i in range(case["adapters"]):
        rows = torch.nonzero(ids == i).flatten()
        y[rows] += float(s["scales"][i]) * (s["x"][rows].double() @ s["a"][i].double().t() @ s["b"][i].double().t())
    return {"y": y}


def work(case):
    T, size = case["tokens"], 4 if case["dtype"] == FP32 else 2
    if case["op"] == "route":
        E, k, passes = case["experts"], case["k"], 2 if case["train"] else 1
        return {"bytes": passes * T * E * size + T * k * (16 + 4 * (passes - 1)) + 4 * (E + 1), "flops": 4 * T * E * passes}
    if case["op"] == "experts":
        M, E, K, N = T * case["k"], case["experts"], case["K"], case["N"]
        used = E * (1.0 - (1.0 - case["k"] / E) ** T)  # experts that have a row
        moved = M * K + used * N * K + M * N
        if case["train"]:
            moved += M * N + M * K + E * N * K  # dy read, dx and dw written
        return {"bytes": 2.0 * moved, "flops": 2.0 * M * N * K * (3 if case["train"] else 1)}
    L, R, K, N = case["adapters"], case["rank"], case["K"], case["N"]
    used = L * (1.0 - (1.0 - 1.0 / L) ** max(1.0, 0.875 * case["requests"]))
    return {"bytes": 2.0 * (T * K + 2 * T * N + used * R * (K + N)), "flops": 2.0 * T * R * (K + N)}
