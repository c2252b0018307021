"""The workloads of the dense-product, routing and log-probability operators.

`run` is one pass of an operator as a serving program calls it: in its plain
form (elementary torch operations in 32 bits, 64 where a border has to be
decided), or, where `own` is true, through firewing_b200.  `exact` computes
the same from the definitions in 64 bits.
"""
import math

import torch

own = False

NEG_INF = float("-inf")
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")


# ---- cases ---------------------------------------------------------------------


def linear_case(tokens, rows, cols, dtype="bf16", out="same", activation="none", bias=False, residual=False, **more):
    return dict(op="linear", tokens=tokens, rows=rows, cols=cols, dtype=dtype, out=out, activation=activation,
                bias=bias, residual=residual, **more)


def route_case(tokens, experts, top_k, dtype="f32", scoring="sigmoid", bias=False, groups=1, top_groups=1,
               group_top=1, renormalize=True, scale=1.0, counts=False, masked=0.0, **more):
    return dict(op="route", tokens=tokens, experts=experts, top_k=top_k, dtype=dtype, scoring=scoring, bias=bias,
                groups=groups, top_groups=top_groups, group_top=group_top, renormalize=renormalize, scale=scale,
                counts=counts, masked=masked, **more)


def logprobs_case(tokens, vocab, dtype="bf16", targets=1, top_k=0, temperature=1.0, masked=0.0, **more):
    return dict(op="logprobs", tokens=tokens, vocab=vocab, dtype=dtype, targets=targets, top_k=top_k,
                temperature=temperature, masked=masked, **more)


def listed():
    return [
        # the gate of one decoded token: 512 experts, hidden 2048, logits kept in 32 bits
        linear_case(1, 512, 2048, out="f32", name="linear gate 1 token"),
        # a decode batch through a dense layer: the weights' bytes are the work
        linear_case(64, 8192, 2048, activation="silu", bias=True, name="linear up 64 tokens"),
        # a pruned layer: no size is a multiple of anything, rows start at odd addresses
        linear_case(333, 1001, 1999, dtype="f16", activation="gelu", bias=True, residual=True,
                    name="linear ragged 333 tokens"),
        # a prompt through a dense layer: the products are the work
        linear_case(8192, 8192, 2048, activation="gelu_tanh", bias=True, name="linear up 8192 tokens"),
        # the same layer's way back onto the residual stream
        linear_case(4096, 2048, 8192, residual=True, name="linear down 4096 tokens"),
        # one decoded token's routing: latency alone
        route_case(1, 512, 10, dtype="bf16", bias=True, groups=8, top_groups=4, group_top=2,
                   name="route 1 token"),
        # a small ragged batch, softmax scores, limited to groups, some experts out of service
        route_case(61, 160, 6, scoring="softmax", groups=8, top_groups=3, group_top=1, renormalize=False, scale=16.0,
                   masked=0.1, name="route softmax 61 tokens"),
        # a prompt's routing with the balance bias and the experts' loads
        route_case(8192, 512, 10, bias=True, groups=8, top_groups=4, group_top=2, scale=2.5, counts=True,
                   name="route 8192 tokens"),
        # one answered token with its alternatives
        logprobs_case(1, 131072, top_k=20, name="logprobs 1 token"),
        # a speculative verification batch, 32-bit logits
        logprobs_case(64, 131072, dtype="f32", top_k=8, name="logprobs 64 tokens"),
        # choices scored under a grammar's mask, odd vocabulary
        logprobs_case(37, 50021, dtype="f16", targets=5, top_k=5, temperature=0.7, masked=0.5,
                      name="logprobs masked 37 tokens"),
        # a prompt scored: every position's token and five alternatives
        logprobs_case(2048, 131072, top_k=5, name="logprobs 2048 tokens"),
    ]


def spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "route", "logprobs"))
    if op == "linear":
        while True:
            t, n, k = spread(rng, 1, 8192), spread(rng, 1, 16384), spread(rng, 1, 8192)
            if rng.random() < 0.6:  # layers are mostly multiples of eight
                n, k = -(-n // 8) * 8, -(-k // 8) * 8
            if t * n * k <= 8192 * 8192 * 2048 and t * n <= 8192 * 8192:
                break
        return linear_case(t, n, k, dtype=rng.choice(("bf16", "f16")), out=rng.choice(("same", "same", "f32")),
                           activation=rng.choice(ACTIVATIONS), bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8, 16))
        per = spread(rng, max(2, 8 // groups), 1024 // groups)
        top_groups = rng.randint(1, groups)
        top_k = min(rng.randint(1, 32), top_groups * per)
        return route_case(spread(rng, 1, 8192), groups * per, top_k, dtype=rng.choice(("bf16", "f16", "f32")),
                          scoring=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.6, groups=groups,
                          top_groups=top_groups, group_top=rng.choice((1, 2)), renormalize=rng.random() < 0.7,
                          scale=rng.choice((1.0, 2.5)), counts=rng.random() < 0.5,
                          masked=rng.choice((0.0, 0.0, 0.2)))
    while True:
        t, v = spread(rng, 1, 4096), spread(rng, 2, 262144)
        if t * v <= 1024 * 131072:
            break
    return logprobs_case(t, v, dtype=rng.choice(("bf16", "f16", "f32")), targets=rng.randint(1, 8),
                         top_k=min(v, rng.randint(0, 32)), temperature=rng.choice((1.0, 1.0, 0.7, 1.3)),
                         masked=rng.choice((0.0, 0.0, 0.5)))


def work(case):
    c = case
    if c["op"] == "linear":
        t, n, k, s = c["tokens"], c["rows"], c["cols"], SIZE[c["dtype"]]
        o = 4 if c["out"] == "f32" else s
        return {"bytes": (t * k + n * k) * s + t * n * o + (n * s if c["bias"] else 0)
                + (t * n * s if c["residual"] else 0), "flops": 2 * t * n * k}
    if c["op"] == "route":
        t, e, k = c["tokens"], c["experts"], c["top_k"]
        return {"bytes": t * e * SIZE[c["dtype"]] + t * k * 8 + e * (4 * c["bias"] + 4 * c["counts"]),
                "flops": 6 * t * e}
    t, v = c["tokens"], c["vocab"]
    return {"bytes": t * v * SIZE[c["dtype"]] + t * (c["targets"] * 8 + 4 + c["top_k"] * 8), "flops": 6 * t * v}


# ---- what a program has in hand --------------------------------------------------


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    def below(p, *shape):
        return torch.rand(*shape, generator=g, device="cuda") < p

    s = dict(case=dict(c))
    dt = DTYPES[c["dtype"]]
    if c["op"] == "linear":
        t, n, k = c["tokens"], c["rows"], c["cols"]
        s["x"] = normal(t, k, dtype=dt)
        s["w"] = normal(n, k, std=1.0 / math.sqrt(k), dtype=dt)
        s["bias"] = normal(n, std=0.5, dtype=dt) if c["bias"] else None
        s["residual"] = normal(t, n, dtype=dt) if c["residual"] else None
        s["y"] = torch.empty(t, n, device="cuda", dtype=torch.float32 if c["out"] == "f32" else dt)
    elif c["op"] == "route":
        t, e, k = c["tokens"], c["experts"], c["top_k"]
        z = normal(t, e, std=1.5) + normal(e, std=0.5)  # some experts are liked by all
        if c["masked"]:
            z = z.masked_fill(below(c["masked"], e), NEG_INF)  # experts out of service
            z[t // 2:][: 1 if t > 1 else 0] = NEG_INF  # a padded row of the batch
        s["logits"] = z.to(dt)
        s["bias"] = normal(e, std=0.1) if c["bias"] else None
        s["indices"] = torch.empty(t, k, device="cuda", dtype=torch.int32)
        s["weights"] = torch.empty(t, k, device="cuda", dtype=torch.float32)
        s["counts"] = torch.empty(e, device="cuda", dtype=torch.int32) if c["counts"] else None
    else:
        t, v, k = c["tokens"], c["vocab"], c["top_k"]
        z = normal(t, v, std=2.5).to(dt)
        best = torch.randint(0, v, (t, 1), generator=g, device="cuda")
        z.scatter_add_(1, best, torch.full((t, 1), 9.0, device="cuda", dtype=dt))  # a head is sure of a token
        if c["masked"]:
            z.masked_fill_(below(c["masked"], v), NEG_INF)  # a grammar allows the rest
        s["logits"] = z
        s["targets"] = torch.randint(0, v, (t, c["targets"]), generator=g, device="cuda", dtype=torch.int32)
        s["targets"][:, :1] = best.to(torch.int32)
        s["logprobs"] = torch.empty(t, c["targets"], device="cuda")
        s["entropy"] = torch.empty(t, device="cuda")
        s["top_idx"] = torch.empty(t, k, device="cuda", dtype=torch.int32) if k else None
        s["top_logprobs"] = torch.empty(t, k, device="cuda") if k else None
    return s


# ---- one pass --------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": own_linear, "route": own_route, "logprobs": own_logprobs}[op](state)
    return {"linear": plain_linear, "route": plain_route, "logprobs": plain_logprobs}[op](state)


def own_linear(s):
    import firewing_b200 as fw

    fw.linear_epilogue(s["w"], s["x"], s["y"], bias=s["bias"], activation=s["case"]["activation"],
                       residual=s["residual"], stream=torch.cuda.current_stream())
    return s["y"]


def own_route(s):
    import firewing_b200 as fw

    c = s["case"]
    fw.route_scores(s["logits"], s["indices"], s["weights"], scoring=c["scoring"], bias=s["bias"],
                    groups=c["groups"], top_groups=c["top_groups"], group_top=c["group_top"],
                    renormalize=c["renormalize"], scale=c["scale"], counts=s["counts"],
                    stream=torch.cuda.current_stream())
    return {"indices": s["indices"], "weights": s["weights"], "counts": s["counts"]}


def own_logprobs(s):
    import firewing_b200 as fw

    fw.token_logprobs(s["logits"], s["targets"], s["logprobs"], entropy=s["entropy"], top_idx=s["top_idx"],
                      top_logprobs=s["top_logprobs"], temperature=s["case"]["temperature"],
                      stream=torch.cuda.current_stream())
    return {"logprobs": s["logprobs"], "entropy": s["entropy"], "top_idx": s["top_idx"],
            "top_logprobs": s["top_logprobs"]}


def plain_linear(s):
    y = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    act = s["case"]["activation"]
    if act == "relu":
        y = torch.clamp(y, min=0.0)
    elif act == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    elif act == "gelu_tanh":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    elif act == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif act == "sigmoid":
        y = 1.0 / (1.0 + torch.exp(-y))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["y"].dtype)


def plain_route(s):
    c = s["case"]
    t, e, k = c["tokens"], c["experts"], c["top_k"]
    z = s["logits"].double()  # the order of two near scores is decided in 64 bits
    gone = torch.isneginf(z)
    if c["scoring"] == "softmax":
        top = z.amax(1, keepdim=True)
        p = torch.exp(z - torch.where(torch.isneginf(top), 0.0, top))
        score = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        score = 1.0 / (1.0 + torch.exp(-z))
    key = (score + s["bias"].double() if s["bias"] is not None else score).masked_fill(gone, NEG_INF)
    order = key if s["bias"] is not None else z  # without a bias the logits themselves say the order
    if c["groups"] > 1:
        inside = torch.sort(key.view(t, c["groups"], -1), dim=2, descending=True).values[:, :, : c["group_top"]]
        group = torch.where(torch.isneginf(inside), 0.0, inside).sum(2)
        group = group.masked_fill(torch.isneginf(inside[:, :, 0]), NEG_INF)
        best = torch.sort(group, dim=1, descending=True, stable=True).indices[:, : c["top_groups"]]
        kept = torch.zeros(t, c["groups"], dtype=torch.bool, device=z.device).scatter_(1, best, True)
        order = order.view(t, c["groups"], -1).masked_fill(~kept.unsqueeze(2), NEG_INF).view(t, e)
    value, index = torch.sort(order, dim=1, descending=True, stable=True)
    none = torch.isneginf(value[:, :k])
    index = index[:, :k]
    weight = torch.gather(score, 1, index).masked_fill(none, 0.0)
    if c["renormalize"]:
        total = weight.sum(1, keepdim=True)
        weight = weight / torch.where(total > 0, total, 1.0)
    out = {"indices": index.masked_fill(none, -1).int(), "weights": (weight * c["scale"]).float(), "counts": None}
    if c["counts"]:
        out["counts"] = torch.bincount(index[~none], minlength=e).int()
    return out


def plain_logprobs(s):
    c = s["case"]
    z = s["logits"].float()
    if c["temperature"] != 1.0:
        z = z / c["temperature"]
    top = z.amax(1, keepdim=True)
    z = z - torch.where(torch.isneginf(top), 0.0, top)
    p = torch.exp(z)
    total = p.sum(1, keepdim=True)
    log_total = torch.log(total)
    out = {"logprobs": torch.gather(z, 1, s["targets"].long()) - log_total, "top_idx": None, "top_logprobs": None}
    out["entropy"] = (log_total - torch.where(p > 0, p * z, 0.0).sum(1, keepdim=True) / total).squeeze(1)
    if c["top_k"]:
        # the k best and every tie of the last one, then the lowest indices among equals
        wide = s["logits"].float()
        last = torch.topk(wide, c["top_k"], dim=1).values[:, -1:]
        lead = torch.where(wide > last, wide, NEG_INF)
        value, index = torch.topk(lead, c["top_k"], dim=1)
        ties = torch.arange(c["vocab"], 0, -1, device=z.device, dtype=torch.int32) * (wide == last)
        tie_index = torch.topk(ties, c["top_k"], dim=1).indices
        number = torch.arange(c["top_k"], device=z.device)
        over = (wide > last).sum(1, keepdim=True)
        pick = torch.gather(tie_index, 1, (number - over).clamp(min=0))
        index = torch.where(number < over, index, pick)
        value = torch.gather(wide, 1, index)
        by_index = torch.sort(index, dim=1)
        by_value = torch.sort(torch.gather(value, 1, by_index.indices), dim=1, descending=True, stable=True)
        index = torch.gather(by_index.values, 1, by_value.indices)
        none = torch.isneginf(by_value.values)
        out["top_logprobs"] = (torch.gather(z, 1, index) - log_total).masked_fill(none, NEG_INF)
        out["top_idx"] = index.masked_fill(none, -1).int()
    return out


# ---- the definitions in 64 bits -----------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": exact_linear, "route": exact_route, "logprobs": exact_logprobs}[case["op"]](case, s)


def exact_linear(c, s):
    from torch.nn import functional as F

    v = F.linear(s["x"].double(), s["w"].double(), s["bias"].double() if c["bias"] else None)
    f = {"none": lambda a: a, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda a: F.gelu(a, approximate="tanh"),
         "silu": F.silu, "sigmoid": torch.sigmoid}[c["activation"]]
    v = f(v)
    return v.add_(s["residual"].double()) if c["residual"] else v


def exact_route(c, s):
    import numpy as np

    if c["tokens"] * c["experts"] > 1 << 22:  # one row at a time on the host: seconds
        return None
    z = s["logits"].double().cpu().numpy()
    bias = s["bias"].double().cpu().numpy() if c["bias"] else np.zeros(c["experts"])
    size = c["experts"] // c["groups"]
    indices = np.full((c["tokens"], c["top_k"]), -1, np.int32)
    weights = np.zeros((c["tokens"], c["top_k"]))
    counts = np.zeros(c["experts"], np.int32)
    for t, row in enumerate(z):
        live = [e for e in range(c["experts"]) if row[e] != NEG_INF]
        if not live:
            continue
        if c["scoring"] == "softmax":
            high = max(row[e] for e in live)
            mass = math.fsum(math.exp(row[e] - high) for e in live)
            score = {e: math.exp(row[e] - high) / mass for e in live}
        else:
            score = {e: 1.0 / (1.0 + math.exp(-row[e])) for e in live}
        if c["groups"] > 1:
            of = {}
            for e in live:
                of.setdefault(e // size, []).append(score[e] + bias[e])
            rank = sorted(of, key=lambda g: (-sum(sorted(of[g], reverse=True)[: c["group_top"]]), g))
            allowed = set(rank[: c["top_groups"]])
            live = [e for e in live if e // size in allowed]
        live.sort(key=lambda e: (-(score[e] + bias[e]) if c["bias"] else -row[e], e))
        chosen = live[: c["top_k"]]
        total = math.fsum(score[e] for e in chosen) if c["renormalize"] else 1.0
        for n, e in enumerate(chosen):
            indices[t, n], weights[t, n] = e, score[e] / total * c["scale"] if total > 0 else 0.0
            counts[e] += 1
    return {"indices": indices, "weights": weights, "counts": counts if c["counts"] else None}


def exact_logprobs(c, s):
    lp, entropy, tops = [], [], []
    for rows, ids in zip(s["logits"].split(64), s["targets"].split(64)):
        z = rows.double() / c["temperature"]
        lse = torch.logsumexp(z, 1, keepdim=True)
        q = z - lse
        lp.append(q.gather(1, ids.long()))
        entropy.append(-torch.xlogy(q.exp(), q.exp()).sum(1))
        if c["top_k"]:
            tops.append(torch.sort(q, dim=1, descending=True).values[:, : c["top_k"]])
    return {"logprobs": torch.cat(lp), "entropy": torch.cat(entropy), "top_idx": None,
            "top_logprobs": torch.cat(tops) if c["top_k"] else None}
