"""Workloads of the token-choice operators: routing, experts' products over routed tokens, products in 8-bit integers.

``run`` computes a case in its plain form (elementary torch operations in float32) or, where ``own`` is true, through the
package's operators; ``exact`` computes the same from the definitions in float64.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- cases -------------------------------------------------------------------------------------------

def _route(name, tokens, E, k, score, dtype, train, bias=False, groups=1, top_groups=1, group_top=2, renorm=True, scale=1.0):
    return {"name": name, "op": "route", "tokens": tokens, "E": E, "k": k, "score": score, "dtype": dtype, "train": train,
            "bias": bias, "groups": groups, "top_groups": top_groups, "group_top": group_top, "renorm": renorm, "scale": scale}


def _experts(name, tokens, E, k, C, N, dtype, train, skew=0.5, idle=0):
    return {"name": name, "op": "experts", "tokens": tokens, "E": E, "k": k, "C": C, "N": N, "dtype": dtype, "train": train,
            "skew": skew, "idle": idle}


def _int8(name, tokens, E, k, C, N, dtype, skew=0.5, idle=0):
    return {"name": name, "op": "int8", "tokens": tokens, "E": E, "k": k, "C": C, "N": N, "dtype": dtype, "skew": skew, "idle": idle}


def listed():
    return [
        # one decoding step of a small batch: the call's latency
        _route("route-decode", 16, 64, 8, "softmax", "bf16", False),
        # a training step: many experts in groups, chosen with a bias that balances their load
        _route("route-train-groups", 32768, 256, 8, "sigmoid", "f32", True, bias=True, groups=8, top_groups=4, scale=2.5),
        # a ragged batch on a number of experts that is no power of two, weights as the softmax gives them
        _route("route-train-odd", 5003, 60, 6, "softmax", "bf16", True, renorm=False),
        # one new token through one projection of its experts
        _experts("experts-decode", 1, 64, 8, 2048, 512, "bf16", False),
        # training steps at the widths of the larger configurations, experts unevenly used
        _experts("experts-train", 16384, 64, 4, 1024, 256, "bf16", True),
        _experts("experts-train-wide", 32768, 64, 4, 2048, 512, "bf16", True),
        # widths that fit no tile and rows that start anywhere, few experts, some that nobody chose
        _experts("experts-train-odd", 1003, 13, 3, 330, 201, "f16", True, skew=1.0, idle=2),
        # float32 training at the smallest configuration's widths
        _experts("experts-train-f32", 16384, 32, 2, 128, 64, "f32", True),
        # 8-bit serving: a few tokens, a whole prompt, and a plain projection of a long batch and of an odd one
        _int8("int8-decode", 3, 64, 8, 2048, 512, "bf16"),
        _int8("int8-prompt", 16384, 64, 4, 2048, 512, "bf16"),
        _int8("int8-dense", 8192, 1, 1, 4096, 4096, "bf16"),
        _int8("int8-dense-odd", 1001, 1, 1, 1030, 777, "f16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges: sizes over their logarithm, at no more work than the largest listed one."""
    op = rng.choice(("route", "experts", "experts", "int8"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32")) if op != "int8" else rng.choice(("bf16", "f16"))
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        E = groups * _log(rng, 2 if groups > 1 else 8, 256 // groups)
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(12, E // groups * top_groups))
        tokens = _log(rng, 1, 32768)
        case = _route("", tokens, E, k, rng.choice(("softmax", "sigmoid")), dtype, rng.random() < 0.5, rng.random() < 0.5,
                      groups, top_groups, rng.choice((1, 2)), rng.random() < 0.7, rng.choice((1.0, 2.5)))
    else:
        E = 1 if op == "int8" and rng.random() < 0.4 else _log(rng, 4, 128)
        k = 1 if E == 1 else rng.randint(1, min(8, E // 2))
        step = rng.choice((1, 8, 16, 64, 64))
        C, N = (max(step, _log(rng, 64, 2048) // step * step) for _ in range(2))
        tokens = _log(rng, 1, 32768)
        limit = 2 * 32768 * 4 * 2048 * 512 if dtype != "f32" else 2 * 32768 * 1024 * 256
        while 2 * tokens * k * C * N > limit // 2:
            tokens = (tokens + 1) // 2
        idle = rng.choice((0, 0, E // 4)) if E - E // 4 >= k else 0
        make = _experts if op == "experts" else _int8
        kinds = {"train": rng.random() < 0.6} if op == "experts" else {}
        case = make("", tokens, E, k, C, N, dtype, skew=rng.choice((0.0, 0.5, 1.5)), idle=idle, **kinds)
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------------------------------

def _keys64(case, logits, bias):
    x = logits.double()
    if case["score"] == "softmax":
        e = (x - x.amax(-1, keepdim=True)).exp()
        s = e / e.sum(-1, keepdim=True)
    else:
        s = 1 / (1 + (-x).exp())
    return s, s + bias.double() if bias is not None else s


def _kept64(case, key):
    """key with the experts of dropped groups at -inf, and the values of the groups."""
    G = case["groups"]
    if G == 1:
        return key, None
    per = key.shape[1] // G
    best = key.view(-1, G, per).sort(-1, descending=True).values
    value = best[..., 0] + best[..., 1] if case["group_top"] == 2 and per > 1 else best[..., 0]
    order = value.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
    keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, order, True)
    return key.masked_fill(~keep.repeat_interleave(per, 1), -math.inf), value


def _undecided(case, logits, bias):
    """Rows whose choice hangs on the last bits of a float32 key, where no expert is the right one (equal logits are fine
    without a bias: they are equal in every precision)."""
    _, key = _keys64(case, logits, bias)
    kept, value = _kept64(case, key)

    def close(v, n):
        top = v.sort(-1, descending=True).values[:, :n + 1]
        gap = top[:, :-1] - top[:, 1:]
        same = gap == 0 if bias is None else torch.zeros_like(gap, dtype=torch.bool)
        return ((gap < 2e-6 * top[:, :-1].abs().clamp(min=1e-30)) & ~same).any(-1)

    bad = close(kept, case["k"])
    return bad | close(value, case["top_groups"]) if value is not None else bad


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, tokens, E, k = _DTYPES[case["dtype"]], case["tokens"], case["E"], case["k"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["op"] == "route":
        bias = 0.1 * randn(E) if case["bias"] else None
        popular = 0.5 * randn(E)
        logits = (1.5 * randn(tokens, E) + popular).to(dtype)
        for attempt in range(40):
            bad = _undecided(case, logits, bias).nonzero().flatten()
            if bad.numel() == 0:
                break
            logits[bad] = (1.5 * randn(bad.numel(), E) + popular).to(dtype)
        return {"case": case, "logits": logits, "bias": bias, "grad": randn(tokens, k) if case["train"] else None}
    C, N = case["C"], case["N"]
    popular = case["skew"] * randn(E)
    if case["idle"]:
        popular[:case["idle"]] = -1e4
    scores = randn(tokens, E) + popular
    top = scores.topk(k, -1)
    state = {"case": case, "X": randn(tokens, C).to(dtype), "experts": top.indices.to(torch.int32),
             "weights": torch.softmax(top.values, -1).to(dtype)}     # in the layer's type, as its products take them
    W = randn(E, C, N) / math.sqrt(C)
    if case["op"] == "experts":
        state["W"] = W.to(dtype)
        state["grad"] = randn(tokens, N).to(dtype) if case["train"] else None
        return state
    # 8-bit weights as a serving program keeps them: one scale a channel, a channel's elements together, rows of whole 16 bytes
    W = W.transpose(1, 2)
    scale = W.abs().amax(-1) / 127
    rows = torch.zeros(E, N, (C + 15) // 16 * 16, device="cuda", dtype=torch.int8)
    rows[..., :C] = (W / scale.unsqueeze(-1)).round()
    state.update(Wq=rows[..., :C], w_scale=scale)
    return state


# ---- the package's operators -------------------------------------------------------------------------

def _run_own(state):
    from expertscattergather_b200 import ops
    case = state["case"]
    if case["op"] == "route":
        opts = {"score": case["score"], "renormalize": case["renorm"], "scale": case["scale"]}
        weights, experts = ops.route_tokens(state["logits"], case["k"], state["bias"], groups=case["groups"],
                                            top_groups=case["top_groups"], group_top=case["group_top"], **opts)
        if not case["train"]:
            return weights, experts
        return weights, experts, ops.route_tokens_backward(state["grad"], state["logits"], experts, **opts)
    X, w = state["X"], state["weights"]
    if case["op"] == "int8":
        q, s = ops.quantize_rows(X)
        if case["E"] == 1:
            return (ops.matmul_int8(q, s, state["Wq"][0], state["w_scale"][0], out_dtype=X.dtype),)
        plan = ops.plan_experts(state["experts"], case["E"])
        Y = ops.expert_matmul_int8(q, s, state["Wq"], state["w_scale"], plan, out_dtype=X.dtype)
        return (ops.combine(Y, w, plan),)
    plan = ops.plan_experts(state["experts"], case["E"])
    Y = ops.expert_matmul(X, state["W"], plan)
    out = ops.combine(Y, w, plan)
    if not case["train"]:
        return (out,)
    dY, dw = ops.combine_backward(state["grad"], Y, w, plan)
    dX = ops.combine(ops.expert_matmul(dY, state["W"], plan, rows="sorted", w_layout="nc"), None, plan)
    return out, dX, ops.expert_dweight(X, dY, plan), dw


# ---- the plain form ----------------------------------------------------------------------------------

def _route_plain(state):
    case, x = state["case"], state["logits"].float()
    if case["score"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        s = e / e.sum(-1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-x))
    key = s + state["bias"] if state["bias"] is not None else s
    G, (tokens, E) = case["groups"], x.shape
    if G > 1:
        best = key.view(tokens, G, E // G).sort(-1, descending=True).values
        value = best[..., 0] + best[..., 1] if case["group_top"] == 2 and E // G > 1 else best[..., 0]
        order = value.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, order, True)
        key = key.masked_fill(~keep.repeat_interleave(E // G, 1), -math.inf)
    experts = key.sort(dim=-1, descending=True, stable=True).indices[:, :case["k"]]
    chosen = s.gather(1, experts)
    total = chosen.sum(-1, keepdim=True)
    share = chosen / total if case["renorm"] else chosen
    weights = share * case["scale"]
    if not case["train"]:
        return weights, experts.to(torch.int32)
    g = state["grad"] * case["scale"]
    ds = (g - (g * share).sum(-1, keepdim=True)) / total if case["renorm"] else g
    full = torch.zeros_like(s).scatter_(1, experts, ds)
    if case["score"] == "softmax":
        dx = s * (full - (full * s).sum(-1, keepdim=True))
    else:
        dx = full * s * (1 - s)
    return weights, experts.to(torch.int32), dx.to(state["logits"].dtype)


def _segments(experts, E):
    """Slots (token * k + j) sorted by expert, and where each expert's begin."""
    flat = experts.flatten().long()
    order = flat.sort(stable=True).indices
    counts = torch.bincount(flat, minlength=E).tolist()
    return order, counts


def _experts_plain(state):
    case = state["case"]
    X, w, W = state["X"].float(), state["weights"].float(), state["W"]
    k, E, dtype = case["k"], case["E"], state["X"].dtype
    order, counts = _segments(state["experts"], E)
    token = order // k
    Xs = X[token]
    Y = torch.empty(order.numel(), case["N"], device=X.device)
    at = 0
    for e, n in enumerate(counts):
        if n:
            Y[at:at + n] = Xs[at:at + n] @ W[e].float()
            at += n
    Yslot = torch.empty_like(Y)
    Yslot[order] = Y
    out = (Yslot.view(-1, k, case["N"]) * w.unsqueeze(-1)).sum(1)
    if not case["train"]:
        return (out.to(dtype),)
    G = state["grad"].float()
    dw = (Yslot.view(-1, k, case["N"]) * G.unsqueeze(1)).sum(-1)
    dY = G[token] * w.flatten()[order].unsqueeze(-1)
    dXs = torch.empty_like(Xs)
    dW = torch.zeros(E, case["C"], case["N"], device=X.device)
    at = 0
    for e, n in enumerate(counts):
        if n:
            part = dY[at:at + n]
            dXs[at:at + n] = part @ W[e].float().t()
            dW[e] = Xs[at:at + n].t() @ part
            at += n
    dXslot = torch.empty_like(dXs)
    dXslot[order] = dXs
    dX = dXslot.view(-1, k, case["C"]).sum(1)
    return out.to(dtype), dX.to(dtype), dW.to(dtype), dw.to(dtype)


def _int8_plain(state):
    case, X = state["case"], state["X"].float()
    s = X.abs().amax(-1, keepdim=True) / 127
    q = (X / s).round()
    Wq, ws = state["Wq"], state["w_scale"]
    if case["E"] == 1:
        return ((q @ Wq[0].float().t() * s * ws[0]).to(state["X"].dtype),)
    k = case["k"]
    order, counts = _segments(state["experts"], case["E"])
    token = order // k
    qs, ss = q[token], s[token]
    Y = torch.empty(order.numel(), case["N"], device=X.device)
    at = 0
    for e, n in enumerate(counts):
        if n:
            Y[at:at + n] = qs[at:at + n] @ Wq[e].float().t() * ss[at:at + n] * ws[e]
            at += n
    Yslot = torch.empty_like(Y)
    Yslot[order] = Y
    out = (Yslot.view(-1, k, case["N"]) * state["weights"].float().unsqueeze(-1)).sum(1)
    return (out.to(state["X"].dtype),)


def run(state):
    if own:
        return _run_own(state)
    return {"route": _route_plain, "experts": _experts_plain, "int8": _int8_plain}[state["case"]["op"]](state)


# ---- the work, and the definitions in float64 --------------------------------------------------------

def work(case):
    tokens, E, k = case["tokens"], case["E"], case["k"]
    es = torch.empty((), dtype=_DTYPES[case["dtype"]]).element_size()
    slots = tokens * k
    if case["op"] == "route":     # the ids and, in float32, the weights and their gradient
        nbytes, flops = tokens * E * es + 8 * slots, 8 * tokens * E
        if case["train"]:
            nbytes, flops = nbytes + tokens * E * es + 4 * slots, flops + 8 * tokens * E
        return {"bytes": nbytes, "flops": flops}
    C, N = case["C"], case["N"]
    used = min(E - case["idle"], slots)
    if case["op"] == "int8":
        routed = 0 if E == 1 else (4 + es) * slots
        return {"bytes": tokens * (C + N) * es + used * (C + 4) * N + routed, "flops": 2 * slots * C * N}
    nbytes, flops = tokens * (C + N) * es + used * C * N * es + (4 + es) * slots, 2 * slots * C * N
    if case["train"]:
        nbytes += tokens * (C + N) * es + E * C * N * es + es * slots
        flops *= 3
    return {"bytes": nbytes, "flops": flops}


def _exact_route(case, state):
    s, key = _keys64(case, state["logits"], state["bias"])
    kept, _ = _kept64(case, key)
    experts = kept.sort(dim=-1, descending=True, stable=True).indices[:, :case["k"]]
    p = torch.gather(s, 1, experts)
    S = p.sum(-1, keepdim=True) if case["renorm"] else torch.ones_like(p[:, :1])
    weights = case["scale"] * p / S
    if not case["train"]:
        return weights, experts.to(torch.int32)
    g = state["grad"].double()
    back = (g * p).sum(-1, keepdim=True) / S if case["renorm"] else torch.zeros_like(S)
    dp = torch.zeros_like(s).scatter_(1, experts, case["scale"] * (g - back) / S)
    if case["score"] == "softmax":
        dx = s * dp - s * (s * dp).sum(-1, keepdim=True)
    else:
        dx = s * (1 - s) * dp
    return weights, experts.to(torch.int32), dx


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, state)
    tokens, k, C, N, E = case["tokens"], case["k"], case["C"], case["N"], case["E"]
    if 2 * tokens * k * C * N > 3e12:
        return None
    X, w, ids = state["X"].double(), state["weights"].double(), state["experts"].long()
    if case["op"] == "int8":
        amax = X.abs().amax(-1, keepdim=True)
        X = (127 * X / amax).round() * amax / 127
        if E == 1:
            return (X @ (state["Wq"][0].double() * state["w_scale"][0].double().unsqueeze(-1)).t(),)
    out = torch.zeros(tokens, N, device="cuda", dtype=torch.float64)
    train = case.get("train", False)
    if train:
        G = state["grad"].double()
        dX = torch.zeros(tokens, C, device="cuda", dtype=torch.float64)
        dW = torch.zeros(E, C, N, device="cuda", dtype=torch.float64)
        dw = torch.zeros(tokens, k, device="cuda", dtype=torch.float64)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        if case["op"] == "int8":
            We = (state["Wq"][e].double() * state["w_scale"][e].double().unsqueeze(-1)).t()
        else:
            We = state["W"][e].double()
        we = w[t, j].unsqueeze(-1)
        y = X[t] @ We
        out.index_put_((t,), we * y, accumulate=True)
        if train:
            dw[t, j] = (y * G[t]).sum(-1)
            dX.index_put_((t,), (we * G[t]) @ We.t(), accumulate=True)
            dW[e] = X[t].t() @ (we * G[t])
    return (out, dX, dW, dw) if train else (out,)
