"""Workloads of the operators in 4 bits and of the whole routed layer for a few tokens.

Rows in 4 bits are blocks of 32 values of sign, two exponent bits and one mantissa bit (0, .5, 1, 1.5, 2, 3, 4, 6) with a power of two for
each block, the smallest one whose seven-fold the block's largest magnitude does not pass.  ``run`` computes a case in its plain form
(elementary torch operations in float32) or, where ``own`` is true, through the package's operators; ``exact`` computes the same from the
definitions in float64.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- cases -------------------------------------------------------------------------------------------

def _rows(name, tokens, C, dtype, silu=False):
    return {"name": name, "op": "rows", "tokens": tokens, "C": C, "dtype": dtype, "silu": silu}


def _product(name, tokens, E, k, C, N, dtype, skew=0.5, idle=0):
    return {"name": name, "op": "product", "tokens": tokens, "E": E, "k": k, "C": C, "N": N, "dtype": dtype, "skew": skew, "idle": idle}


def _layer(name, tokens, E, k, C, N, dtype, skew=0.5, idle=0):
    return {"name": name, "op": "layer", "tokens": tokens, "E": E, "k": k, "C": C, "N": N, "dtype": dtype, "skew": skew, "idle": idle}


def _few(name, tokens, E, k, C, N, dtype, fp4=False, score="softmax", bias=False, groups=1, top_groups=1, renorm=True, scale=1.0):
    return {"name": name, "op": "few", "tokens": tokens, "E": E, "k": k, "C": C, "N": N, "dtype": dtype, "fp4": fp4, "score": score,
            "bias": bias, "groups": groups, "top_groups": top_groups, "renorm": renorm, "scale": scale}


def listed():
    return [
        # the rows of a prompt into 4 bits, as a projection's input
        _rows("fp4-rows-prompt", 16384, 2048, "bf16"),
        # an activation's output of a ragged batch, rows of no whole number of blocks
        _rows("fp4-rows-odd", 1003, 1030, "f16", silu=True),
        # a plain projection of a long batch in 4 bits, and of an odd one
        _product("fp4-dense", 8192, 1, 1, 4096, 4096, "bf16"),
        _product("fp4-dense-odd", 1001, 1, 1, 1030, 777, "f16"),
        # a prompt through one projection of its experts, some of them idle
        _product("fp4-experts-prompt", 16384, 64, 4, 2048, 512, "bf16", idle=4),
        # a few new tokens through one projection of their experts
        _product("fp4-experts-decode", 3, 64, 8, 2048, 512, "bf16"),
        # a prompt through both projections of a layer, the rows between them in 4 bits too
        _layer("fp4-layer-prompt", 16384, 64, 4, 2048, 512, "bf16"),
        # one new token through a whole layer, router and all: the call's latency and the weights' bytes
        _few("few-one", 1, 64, 8, 2048, 512, "bf16"),
        # a small batch that decodes, experts shared by its tokens
        _few("few-batch", 16, 64, 4, 1024, 256, "bf16"),
        # widths that fit no vector, few experts, scores of a sigmoid with a bias that balances the load
        _few("few-odd", 5, 13, 3, 330, 201, "f16", score="sigmoid", bias=True, scale=2.5),
        # float32 at the smallest configuration's widths
        _few("few-f32", 2, 32, 2, 128, 64, "f32", renorm=False),
        # a small batch on weights in 4 bits, experts in groups
        _few("few-fp4", 8, 64, 8, 2048, 512, "bf16", fp4=True, score="sigmoid", bias=True, groups=8, top_groups=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges: sizes over their logarithm, at no more work than the largest listed one."""
    op = rng.choice(("rows", "product", "product", "layer", "few", "few", "few"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    step = rng.choice((1, 8, 32, 64, 64))
    C, N = (max(step, _log(rng, 64, 2048) // step * step) for _ in range(2))
    if op == "rows":
        case = _rows("", _log(rng, 1, 16384), C, rng.choice((dtype, "f32")), rng.random() < 0.3)
    elif op == "few":
        groups = rng.choice((1, 1, 1, 2, 4))
        E = groups * _log(rng, 4, 128 // groups)
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(8, E // groups * top_groups))
        tokens = _log(rng, 1, 32)
        fp4 = rng.random() < 0.4                               # (in float32 a rounding of 4 bits that falls the other way would decide)
        case = _few("", tokens, E, k, C, N, dtype if fp4 else rng.choice((dtype, dtype, "f32")), fp4, rng.choice(("softmax", "sigmoid")),
                    rng.random() < 0.5, groups, top_groups, rng.random() < 0.7, rng.choice((1.0, 2.5)))
    else:
        E = 1 if op == "product" and rng.random() < 0.4 else _log(rng, 4, 128)
        k = 1 if E == 1 else rng.randint(1, min(8, E // 2))
        tokens = _log(rng, 1, 16384)
        while tokens * k * C * N > 16384 * 4 * 2048 * 512:
            tokens = (tokens + 1) // 2
        idle = rng.choice((0, 0, E // 4)) if E - E // 4 >= k else 0
        make = _product if op == "product" else _layer
        case = make("", tokens, E, k, C, N, dtype, rng.choice((0.0, 0.5, 1.5)), idle)
    del case["name"]
    return case


# ---- rows in 4 bits, in float32 ----------------------------------------------------------------------

def _blocks(x):
    """[..., C] -> [..., blocks, 32], zeros behind the row's end."""
    C = x.shape[-1]
    n = (C + 31) // 32
    if n * 32 != C:
        x = torch.cat((x, x.new_zeros(*x.shape[:-1], n * 32 - C)), -1)
    return x.unflatten(-1, (n, 32))


def _power(byte):
    """2 ** (byte - 127) of bytes below 255, as float32."""
    byte = byte.to(torch.int32)
    return torch.where(byte > 0, byte << 23, torch.full_like(byte, 1 << 22)).view(torch.float32)


def _rounded(x):
    """Blocks [..., 32] in float32 -> the values of their 4 bits (not scaled) and the scale's byte."""
    top = x.abs().amax(-1, keepdim=True)
    byte = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 2).clamp(min=0)
    y = x / _power(byte)
    m = y.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    return ((m / step).round() * step).clamp(max=6).copysign(y), byte


def _values(x):
    """Rows [..., C] in float32 -> what their 4 bits stand for."""
    v, byte = _rounded(_blocks(x))
    return (v * _power(byte)).flatten(-2)[..., :x.shape[-1]]


def _pack(x):
    """Rows [..., C] -> 4 bits [..., ceil(C / 2)], two to a byte, the first in the lower half, and bytes of the scales [..., blocks]: rows
    a multiple of 16 bytes apart, as a serving program keeps them."""
    v, byte = _rounded(_blocks(x))
    m = v.abs()
    code = torch.where(m < 2, 2 * m, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    code = code.flatten(-2)
    packed, byte = code[..., ::2] | (code[..., 1::2] << 4), byte.squeeze(-1).to(torch.uint8)
    scale = byte.new_zeros(*byte.shape[:-1], (byte.shape[-1] + 15) // 16 * 16)
    scale[..., :byte.shape[-1]] = byte
    return packed[..., :(x.shape[-1] + 1) // 2], scale[..., :byte.shape[-1]]


def _unpacked(packed, byte, C):
    """The values of packed rows [..., C], in float32."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=packed.device)
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)[..., :C]
    return table[code.int()] * _power(byte).repeat_interleave(32, -1)[..., :C]


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
    """key with the experts of dropped groups at -inf, and the values of the groups (their two best keys)."""
    G = case["groups"]
    if G == 1:
        return key, None
    per = key.shape[1] // G
    value = key.view(-1, G, per).sort(-1, descending=True).values[..., :2].sum(-1)
    order = value.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
    keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, order, True)
    return key.masked_fill(~keep.repeat_interleave(per, 1), -math.inf), value


def _undecided(case, logits, bias):
    """Tokens whose choice, or whose order, hangs on the last bits of float32 sums."""
    _, key = _keys64(case, logits, bias)
    kept, value = _kept64(case, key)

    def close(v, n):
        top = v.sort(-1, descending=True).values[:, :n + 1]
        return (top[:, :-1] - top[:, 1:] < 3e-5 * top[:, :-1].abs().clamp(min=1e-30)).any(-1)

    bad = close(kept, case["k"])
    return bad | close(value, case["top_groups"]) if value is not None else bad


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, tokens, C = _DTYPES[case["dtype"]], case["tokens"], case["C"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["op"] == "rows":                                   # rows of different size, as activations are
        return {"case": case, "X": (randn(tokens, C) * torch.exp(randn(tokens, 1))).to(dtype)}
    E, k, N = case["E"], case["k"], case["N"]
    if case["op"] == "few":
        router = randn(E, C) / math.sqrt(C) * 1.5
        router = router.to(dtype)
        bias = 0.1 * randn(E) if case["bias"] else None
        X = randn(tokens, C).to(dtype)
        for attempt in range(40):
            bad = _undecided(case, X.double() @ router.double().t(), bias).nonzero().flatten()
            if bad.numel() == 0:
                break
            X[bad] = randn(bad.numel(), C).to(dtype)
        up, down = randn(E, C, N) * (2 / math.sqrt(C)), randn(E, N, C) / math.sqrt(N)
        state = {"case": case, "X": X, "router": router, "bias": bias}
        if not case["fp4"]:
            return {**state, "up": up.to(dtype), "down": down.to(dtype)}
        (uq, us), (dq, ds) = _pack(up.transpose(1, 2)), _pack(down.transpose(1, 2))
        return {**state, "up": uq, "up_scale": us, "down": dq, "down_scale": ds}
    popular = case["skew"] * randn(E)
    if case["idle"]:
        popular[:case["idle"]] = -1e4
    top = (randn(tokens, E) + popular).topk(k, -1)
    state = {"case": case, "X": randn(tokens, C).to(dtype), "experts": top.indices.to(torch.int32), "weights": torch.softmax(top.values, -1)}
    state["up"], state["up_scale"] = _pack(randn(E, N, C) * (2 / math.sqrt(C)))
    if case["op"] == "layer":
        state["down"], state["down_scale"] = _pack(randn(E, C, N) / math.sqrt(N))
    return state


# ---- the package's operators -------------------------------------------------------------------------

def _run_own(state):
    from expertscattergather_b200 import ops
    case, X = state["case"], state["X"]
    if case["op"] == "rows":
        q, s = ops.quantize_rows_fp4(X, activation="silu" if case["silu"] else None)
        return (ops.dequantize_rows_fp4(q, s, case["C"], dtype=X.dtype),)
    if case["op"] == "few":
        return ops.routed_experts_few(X, state["router"], state["up"], state["down"], case["k"], state["bias"], up_scale=state.get("up_scale"),
                                      down_scale=state.get("down_scale"), score=case["score"], groups=case["groups"],
                                      top_groups=case["top_groups"], renormalize=case["renorm"], scale=case["scale"])
    q, s = ops.quantize_rows_fp4(X)
    if case["E"] == 1:
        return (ops.matmul_fp4(q, s, state["up"][0], state["up_scale"][0], out_dtype=X.dtype),)
    plan = ops.plan_experts(state["experts"], case["E"])
    # rows stay float32 until a token's sum has been formed, which is rounded once
    if case["op"] == "product":
        Y = ops.expert_matmul_fp4(q, s, state["up"], state["up_scale"], plan, out_dtype=torch.float32)
    else:
        h, hs = ops.expert_matmul_fp4_rows(q, s, state["up"], state["up_scale"], plan, activation="silu")
        Y = ops.expert_matmul_fp4(h, hs, state["down"], state["down_scale"], plan, rows="sorted", out_dtype=torch.float32)
    return (ops.combine(Y, state["weights"], plan, out_dtype=X.dtype),)


# ---- the plain form ----------------------------------------------------------------------------------

def _silu(x):
    return x / (1 + torch.exp(-x))


def _rows_plain(state):
    X = state["X"].float()
    return (_values(_silu(X) if state["case"]["silu"] else X).to(state["X"].dtype),)


def _segments(experts, E):
    """Slots (token * k + j) sorted by expert, and where each expert's begin."""
    flat = experts.flatten().long()
    return flat.sort(stable=True).indices, torch.bincount(flat, minlength=E).tolist()


def _products_plain(state):
    case, X = state["case"], state["X"]
    q, k, C, N = _values(X.float()), case["k"], case["C"], case["N"]
    if case["E"] == 1:
        return ((q @ _unpacked(state["up"][0], state["up_scale"][0], C).t()).to(X.dtype),)
    order, counts = _segments(state["experts"], case["E"])
    rows = q[order // k]
    Y = torch.empty(order.numel(), C if case["op"] == "layer" else N, device=X.device)
    at = 0
    for e, n in enumerate(counts):
        if n:
            y = rows[at:at + n] @ _unpacked(state["up"][e], state["up_scale"][e], C).t()
            if case["op"] == "layer":
                y = _values(_silu(y)) @ _unpacked(state["down"][e], state["down_scale"][e], N).t()
            Y[at:at + n] = y
            at += n
    slots = torch.empty_like(Y)
    slots[order] = Y * state["weights"].flatten()[order].unsqueeze(-1)
    return (slots.view(X.shape[0], k, -1).sum(1).to(X.dtype),)


def _few_plain(state):
    case, x = state["case"], state["X"].float()
    logits = x @ state["router"].float().t()
    if case["score"] == "softmax":
        e = torch.exp(logits - logits.amax(-1, keepdim=True))
        s = e / e.sum(-1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-logits))
    key = s + state["bias"] if state["bias"] is not None else s
    (tokens, E), G, k = key.shape, case["groups"], case["k"]
    if G > 1:
        value = key.view(tokens, G, E // G).sort(-1, descending=True).values[..., :2].sum(-1)
        order = value.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, order, True)
        key = key.masked_fill(~keep.repeat_interleave(E // G, 1), -math.inf)
    experts = key.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, experts)
    if case["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    w = w * case["scale"]
    ids, rows = experts.flatten(), (_values(x) if case["fp4"] else x).repeat_interleave(k, 0).unsqueeze(1)
    if case["fp4"]:
        up = _unpacked(state["up"][ids], state["up_scale"][ids], case["C"]).transpose(1, 2)
        down = _unpacked(state["down"][ids], state["down_scale"][ids], case["N"]).transpose(1, 2)
    else:
        up, down = state["up"][ids].float(), state["down"][ids].float()
    h = _silu(torch.bmm(rows, up))
    y = torch.bmm(_values(h) if case["fp4"] else h, down).view(tokens, k, -1)
    return (y * w.unsqueeze(-1)).sum(1).to(state["X"].dtype), w, experts.to(torch.int32)


def run(state):
    if own:
        return _run_own(state)
    return {"rows": _rows_plain, "product": _products_plain, "layer": _products_plain, "few": _few_plain}[state["case"]["op"]](state)


# ---- the work, and the definitions in float64 --------------------------------------------------------

def _bytes4(rows, C):
    return rows * (C / 2 + math.ceil(C / 32))


def work(case):
    tokens, C = case["tokens"], case["C"]
    es = torch.empty((), dtype=_DTYPES[case["dtype"]]).element_size()
    if case["op"] == "rows":      # the rows, their 4 bits, and the values that those stand for
        return {"bytes": 2 * tokens * C * es + _bytes4(tokens, C), "flops": 4 * tokens * C}
    E, k, N = case["E"], case["k"], case["N"]
    slots = tokens * k
    if case["op"] == "few":       # experts that a balanced choice uses
        used = E * (1 - (1 - k / E) ** tokens)
        each = _bytes4(2 * N, C) if case["fp4"] else 2 * C * N * es
        return {"bytes": 2 * tokens * C * es + E * C * es + used * each + 8 * slots, "flops": 4 * slots * C * N + 2 * tokens * E * C}
    used = min(E - case["idle"], slots)
    routed = 0 if E == 1 else 8 * slots
    both = 2 if case["op"] == "layer" else 1
    return {"bytes": tokens * (C + (C if both == 2 else N)) * es + both * used * _bytes4(N, C) + routed, "flops": both * 2 * slots * C * N}


def _exact_values(x):
    """What rows [..., C] in float64 are in 4 bits: from the borders between the values, ties to the even mantissa."""
    C = x.shape[-1]
    pad = torch.nn.functional.pad(x, (0, -C % 32)).unflatten(-1, (-1, 32))
    mantissa, exponent = torch.frexp(pad.abs().amax(-1, keepdim=True))
    exponent = (exponent - 3 + (mantissa > 0.875)).clamp(min=-127)
    m = torch.ldexp(pad.abs(), -exponent)
    index = sum((m > b).long() for b in (0.25, 1.25, 2.5, 5.0)) + sum((m >= b).long() for b in (0.75, 1.75, 3.5))
    level = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    return torch.ldexp(level[index], exponent).copysign(pad).flatten(-2)[..., :C]


def _exact_weights(packed, byte, C):
    code = torch.stack((packed % 16, packed // 16), -1).flatten(-2)[..., :C].long()
    e, m = code % 8 // 2, code % 2
    v = torch.where(e > 0, (2.0 + m) * 2.0 ** (e - 2.0).double(), m * 0.5)
    return torch.where(code > 7, -v, v) * 2.0 ** (byte.double() - 127).repeat_interleave(32, -1)[..., :C]


def exact(case, seed):
    state = prepare(case, seed)
    X, C = state["X"].double(), case["C"]
    if case["op"] == "rows":
        return (_exact_values(X * torch.sigmoid(X) if case["silu"] else X),)
    N, E, k, tokens = case["N"], case["E"], case["k"], case["tokens"]
    layers = 1 if case["op"] == "product" else 2
    if 2 * layers * tokens * k * C * N > 3e12:
        return None
    fp4 = case.get("fp4", True)
    if case["op"] == "few":
        s, key = _keys64(case, X @ state["router"].double().t(), state["bias"])
        ids = _kept64(case, key)[0].sort(dim=-1, descending=True, stable=True).indices[:, :k]
        w = s.gather(1, ids)
        w = w / w.sum(-1, keepdim=True) * case["scale"] if case["renorm"] else w * case["scale"]
    else:
        ids, w = state["experts"].long(), state["weights"].double()
    x = _exact_values(X) if fp4 else X
    if E == 1:
        return (x @ _exact_weights(state["up"][0], state["up_scale"][0], C).t(),)
    out = torch.zeros(tokens, C if layers == 2 else N, device="cuda", dtype=torch.float64)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        y = x[t] @ (_exact_weights(state["up"][e], state["up_scale"][e], C).t() if fp4 else state["up"][e].double())
        if layers == 2:
            y = y * torch.sigmoid(y)
            y = _exact_values(y) @ _exact_weights(state["down"][e], state["down_scale"][e], N).t() if fp4 else y @ state["down"][e].double()
        out.index_put_((t,), w[t, j].unsqueeze(-1) * y, accumulate=True)
    return (out, w, ids.to(torch.int32)) if case["op"] == "few" else (out,)
