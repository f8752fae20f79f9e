"""Operators for tokens that choose experts against their definitions in float64.

Tolerances are bounds, not fits.  With u = 2^-24: a float32 sum of n products is off by at most (n + 2) * 2 * u times the sum of their
magnitudes (2 u an addition: the tensor core truncates), a rounding to bfloat16 / float16 by 2^-8 / 2^-11 of the value (and by half of the
smallest float16, 2^-25).  Scores are off by a few u relative to themselves: expf (2 ulp), the subtraction in its argument (u times the
argument's size, at most 32 here), a division, a sum of positive terms.
"""
import itertools
import math

import pytest
import torch

from expertscattergather_b200 import RoutedExperts, ops, token_choice
from oracle import choice_oracle as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def close(got, ref, size, terms, dtype=None, extra=0.0):
    dtype = dtype or got.dtype
    tol = (terms + 2) * 2 * U * size + (HALF[dtype] + 4 * U) * ref.abs() + TINY[dtype] + extra
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} elements off, first at {bad.nonzero()[0].tolist()}: " \
        f"{got[bad][0].item()} for {ref[bad][0].item()} +- {tol[bad][0].item()}"


def draw_experts(g, tokens, k, E, kind="even"):
    scores = torch.rand(tokens, E, device="cuda", generator=g)
    if kind == "skewed":
        scores += 2.0 / (1 + torch.arange(E, device="cuda"))
    ids = scores.topk(k, -1).indices.int()
    if kind == "one":                                     # every token's first choice is the same expert, the others are dropped
        ids[:] = -1
        ids[:, 0] = E // 2
    if kind == "none":
        ids[:] = -1
    if kind == "holes":
        ids[torch.rand(tokens, k, device="cuda", generator=g) < 0.4] = -1
    return ids


# ---- routing -------------------------------------------------------------------------------------------

ROUTE_SHAPES = [(1, 1, 1), (3, 8, 2), (7, 31, 5), (33, 33, 32), (64, 64, 8), (65, 60, 6), (1000, 128, 4), (257, 256, 8), (19, 515, 9), (9, 1024, 32)]


@pytest.mark.parametrize("tokens,E,k", ROUTE_SHAPES)
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_weights(cuda_device, tokens, E, k, score, renorm):
    for dtype, with_bias in itertools.product(DTYPES, (False, True)):
        g = gen(E + tokens)
        logits = randn(g, tokens, E, dtype=dtype) * 2
        bias = 0.3 * randn(g, E) if with_bias else None
        w, ids = ops.route_tokens(logits, k, bias, score=score, renormalize=renorm, scale=1.7)
        assert w.shape == ids.shape == (tokens, k) and w.dtype == torch.float32 and ids.dtype == torch.int32
        s = orc.scores(logits, score)
        check_choice(s if bias is None else s + bias.double(), ids, 1e-6)
        if not with_bias:                                  # equal logits: lower expert first
            assert torch.equal(ids.long(), logits.float().sort(dim=-1, descending=True, stable=True).indices[:, :k])
        ref = orc.weights_of(s, ids, renorm, 1.7)
        # argument of the exponential: u * 32; expf, sum, division and scale: another 16 u with the sum's (log-like tree) terms
        assert ((w.double() - ref).abs() <= 64 * U * ref + 1e-40).all()


def check_choice(key, ids, tol, kept=None):
    """ids are distinct, best first, and nothing better was left out, within a rounding of the keys."""
    ids = ids.long()
    assert ((ids >= 0) & (ids < key.shape[-1])).all()
    assert (ids.sort(-1).values.diff(dim=-1) > 0).all()
    got = key.gather(-1, ids)
    assert (got[..., :-1] >= got[..., 1:] - tol).all()
    left = key.scatter(-1, ids, -float("inf"))
    if kept is not None:
        left = left.masked_fill(~kept, -float("inf"))
        assert kept.gather(-1, ids).all()
    assert (left.amax(-1) <= got[..., -1] + tol).all()


@pytest.mark.parametrize("groups,per,top_groups,k", [(1, 40, 1, 5), (2, 1, 2, 2), (4, 15, 2, 6), (8, 32, 4, 8), (32, 32, 1, 32), (3, 7, 3, 21), (5, 13, 2, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups(cuda_device, groups, per, top_groups, k, score):
    E, tokens = groups * per, 333
    for group_top, with_bias in itertools.product((1, 2), (False, True)):
        g = gen(per)
        logits = randn(g, tokens, E) * 1.5
        bias = 0.2 * randn(g, E) if with_bias else None
        w, ids = ops.route_tokens(logits, k, bias, score=score, groups=groups, top_groups=top_groups, group_top=group_top)
        s = orc.scores(logits, score)
        key = s + bias.double() if with_bias else s
        value = orc.group_values(key, groups, group_top)
        kept = value.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
        # tokens whose groups are apart by more than a rounding: their groups are known
        order = value.sort(-1, descending=True).values
        clear = torch.ones(tokens, dtype=torch.bool, device="cuda") if top_groups == groups else order[:, top_groups - 1] - order[:, top_groups] > 1e-6
        mask = torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True).repeat_interleave(per, 1)
        check_choice(key[clear], ids[clear], 1e-6, mask[clear])
        assert clear.float().mean() > 0.95
        ref = orc.weights_of(s, ids, True, 1.0)
        assert ((w.double() - ref).abs() <= 64 * U * ref + 1e-40).all()


def test_route_equal_keys_and_groups(cuda_device):
    """Small integers: ties everywhere, between experts and between groups; the lower one comes first."""
    g = gen(5)
    logits = torch.randint(-1, 2, (500, 48), device="cuda", generator=g).float()
    _, ids = ops.route_tokens(logits, 10, score="sigmoid")
    assert torch.equal(ids.long(), logits.sort(dim=-1, descending=True, stable=True).indices[:, :10])
    _, ids = ops.route_tokens(logits, 5, score="sigmoid", groups=6, top_groups=2, group_top=1)
    value = logits.view(500, 6, 8).amax(-1)
    keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, value.sort(dim=-1, descending=True, stable=True).indices[:, :2], True)
    masked = logits.masked_fill(~keep.repeat_interleave(8, 1), -float("inf"))
    assert torch.equal(ids.long(), masked.sort(dim=-1, descending=True, stable=True).indices[:, :5])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_masked_and_extreme_logits(cuda_device, score):
    inf = float("inf")
    lowest = torch.finfo(torch.float32).min
    logits = torch.zeros(6, 40, device="cuda")
    logits[0] = -inf                                       # nothing left
    logits[1] = lowest                                     # the type's lowest value everywhere
    logits[2] = -inf
    logits[2, 7] = 0.5                                     # one expert left of the four asked for
    logits[3, 5] = float("nan")
    logits[4] = torch.arange(40, device="cuda") * 100.0 - 2000
    logits[5, 3], logits[5, 30] = -0.0, 1e-30
    for renorm in (True, False):
        w, ids = ops.route_tokens(logits, 4, score=score, renormalize=renorm)
        d = ops.route_tokens_backward(torch.ones_like(w), logits, ids, score=score, renormalize=renorm)
        for row in ids.long().tolist():
            assert len(set(row)) == 4 and all(0 <= e < 40 for e in row)
        assert ids[0].tolist() == [0, 1, 2, 3] and (w[0] == 0).all() and (d[0] == 0).all()
        assert ids[1].tolist() == [0, 1, 2, 3]
        share = 0.25 if renorm else 1 / 40
        if score == "softmax":
            assert torch.allclose(w[1], torch.full_like(w[1], share))
        else:
            assert (w[1] == 0).all() and (d[1] == 0).all()         # scores of exactly 0
        assert ids[2].tolist() == [7, 0, 1, 2] and (w[2, 1:] == 0).all() and w[2, 0] > 0
        assert not torch.isnan(d[2]).any()
        assert 5 not in ids[3].tolist()                            # NaN comes last
        assert ids[4].tolist() == [39, 38, 37, 36]
        assert ids[5].tolist() == [30, 0, 1, 2]
    w, ids = ops.route_tokens(logits[3:4], 32, score=score)
    assert 5 not in ids[0].tolist()


def test_route_strides_and_shapes(cuda_device):
    g = gen(1)
    wide = randn(g, 50, 3, 100, dtype=torch.bfloat16)
    for logits in (wide[:, 1, 10:74], wide[..., 3:67], wide[::2, 0, :64], wide.transpose(0, 2)[:64, 1].t(), wide[0, 0, :64].expand(9, 64)):
        w, ids = ops.route_tokens(logits, 6)
        w2, ids2 = ops.route_tokens(logits.contiguous().clone(), 6)
        assert torch.equal(w, w2) and torch.equal(ids, ids2) and w.shape == (*logits.shape[:-1], 6)
        gr = randn(g, *w.shape)
        assert torch.equal(ops.route_tokens_backward(gr, logits, ids), ops.route_tokens_backward(gr, logits.contiguous(), ids))
    w, ids = ops.route_tokens(wide[0, 0, :64], 6)
    assert w.shape == (6,)
    w, ids = ops.route_tokens(torch.empty(0, 64, device="cuda"), 6)
    assert w.shape == ids.shape == (0, 6)
    assert ops.route_tokens_backward(w, torch.empty(0, 64, device="cuda"), ids).shape == (0, 64)


@pytest.mark.parametrize("tokens,E,k", ROUTE_SHAPES)
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_gradient(cuda_device, tokens, E, k, score, renorm):
    for dtype in DTYPES:
        g = gen(tokens * E)
        logits = randn(g, tokens, E, dtype=dtype) * 2
        _, ids = ops.route_tokens(logits, k, score=score, renormalize=renorm)
        dw = randn(g, tokens, k)
        got = ops.route_tokens_backward(dw, logits, ids, score=score, renormalize=renorm, scale=0.7)
        x = logits.double().requires_grad_(True)
        w = orc.weights_of(orc.scores_of_gradient(x, score), ids, renorm, 0.7)
        (w * dw.double()).sum().backward()
        # terms of a row's sums of up to |dw| * weight, each off by a few u (see test_route_weights)
        size = (w.abs() * dw.double().abs()).sum(-1, keepdim=True) + (w.abs() * dw.double().abs()).amax(-1, keepdim=True)
        tol = (128 + k) * U * size + HALF[dtype] * x.grad.abs() + TINY[dtype]
        assert ((got.double() - x.grad).abs() <= tol).all()
        assert got.dtype == dtype


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_gradient_against_differences(cuda_device, score, renorm):
    """Along a direction, with steps that change no choice: central differences of the forward pass.  Step h = 2^-6: the third
    derivative of a score is at most 1, the truncation h^2 / 6 * |direction|^3-like terms; rounding u / h."""
    g = gen(3)
    tokens, E, k, h = 200, 24, 4, 2.0 ** -6
    logits = torch.stack([torch.randperm(E, device="cuda", generator=g) for _ in range(tokens)]).float() * 0.25
    v = torch.rand(tokens, E, device="cuda", generator=g) * 2 - 1
    opts = {"score": score, "renormalize": renorm}
    w, ids = ops.route_tokens(logits, k, **opts)
    dw = randn(g, tokens, k)
    up, ids_up = ops.route_tokens(logits + h * v, k, **opts)
    down, ids_down = ops.route_tokens(logits - h * v, k, **opts)
    assert torch.equal(ids, ids_up) and torch.equal(ids, ids_down)
    diff = ((up.double() - down.double()) * dw.double()).sum(-1) / (2 * h)
    got = (ops.route_tokens_backward(dw, logits, ids, **opts).double() * v.double()).sum(-1)
    tol = (h * h + 64 * U / h) * dw.double().abs().sum(-1)
    assert ((got - diff).abs() <= tol).all()


def test_route_gradient_ignores_choices_taken_away(cuda_device):
    g = gen(4)
    logits = randn(g, 30, 20)
    _, ids = ops.route_tokens(logits, 5, score="sigmoid")
    dw = randn(g, 30, 5)
    cut = ids.clone()
    cut[:, 3:] = -1
    cut[3] = -1
    got = ops.route_tokens_backward(dw, logits, cut, score="sigmoid")
    assert torch.equal(got[4:], ops.route_tokens_backward(dw[:, :3].contiguous(), logits, ids[:, :3].contiguous(), score="sigmoid")[4:])
    assert (got[3] == 0).all()


def test_route_refusals(cuda_device):
    x = torch.zeros(4, 12, device="cuda")
    for kw in ({"top_k": 0}, {"top_k": 13}, {"top_k": 2, "groups": 5}, {"top_k": 2, "groups": 4, "top_groups": 5}, {"top_k": 4, "groups": 4},
               {"top_k": 2, "groups": 4, "top_groups": 0}, {"top_k": 2, "group_top": 3}, {"top_k": 2, "score": "relu"}, {"top_k": 2, "groups": 0}):
        with pytest.raises(ValueError):
            ops.route_tokens(x, **kw)
    with pytest.raises(ValueError):
        ops.route_tokens(torch.zeros(2, 1025, device="cuda"), 2)
    with pytest.raises(ValueError):
        ops.route_tokens(torch.zeros(2, 64, device="cuda"), 33)
    with pytest.raises(ValueError):
        ops.route_tokens(x.double(), 2)
    with pytest.raises(ValueError):
        ops.route_tokens(x, 2, torch.zeros(11, device="cuda"))
    with pytest.raises(RuntimeError):
        ops.route_tokens(x.cpu(), 2)
    with pytest.raises(RuntimeError):
        ops.route_tokens(x, 2, torch.zeros(12))
    w, ids = ops.route_tokens(x, 2)
    with pytest.raises(ValueError):
        ops.route_tokens_backward(w[:3], x, ids)
    with pytest.raises(ValueError):
        ops.route_tokens_backward(w, x, ids.float())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_one_choice_of_weight_one_has_no_gradient(cuda_device, dtype, score):
    g = gen(3)
    x, d = randn(g, 4000, 24, dtype=dtype), torch.randn(4000, 1, device="cuda", generator=g)
    w, ids = ops.route_tokens(x, 1, score=score, scale=2.5)
    assert (w == 2.5).all() and torch.equal(ids[:, 0].long(), x.argmax(-1))
    assert not ops.route_tokens_backward(d, x, ids, score=score, scale=2.5).any()


# ---- the plan ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens,k,E", [(0, 2, 4), (1, 1, 1), (1, 8, 64), (5, 3, 7), (300, 4, 60), (1024, 2, 33), (4096, 8, 256), (700, 3, 1024), (40000, 4, 64), (150000, 8, 13)])
@pytest.mark.parametrize("kind", ["even", "skewed", "one", "none", "holes"])
def test_plan(cuda_device, tokens, k, E, kind):
    ids = draw_experts(gen(tokens), tokens, k, E, kind)
    plan = ops.plan_experts(ids, E)
    offsets, slots, position = orc.plan(ids, E)
    assert torch.equal(plan.offsets.long(), offsets)
    assert torch.equal(plan.slots.long(), slots)
    assert torch.equal(plan.position.long(), position)
    assert (plan.tokens, plan.k, plan.E) == (tokens, k, E)
    assert torch.equal(plan.counts().long(), offsets.diff())
    ops.check_status()


# one CTA, clusters of 2 to 16, more of a warp's slots, and stretches counted before; the last stretch with one slot, or whole
@pytest.mark.parametrize("n", [2048, 2049, 4096, 4097, 6145, 8193, 16384, 16385, 31000, 32768, 32769, 65536, 65537, 131072, 131073, 600001])
@pytest.mark.parametrize("E", [1, 64, 1024])
def test_plan_of_every_size_of_cluster(cuda_device, n, E):
    g = gen(n + E)
    ids = (torch.rand(n, 1, device="cuda", generator=g) ** 2 * E).int().clamp_(max=E - 1)
    ids[torch.rand(n, 1, device="cuda", generator=g) < 0.1] = -1
    plan = ops.plan_experts(ids, E)
    for mine, ref in zip((plan.offsets, plan.slots, plan.position), orc.plan(ids, E)):
        assert torch.equal(mine.long(), ref)
    ops.check_status()
    ids[n - 1, 0] = E
    assert ops.plan_experts(ids, E).position[n - 1].item() < 0
    with pytest.raises(RuntimeError):
        ops.check_status()


def test_plan_types_and_ids_out_of_range(cuda_device):
    ids = torch.tensor([[0, 5], [2, -1], [4, 1]], device="cuda")
    for dtype in (torch.int64, torch.int16, torch.int8, torch.int32):
        plan = ops.plan_experts(ids.to(dtype), 6)
        assert plan.offsets.tolist() == [0, 1, 2, 3, 3, 4, 5] and plan.position.tolist() == [0, 4, 2, ~5, 3, 1]
    ops.check_status()
    for bad in (6, -2, 2 ** 40, -2 ** 40):
        t = ids.clone()
        t[0, 0] = bad
        plan = ops.plan_experts(t, 6)
        assert plan.offsets.tolist() == [0, 0, 1, 2, 2, 3, 4] and plan.position.tolist() == [~4, 3, 1, ~5, 2, 0]
        with pytest.raises(RuntimeError):
            ops.check_status()
    for E in (0, 1025):
        with pytest.raises(ValueError):
            ops.plan_experts(ids, E)
    with pytest.raises(ValueError):
        ops.plan_experts(ids.float(), 6)
    with pytest.raises(RuntimeError):
        ops.plan_experts(ids.cpu(), 6)


# ---- products ------------------------------------------------------------------------------------------

# tokens, k, E, C, N: one token, tiles and parts of tiles, rows that start anywhere, wide and narrow widths, one expert
MATMUL_SHAPES = [(1, 1, 1, 1, 1), (1, 8, 64, 256, 128), (2, 3, 5, 17, 9), (40, 2, 3, 64, 64), (129, 1, 1, 72, 136), (150, 2, 4, 72, 100), (257, 2, 4, 128, 264), (500, 4, 13, 330, 201),
                 (6, 4, 64, 264, 136), (4, 5, 64, 1001, 77), (3, 8, 64, 2600, 300), (30, 4, 64, 264, 136), (25, 5, 64, 1001, 77), (20, 1, 64, 2600, 300), (1000, 3, 8, 1024, 256), (64, 2, 16, 2050, 70), (2000, 2, 4, 96, 520), (3, 2, 300, 40, 24), (700, 8, 40, 512, 16)]


@pytest.mark.parametrize("tokens,k,E,C,N", MATMUL_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["even", "skewed", "holes"])
def test_expert_matmul(cuda_device, tokens, k, E, C, N, dtype, kind):
    g = gen(C + N)
    k = min(k, E)
    ids = draw_experts(g, tokens, k, E, kind)
    plan = ops.plan_experts(ids, E)
    X, W = randn(g, tokens, C, dtype=dtype), randn(g, E, C, N, dtype=dtype)
    Xs = randn(g, tokens * k, C, dtype=dtype)
    paths = ("auto", "generic")
    for rows, x in (("tokens", X), ("sorted", Xs)):
        ref, size = orc.matmul(x, W, ids, E, rows)
        for path, (layout, w) in itertools.product(paths, (("cn", W), ("nc", W.transpose(1, 2).contiguous()))):
            close(ops.expert_matmul(x, w, plan, rows=rows, w_layout=layout, path=path), ref, size, C)
    dY = randn(g, tokens * k, N, dtype=dtype)
    for rows, x in (("tokens", X), ("sorted", Xs)):
        ref, size = orc.dweight(x, dY, ids, E, rows)
        most = int(plan.counts().max())
        for path in paths:
            close(ops.expert_dweight(x, dY, plan, rows=rows, path=path), ref, size, most)
    ops.check_status()


# experts of 0, 1, 2 .. rows up to two blocks of 32 and one more; contractions around the steps of 32, rows that are no whole 16 bytes
@pytest.mark.parametrize("C,N", [(1, 1), (3, 5), (31, 64), (32, 65), (33, 68), (64, 130), (100, 63), (132, 260), (1027, 66)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_experts_of_every_small_number_of_rows(cuda_device, C, N, dtype):
    E, g = 66, gen(C * 1000 + N)
    ids = torch.arange(E, device="cuda", dtype=torch.int32).repeat_interleave(torch.arange(E, device="cuda"))
    ids = ids[torch.randperm(len(ids), device="cuda", generator=g)].view(-1, 1)
    tokens = len(ids)
    plan = ops.plan_experts(ids, E)
    X, W = randn(g, tokens, C, dtype=dtype), randn(g, E, C, N, dtype=dtype)
    for rows in ("tokens", "sorted"):
        ref, size = orc.matmul(X, W, ids, E, rows)
        for layout, w in (("cn", W), ("nc", W.transpose(1, 2).contiguous())):
            close(ops.expert_matmul(X, w, plan, rows=rows, w_layout=layout), ref, size, C)
    wide = randn(g, tokens, C + 5, dtype=dtype)                  # rows that begin anywhere
    ref, size = orc.matmul(wide[:, 1:C + 1], W, ids, E, "tokens")
    close(ops.expert_matmul(wide[:, 1:C + 1], W, plan), ref, size, C)
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["one", "none"])
def test_expert_products_of_one_expert_or_none(cuda_device, dtype, kind):
    g = gen(8)
    tokens, k, E, C, N = 400, 2, 6, 128, 192
    ids = draw_experts(g, tokens, k, E, kind)
    plan = ops.plan_experts(ids, E)
    X, W, dY = randn(g, tokens, C, dtype=dtype), randn(g, E, C, N, dtype=dtype), randn(g, tokens * k, N, dtype=dtype)
    ref, size = orc.matmul(X, W, ids, E, "tokens")
    close(ops.expert_matmul(X, W, plan), ref, size, C)
    ref, size = orc.dweight(X, dY, ids, E, "tokens")
    close(ops.expert_dweight(X, dY, plan), ref, size, tokens)


@pytest.mark.parametrize("tokens,k,E,C,N", [(300, 2, 6, 128, 192), (9, 2, 6, 128, 192), (301, 3, 5, 130, 67)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_leaks_between_experts(cuda_device, tokens, k, E, C, N, dtype):
    """Infinities and NaN in the rows and weights of one expert, and in rows that are not routed, stay there."""
    g = gen(9)
    ids = draw_experts(g, tokens, k, E, "even")
    ids[tokens - 3:] = -1
    plan = ops.plan_experts(ids, E)
    X, W, dY = randn(g, tokens, C, dtype=dtype), randn(g, E, C, N, dtype=dtype), randn(g, tokens * k, N, dtype=dtype)
    bad = 2
    touched = (ids == bad).any(-1)
    Xn, Wn, Yn = X.clone(), W.clone(), dY.clone()
    Wn[bad] = float("nan")
    Xn[tokens - 3:] = float("nan")
    a, b = plan.offsets[bad].item(), plan.offsets[bad + 1].item()
    Yn[a:b] = float("inf")
    Yn[plan.offsets[E].item():] = float("nan")
    rows = torch.ones(tokens * k, dtype=torch.bool, device="cuda")
    rows[a:b] = False
    for path in ("auto", "generic"):
        ref, got = ops.expert_matmul(X, W, plan, path=path), ops.expert_matmul(Xn, Wn, plan, path=path)
        assert torch.equal(ref[rows], got[rows]) and (b == a or torch.isnan(got[a:b]).all())
        ref, got = ops.expert_matmul(dY, W, plan, rows="sorted", w_layout="cn", path=path) if C == N else (None, None), None
        ref, got = ops.expert_dweight(X, dY, plan, path=path), ops.expert_dweight(Xn, Yn, plan, path=path)
        keep = torch.ones(E, dtype=torch.bool, device="cuda")
        keep[bad] = False
        assert torch.equal(ref[keep], got[keep])
        out = ops.combine(ops.expert_matmul(Xn, Wn, plan, path=path), None, plan)
        assert not torch.isnan(out[~touched]).any()
    ops.check_status()


def test_products_do_not_depend_on_strides_or_alignment(cuda_device):
    g = gen(10)
    ids = draw_experts(g, 100, 2, 4, "even")
    plan = ops.plan_experts(ids, 4)
    for dtype in DTYPES:
        X, W, dY = randn(g, 100, 64, dtype=dtype), randn(g, 4, 64, 48, dtype=dtype), randn(g, 200, 48, dtype=dtype)
        Y, dW = ops.expert_matmul(X, W, plan), ops.expert_dweight(X, dY, plan)
        odd = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)       # starts one element into its storage
        wide = lambda t: torch.stack([t, t], -1)[..., 0]
        for f in (odd, wide, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):
            assert torch.equal(ops.expert_matmul(f(X), f(W), plan), Y) and torch.equal(ops.expert_dweight(f(X), f(dY), plan), dW)
            out = ops.combine(f(Y), None, plan)
            assert torch.equal(out, ops.combine(Y, None, plan))
        assert torch.equal(ops.expert_matmul(X.view(10, 10, 64), W, plan), Y)


def test_product_widths_of_zero(cuda_device):
    ids = draw_experts(gen(1), 10, 2, 4, "even")
    plan = ops.plan_experts(ids, 4)
    for dtype in DTYPES:
        z = lambda *s: torch.zeros(*s, device="cuda", dtype=dtype)
        assert ops.expert_matmul(z(10, 0), z(4, 0, 8), plan).eq(0).all()
        assert ops.expert_matmul(z(10, 8), z(4, 8, 0), plan).shape == (20, 0)
        assert ops.expert_dweight(z(10, 0), z(20, 8), plan).shape == (4, 0, 8)
        empty = ops.plan_experts(ids[:0], 4)
        assert ops.expert_matmul(z(0, 8), z(4, 8, 8), empty).shape == (0, 8)
        assert ops.expert_dweight(z(0, 8), z(0, 8), empty).eq(0).all() and ops.expert_dweight(z(0, 8), z(0, 8), empty).shape == (4, 8, 8)
        assert ops.combine(z(0, 8), None, empty).shape == (0, 8)


def test_product_refusals(cuda_device):
    ids = draw_experts(gen(1), 10, 2, 4, "even")
    plan = ops.plan_experts(ids, 4)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dtype)
    for X, W, kw in ((z(11, 8), z(4, 8, 8), {}), (z(10, 8), z(5, 8, 8), {}), (z(10, 8), z(4, 9, 8), {}), (z(10, 8), z(4, 8, 8), {"rows": "sorted"}),
                     (z(10, 8), z(4, 8, 8), {"rows": "x"}), (z(10, 8), z(4, 8, 8), {"w_layout": "x"}), (z(10, 8), z(4, 8, 8, dtype=torch.float16), {}),
                     (z(10, 8, dtype=torch.float64), z(4, 8, 8, dtype=torch.float64), {}), (z(10, 8), z(8, 8), {})):
        with pytest.raises(ValueError):
            ops.expert_matmul(X, W, plan, **kw)
    with pytest.raises(RuntimeError):
        ops.expert_matmul(z(10, 8).cpu(), z(4, 8, 8), plan)
    for X, dY in ((z(11, 8), z(20, 8)), (z(10, 8), z(10, 8)), (z(10, 8), z(20, 8, dtype=torch.float32))):
        with pytest.raises(ValueError):
            ops.expert_dweight(X, dY, plan)
    for Y, w in ((z(10, 8), None), (z(20, 8), z(10, 3)), (z(20, 8), z(10, 2, dtype=torch.float16))):
        with pytest.raises(ValueError):
            ops.combine(Y, w, plan)
    with pytest.raises(ValueError):
        ops.combine_backward(z(9, 8), z(20, 8), z(10, 2), plan)


@pytest.mark.parametrize("tokens,k,N", [(1, 1, 1), (1, 8, 512), (7, 3, 13), (300, 4, 200), (129, 32, 8), (1000, 2, 1032)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["even", "holes"])
def test_combine(cuda_device, tokens, k, N, dtype, kind):
    E = max(40, k)
    g = gen(N)
    ids = draw_experts(g, tokens, k, E, kind)
    plan = ops.plan_experts(ids, E)
    Y = randn(g, tokens * k, N, dtype=dtype)
    Y[plan.offsets[E].item():] = float("nan")              # rows of slots that were not routed are not read
    dOut = randn(g, tokens, N, dtype=dtype)
    routed = plan.position.view(tokens, k) >= 0
    for w in (None, torch.rand(tokens, k, device="cuda", generator=g), torch.rand(tokens, k, device="cuda", generator=g).to(dtype)):
        out = ops.combine(Y, w, plan)
        ref, size = orc.combine(Y, w, plan.position, tokens, k)
        close(out, ref, size, k)
        dY, dw = ops.combine_backward(dOut, Y, w, plan)
        wd = torch.ones(tokens * k, device="cuda", dtype=torch.float64) if w is None else w.double().flatten()
        ref = (dOut.double()[plan.slots.long() // k] * wd[plan.slots.long()].unsqueeze(-1))
        ref[plan.offsets[E].item():] = 0
        close(dY, ref, ref.abs(), 0)
        if w is None:
            assert dw is None
            continue
        rows = Y.double().nan_to_num(0)[torch.where(routed, plan.position.view(tokens, k), 0).long()]
        prod = rows * dOut.double().unsqueeze(1)
        close(dw, prod.sum(-1) * routed, prod.abs().sum(-1), N)
        assert dw.dtype == w.dtype


# short rows, slots enough for warps that have several one after the other; 4, 8 and 16 lanes to a slot
@pytest.mark.parametrize("tokens,k,N", [(20000, 4, 8), (30001, 3, 32), (50001, 2, 1), (16000, 4, 60), (9001, 4, 128), (24001, 2, 17)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["skewed", "holes"])
def test_combine_of_many_short_rows(cuda_device, tokens, k, N, dtype, kind):
    test_combine(cuda_device, tokens, k, N, dtype, kind)


def test_layer_gradients(cuda_device):
    """Products and combine through autograd, float32: the formulas' gradients in float64 (by autograd of the definition)."""
    g = gen(11)
    tokens, k, E, C, N = 60, 3, 5, 20, 12
    ids = draw_experts(g, tokens, k, E, "even")
    plan = ops.plan_experts(ids, E)
    X, W, w = (t.requires_grad_(True) for t in (randn(g, tokens, C), randn(g, E, C, N), torch.rand(tokens, k, device="cuda", generator=g)))
    dOut = randn(g, tokens, N)
    token_choice.combine(token_choice.expert_matmul(X, W, plan), w, plan).backward(dOut)
    X2, W2, w2 = (t.detach().double().requires_grad_(True) for t in (X, W, w))
    out = (w2.unsqueeze(-1) * torch.einsum("tc,tkcn->tkn", X2, W2[ids.long()])).sum(1)
    out.backward(dOut.double())
    for a, b in ((X, X2), (W, W2), (w, w2)):
        # sums of at most k * N, tokens and C * N products of normal numbers: magnitudes below 4 sigma a factor
        assert (a.grad.double() - b.grad).abs().max() <= (tokens + C * N) * 2 * U * 4 * 4 * 4 * math.sqrt(C)


def test_layer_against_differences(cuda_device):
    """The whole layer: a loss' change along a direction of all parameters against its gradient."""
    g = gen(12)
    torch.manual_seed(1)
    layer = RoutedExperts(8, 24, 16, 2).cuda()
    x = randn(g, 3, 50, 24)
    c = randn(g, 3, 50, 24)
    params = list(layer.parameters())
    loss = lambda: (layer(x).double() * c.double()).sum()
    loss().backward()
    slope, dirs = 0.0, []
    for p in params:
        v = randn(g, *p.shape)
        dirs.append(v)
        slope += (p.grad.double() * v.double()).sum().item()
    ids = layer.router(x)[1].clone()
    h, vals = 2.0 ** -13, []
    with torch.no_grad():
        for sign in (1, -2):
            for p, v in zip(params, dirs):
                p += sign * h * v
            assert torch.equal(layer.router(x)[1], ids)
            vals.append(loss().item())
    diff = (vals[0] - vals[1]) / (2 * h)
    assert abs(diff - slope) <= 2e-2 * abs(slope) + 2e-2, (diff, slope)


# ---- 8-bit integers ------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,C", [(0, 8), (1, 1), (3, 7), (5, 16), (100, 330), (33, 1024), (9, 4096), (7, 9001), (4, 20000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows(cuda_device, rows, C, dtype):
    g = gen(C)
    X = randn(g, rows, C, dtype=dtype) * torch.rand(rows, 1, device="cuda", generator=g).to(dtype)
    if rows > 2:
        X[1] = 0
        X[2] = X[2, 0]
    q, s = ops.quantize_rows(X)
    assert q.shape == X.shape and q.dtype == torch.int8 and s.shape == (rows,) and (rows < 2 or q.stride(0) % 16 == 0)
    ref = (X.double().abs().amax(-1) / 127).float() if rows else s      # (torch multiplies float32 by a rounded 1 / 127)
    assert torch.equal(s, ref)
    want = torch.where(s.unsqueeze(-1) == 0, torch.zeros_like(X, dtype=torch.float32), X.float() / s.unsqueeze(-1)).round()
    assert torch.equal(q.float(), want)
    exact_q, exact_s = orc.quantize(X)
    # off by one only where the exact quotient lies within a rounding of a half
    off = (q.double() - exact_q).abs()
    assert off.max().item() <= (1 if rows else 0) if rows else True
    assert ((s.double() - exact_s).abs() <= U * exact_s).all()


# rows enough for warps that have one after the other (beside: too few, rows that are no whole 16 bytes, rows too long)
@pytest.mark.parametrize("rows,C", [(7104, 64), (7105, 8), (7300, 520), (15000, 1024), (30000, 136), (8000, 132), (7200, 1032), (14209, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_many_rows(cuda_device, rows, C, dtype):
    g = gen(rows)
    X = randn(g, rows, C + 16, dtype=dtype)[:, :C]                    # (rows with a pitch)
    X[5], X[rows - 2, C - 1], X[rows - 1] = 0, float("inf"), X[rows - 1] * 1e-3
    X[rows // 2, 0] = float("nan")
    q, s = ops.quantize_rows(X)
    fine = torch.isfinite(X).all(-1)
    assert torch.isnan(s[~fine]).all() and not q[~fine].any() and int((~fine).sum()) == 2
    X, q, s = X[fine], q[fine], s[fine]
    assert torch.equal(s, (X.double().abs().amax(-1) / 127).float())
    want = torch.where(s.unsqueeze(-1) == 0, torch.zeros_like(X, dtype=torch.float32), X.float() / s.unsqueeze(-1)).round()
    assert torch.equal(q.float(), want)
    ops.check_status()


def test_quantize_rows_extremes(cuda_device):
    X = torch.zeros(6, 40, device="cuda")
    X[0, 3] = float("inf")
    X[1, 4] = float("nan")
    X[2] = torch.finfo(torch.float32).max
    X[3] = 1e-45                                           # the smallest number: its 127th part is 0
    X[4, :2] = torch.tensor([127.0, 2.5])
    X[4, 2] = -3.5
    q, s = ops.quantize_rows(X)
    assert torch.isnan(s[:2]).all() and (q[:2] == 0).all()
    assert (q[2] == 127).all() and s[3] == 0 and (q[3] == 0).all()
    assert q[4, :3].tolist() == [127, 2, -4] and s[4] == 1 and (q[5] == 0).all() and s[5] == 0
    wide = torch.randn(20, 3, 50, device="cuda")
    for t in (wide[:, 1], wide[:, :, 5:20], wide.transpose(0, 2), wide[::3]):
        a, b = ops.quantize_rows(t), ops.quantize_rows(t.contiguous())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(ValueError):
        ops.quantize_rows(wide.double())
    with pytest.raises(RuntimeError):
        ops.quantize_rows(wide.cpu())


INT8_SHAPES = [(1, 1, 1, 1, 1), (1, 8, 64, 256, 128), (2, 3, 5, 17, 9), (129, 1, 1, 72, 136), (150, 2, 4, 72, 100), (257, 2, 4, 128, 264), (500, 4, 13, 330, 201), (1000, 3, 8, 1024, 256), (3, 2, 300, 40, 24),
               (6, 4, 64, 264, 136), (4, 5, 64, 1001, 77), (30, 4, 64, 264, 136), (25, 5, 64, 1001, 77), (64, 2, 16, 4112, 70), (700, 8, 40, 512, 16)]


def int8_product(q, s, Wq, ws, ids, E, rows):
    """The integer sums are exact in float64 before they are scaled."""
    sums, _ = orc.matmul(q, Wq.transpose(1, 2), ids, E, rows)
    offsets, slots, _ = orc.plan(ids, E)
    expert = torch.bucketize(torch.arange(slots.numel(), device="cuda"), offsets[1:], right=True).clamp(max=E - 1)
    row_scale = s.double()[slots // ids.shape[-1]] if rows == "tokens" else s.double()
    return sums * row_scale.unsqueeze(-1) * ws.double()[expert]


def close8(got, ref):
    """The int32 sum is rounded to float32, then multiplied twice, then rounded; beyond float16's range there are infinities."""
    if got.dtype == torch.float16:
        ok = ref.abs() < 65520
        assert torch.equal(got[~ok].double(), torch.sign(ref[~ok]) * float("inf"))
        got, ref = got[ok], ref[ok]
    close(got, ref, torch.zeros_like(ref), 0)


@pytest.mark.parametrize("tokens,k,E,C,N", INT8_SHAPES)
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("kind", ["even", "holes"])
def test_int8_products(cuda_device, tokens, k, E, C, N, out_dtype, kind):
    g = gen(C * N)
    k = min(k, E)
    ids = draw_experts(g, tokens, k, E, kind)
    plan = ops.plan_experts(ids, E)
    draw8 = lambda *s: torch.randint(-128, 128, s, device="cuda", generator=g).to(torch.int8)
    Wq = draw8(E, N, C)
    ws = torch.rand(E, N, device="cuda", generator=g) + 0.5
    n_rows = {"tokens": tokens, "sorted": tokens * k}
    for rows in ("tokens", "sorted"):
        q, s = draw8(n_rows[rows], C), torch.rand(n_rows[rows], device="cuda", generator=g) + 0.5
        ref = int8_product(q, s, Wq, ws, ids, E, rows)
        for path in ("auto", "generic"):
            close8(ops.expert_matmul_int8(q, s, Wq, ws, plan, rows=rows, out_dtype=out_dtype, path=path), ref)
    if kind == "even":
        q, s = draw8(tokens, C), torch.rand(tokens, device="cuda", generator=g) + 0.5
        ref = (q.double() @ Wq[0].double().t()) * s.double().unsqueeze(-1) * ws[0].double()
        for path in ("auto", "generic"):
            got = ops.matmul_int8(q, s, Wq[0], ws[0], out_dtype=out_dtype, path=path)
            close8(got, ref)
    ops.check_status()


def test_int8_sums_are_exact(cuda_device):
    """Longest contraction, largest magnitudes: 131071 * 2^14 fits in 31 bits; the next longer one is refused."""
    C = 131071
    q, W = torch.full((2, C), -128, device="cuda", dtype=torch.int8), torch.full((3, C), -128, device="cuda", dtype=torch.int8)
    W[1] = 127
    one = lambda n: torch.ones(n, device="cuda")
    for path in ("auto", "generic"):
        y = ops.matmul_int8(q, one(2), W, one(3), out_dtype=torch.float32, path=path)
        assert torch.equal(y.double(), torch.tensor([C * 2.0 ** 14, -C * 128.0 * 127, C * 2.0 ** 14], device="cuda").float().double().expand(2, 3))
    with pytest.raises(ValueError):
        z = torch.zeros(2, C + 1, device="cuda", dtype=torch.int8)
        ops.matmul_int8(z, one(2), z, one(2))


def test_int8_views_and_refusals(cuda_device):
    g = gen(2)
    big = torch.randint(-128, 128, (40, 3, 130), device="cuda", generator=g).to(torch.int8)
    s, ws = torch.rand(40, device="cuda"), torch.rand(3, device="cuda")
    W = big[0, :, :64]
    for q in (big[:, 1, :64], big[:, 1, 1:65], big.transpose(0, 2)[:64, 2].t(), big[:, 2, ::2][:, :64]):
        assert torch.equal(ops.matmul_int8(q, s, W, ws), ops.matmul_int8(q.contiguous(), s, W.contiguous(), ws))
    q = big[:, 0, :64]
    assert torch.equal(ops.matmul_int8(q.reshape(8, 5, 64), s.view(8, 5), W, ws).view(40, 3), ops.matmul_int8(q, s, W, ws))
    for args in ((q.float(), s, W, ws), (q, s[:39], W, ws), (q, s, W[:, :63], ws), (q, s, W, ws[:2]), (q, s.half(), W, ws), (q, s, W.unsqueeze(0), ws)):
        with pytest.raises(ValueError):
            ops.matmul_int8(*args)
    with pytest.raises(ValueError):
        ops.matmul_int8(q, s, W, ws, out_dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.matmul_int8(q.cpu(), s, W, ws)


# ---- the layer -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_trains_and_is_served(cuda_device, dtype):
    g = gen(20)
    torch.manual_seed(2)
    E, I, J, k = 16, 128, 64, 4
    layer = RoutedExperts(E, I, J, k, balance=True, score="sigmoid", groups=4, top_groups=2).cuda().to(dtype)
    x = randn(g, 5, 60, I, dtype=dtype)
    out = layer(x)
    w, ids = layer.router(x)
    w, ids = w.view(-1, k).double(), ids.view(-1, k)
    xs = x.view(-1, I).double()
    ref = torch.zeros_like(xs)
    for j in range(k):
        h = torch.nn.functional.silu(torch.einsum("tc,tcn->tn", xs, layer.up.double()[ids[:, j].long()]))
        ref += w[:, j:j + 1] * torch.einsum("tc,tcn->tn", h, layer.down.double()[ids[:, j].long()])
    # the middle rows are rounded twice, the last once, before the sum
    assert out.shape == x.shape
    assert (out.view(-1, I).double() - ref).norm() <= (4 * HALF[dtype] + 1e-5) * ref.norm()
    layer.router.adjust(layer.plan, 0.01)
    assert layer.router.balance.shape == (E,) and layer.router.balance.abs().max() <= 0.011 and layer.router.balance.dtype == torch.float32
    other = RoutedExperts(E, I, J, k, balance=True).to(dtype)
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other.cuda().router.balance, layer.router.balance)
    out = layer(x)
    out.float().square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in layer.parameters())
    served = layer.quantized()
    for one in (x, x[0, :1], x[0, 0]):
        with torch.no_grad():
            full = layer(one)
        small = served(one)
        assert small.shape == one.shape and (small.double() - full.double()).norm() <= 0.04 * full.double().norm()
    ops.check_status()


def test_operators_on_another_stream_and_in_a_graph(cuda_device):
    g = gen(21)
    torch.manual_seed(3)
    layer = RoutedExperts(8, 64, 32, 2).cuda().bfloat16()
    served = layer.quantized()
    x = randn(g, 40, 64, dtype=torch.bfloat16)
    ref = served(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            out = served(x)
    side.synchronize()
    assert torch.equal(out, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = served(x)
    x.copy_(randn(g, 40, 64, dtype=torch.bfloat16))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, served(x))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_rows_beyond_two_to_the_31_elements(cuda_device, dtype):
    """70000 sorted rows of 32768: what lies at the end is compared (and a product whose weights end beyond 2^31 elements)."""
    g = gen(31)
    tokens, k, E, C, N = 17500, 4, 4, 64, 32768
    ids = torch.arange(k, device="cuda", dtype=torch.int32).repeat(tokens, 1)
    plan = ops.plan_experts(ids, E)
    X, W, w = randn(g, tokens, C, dtype=dtype), randn(g, E, C, N, dtype=dtype), torch.rand(tokens, k, device="cuda", generator=g)
    Y = ops.expert_matmul(X, W, plan)
    end = slice(tokens - 200, None)
    ref, size = X[end].double() @ W[3].double(), X[end].double().abs() @ W[3].double().abs()
    close(Y[-200:], ref, size, C)
    out = ops.combine(Y, w, plan)
    rows = Y.view(k, tokens, N)[:, end].double()                      # (every expert has the tokens in order)
    want = (rows * w[end].t().unsqueeze(-1).double()).sum(0)
    close(out[end], want, (rows.abs() * w[end].t().unsqueeze(-1).double()).sum(0), k)
    del rows, want
    dY, dw = ops.combine_backward(out, Y, w, plan)
    want = out[end].double() * w[end, 3:].double()
    close(dY[-200:], want, want.abs(), 1)
    want = (out[end].double() * Y[-200:].double()).sum(-1)
    assert ((dw[end, 3].double() - want).abs() <= N * 2.0 ** -24 * (out[end].double() * Y[-200:].double()).abs().sum(-1)).all()
    del out, Y
    dX = ops.expert_matmul(dY, W, plan, rows="sorted", w_layout="nc")
    close(dX[-200:], dY[-200:].double() @ W[3].double().t(), dY[-200:].double().abs() @ W[3].double().abs().t(), N)
    dW = ops.expert_dweight(X, dY, plan)
    last = dY[-tokens:, -300:].double()
    close(dW[3][:, -300:], X.double().t() @ last, X.double().abs().t() @ last.abs(), tokens)
    del dY, dX, dW, last
    E, C, N = 40, 8192, 8192                                          # (one row, and 300 rows of the last expert)
    W = torch.empty(E, C, N, device="cuda", dtype=dtype)
    W[-1] = randn(g, C, N, dtype=dtype)
    for n in (1, 300):
        X = randn(g, n, C, dtype=dtype)
        plan = ops.plan_experts(torch.full((n, 1), E - 1, device="cuda"), E)
        for layout in ("cn", "nc"):
            V = W[-1] if layout == "cn" else W[-1].t()
            close(ops.expert_matmul(X, W, plan, w_layout=layout), X.double() @ V.double(), X.double().abs() @ V.double().abs(), C)
    dW = ops.expert_dweight(X, X, plan)
    close(dW[-1, -100:], X[:, -100:].double().t() @ X.double(), X[:, -100:].double().abs().t() @ X.double().abs(), 300)
    assert not dW[:-1].any()
    ops.check_status()


def test_results_do_not_change_from_run_to_run(cuda_device):
    g = gen(22)
    ids = draw_experts(g, 3000, 4, 16, "skewed")
    X, W = randn(g, 3000, 256, dtype=torch.bfloat16), randn(g, 16, 256, 128, dtype=torch.bfloat16)
    w = torch.rand(3000, 4, device="cuda", generator=g)

    def once():
        plan = ops.plan_experts(ids, 16)
        Y = ops.expert_matmul(X, W, plan)
        dY, dw = ops.combine_backward(X[:, :128].contiguous(), Y, w, plan)
        return Y, ops.combine(Y, w, plan), dY, dw, ops.expert_dweight(X, dY, plan)

    first = once()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))
