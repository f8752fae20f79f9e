"""Operators for tokens that choose experts, where a call is at the edge of what it takes: plans made by hand, plans that lie elsewhere,
groups whose values are almost equal, weight gradients in every variant, second derivatives, casts of the served layer.

Tolerances are those of the tests of the operators: float32 sums of n products are off by at most (n + 2) * 2 * u times the sum of the
products' magnitudes (u = 2^-24), a rounding to 16 bits by half a unit.
"""
import ctypes

import pytest
import torch

from expertscattergather_b200 import RoutedExperts, _lib, ops, token_choice
from oracle import choice_oracle as orc
from test_gpu_token_choice import MATMUL_SHAPES, close, draw_experts

pytestmark = pytest.mark.gpu

DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


# ---- plans made by hand ----------------------------------------------------------------------------------

# rows of one vector, of 32, of more; rows that do not begin on 4 bytes; no columns
@pytest.mark.parametrize("tokens,N", [(5, 8), (7, 256), (3, 264), (300, 2048), (9, 4097), (1, 1), (4, 0), (0, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_without_a_choice(cuda_device, tokens, N, dtype):
    none = torch.empty(0, device="cuda", dtype=torch.int32)
    plan = ops.ExpertPlan(torch.zeros(5, device="cuda", dtype=torch.int32), none, none, tokens, 0, 4)
    Y = torch.empty(0, N, device="cuda", dtype=dtype)
    for weights in (None, torch.empty(tokens, 0, device="cuda")):
        torch.full((tokens, N), float("nan"), device="cuda", dtype=dtype)          # (what the output's memory held)
        out = ops.combine(Y, weights, plan)
        assert out.shape == (tokens, N) and out.dtype == dtype and not out.any()
        dY, dweights = ops.combine_backward(torch.ones(tokens, N, device="cuda", dtype=dtype), Y, weights, plan)
        assert dY.shape == (0, N) and (dweights is None if weights is None else dweights.shape == (tokens, 0))
    ops.check_status()


def test_plans_that_lie_elsewhere_are_refused(cuda_device):
    """Before any launch: no kernel gets their addresses."""
    E, k, tokens = 4, 2, 10
    ids = torch.arange(tokens * k, device="cuda", dtype=torch.int32).view(tokens, k) % E
    plan = ops.plan_experts(ids, E)
    arrays = (plan.offsets, plan.slots, plan.position)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dtype)
    ones = lambda *s: torch.ones(*s, device="cuda")
    q, Wq = z(tokens, 16, dtype=torch.int8), z(E, 8, 16, dtype=torch.int8)
    before = ops.launch_count()
    for away in ((0,), (1,), (2,), (0, 1, 2)):
        other = ops.ExpertPlan(*(a.cpu() if i in away else a for i, a in enumerate(arrays)), tokens, k, E)
        calls = [lambda: ops.combine(z(tokens * k, 8), None, other), lambda: ops.combine_backward(z(tokens, 8), z(tokens * k, 8), z(tokens, k), other)] if 2 in away else []
        if away != (2,):
            calls += [lambda: ops.expert_matmul(z(tokens, 8), z(E, 8, 8), other), lambda: ops.expert_matmul(z(tokens * k, 8), z(E, 8, 8), other, rows="sorted"),
                      lambda: ops.expert_dweight(z(tokens, 8), z(tokens * k, 8), other), lambda: ops.expert_matmul_int8(q, ones(tokens), Wq, ones(E, 8), other),
                      lambda: ops.expert_matmul_int8(z(tokens * k, 16, dtype=torch.int8), ones(tokens * k), Wq, ones(E, 8), other, rows="sorted")]
        for call in calls:
            with pytest.raises(RuntimeError):
                call()
    assert ops.launch_count() == before
    ops.expert_matmul_int8(q, ones(tokens), Wq, ones(E, 8), plan)
    ops.check_status()


# ---- groups whose values are almost equal -----------------------------------------------------------------

def kept_groups(key, groups, top_groups, group_top):
    value = orc.group_values(key, groups, group_top)
    kept = value.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
    return torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True), value


# logits around `at`, where the groups' differ by whole `step`s: scores of a few units' error tell them apart, those of a fast
# exponential (2 + 1.17 |x| units) need not; at -88 a fast reciprocal gives 0
@pytest.mark.parametrize("at,step", [(-6.0, 2.0 ** -19), (-15.0, 2.0 ** -19), (-30.0, 2.0 ** -19), (-60.0, 2.0 ** -18), (-80.0, 2.0 ** -17), (-88.0, 2.0 ** -17)])
@pytest.mark.parametrize("groups,per,top_groups", [(8, 32, 4), (6, 5, 1), (4, 15, 3), (2, 1, 1)])
def test_groups_of_low_scores_are_compared_exactly(cuda_device, at, step, groups, per, top_groups):
    """One score is off by at most 2 (exponential) + 1 (sum) + 1 (division) units: two values by 8 of 2^-23, 9.5e-7; a step changes a value
    by 2^-19 = 1.9e-6 at least."""
    g = gen(int(-at) + groups)
    tokens = 4000
    place = torch.stack([torch.randperm(groups, device="cuda", generator=g) for _ in range(tokens)]).float() * step
    base = at + torch.randint(0, 64, (tokens, 1), device="cuda", generator=g).float() * step
    logits = (base + place).unsqueeze(-1) - 0.25 * torch.rand(tokens, groups, per, device="cuda", generator=g).mul(64).floor().div(64) - 0.5
    where = torch.rand(tokens, groups, per, device="cuda", generator=g).topk(min(2, per), -1).indices
    logits.scatter_(2, where, (base + place).unsqueeze(-1).expand(-1, -1, where.shape[-1]))            # a group's best two
    logits = logits.view(tokens, groups * per)
    k = min(3, per * top_groups)
    weights, ids = ops.route_tokens(logits, k, score="sigmoid", groups=groups, top_groups=top_groups, group_top=2)
    kept, _ = kept_groups(orc.scores(logits, "sigmoid"), groups, top_groups, 2)
    assert kept.gather(1, ids.long() // per).all()
    # the best of the kept groups are chosen, by their logits
    masked = logits.masked_fill(~kept.repeat_interleave(per, 1), -float("inf"))
    assert torch.equal(ids.long(), masked.sort(dim=-1, descending=True, stable=True).indices[:, :k])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_top", [1, 2])
def test_groups_with_a_bias_are_compared_exactly(cuda_device, score, group_top):
    """Keys of 0.2 to 2 whose groups differ by steps of 2^-20.  A key is off by 4 units of a score below 1 and by half a unit of the key below
    2, 2^-21 + 2^-24 at most, less than half of what two steps make; values that lie closer are not looked at."""
    g = gen(group_top)
    tokens, groups, per, top_groups, k = 4000, 8, 32, 3, 6
    logits = torch.rand(tokens, groups, per, device="cuda", generator=g) * 0.5
    place = torch.stack([torch.randperm(groups, device="cuda", generator=g) for _ in range(tokens)])
    logits[..., 3] = 0.75 + 2.0 ** -17 * place
    logits[..., 7] = 0.75 + 2.0 ** -17 * place
    bias = torch.zeros(groups, per, device="cuda")
    bias[:, (3, 7)] = 0.5
    logits, bias = logits.view(tokens, -1), bias.flatten()
    _, ids = ops.route_tokens(logits, k, bias, score=score, groups=groups, top_groups=top_groups, group_top=group_top)
    kept, value = kept_groups(orc.scores(logits, score) + bias.double(), groups, top_groups, group_top)
    order = value.sort(-1, descending=True).values
    clear = order[:, top_groups - 1] - order[:, top_groups] > group_top * (2.0 ** -20 + 2.0 ** -22)
    if score == "sigmoid":                                 # (a softmax over 256 experts makes the steps smaller than a unit of the key)
        assert clear.float().mean() > 0.9
    assert kept.gather(1, ids.long() // per)[clear].all()


@pytest.mark.parametrize("with_bias", [False, True])
def test_groups_that_are_masked_or_equal(cuda_device, with_bias):
    """Groups of equal values: the lower ones.  A bias of -infinity takes experts, and whole groups, out of the choice."""
    tokens, groups, per = 70, 8, 4
    logits = torch.full((tokens, groups * per), -20.0, device="cuda")
    bias = torch.zeros(groups * per, device="cuda") if with_bias else None
    for group_top in (1, 2):
        _, ids = ops.route_tokens(logits, 6, bias, score="sigmoid", groups=groups, top_groups=3, group_top=group_top)
        assert torch.equal(ids, torch.arange(6, device="cuda", dtype=torch.int32).expand(tokens, 6))
        if not with_bias:
            continue
        masked = bias.clone()
        masked[:4 * per] = -float("inf")                   # four groups
        masked[6 * per:6 * per + 3] = -float("inf")        # all but one expert of another
        _, ids = ops.route_tokens(logits, 9, masked, score="sigmoid", groups=groups, top_groups=3, group_top=group_top)
        # (two experts of a group: the group with one left counts as lowest, with the masked ones)
        want = [*range(4 * per, 6 * per), 6 * per + 3] if group_top == 1 else [*range(4 * per, 6 * per), 7 * per]
        assert torch.equal(ids, torch.tensor(want, device="cuda", dtype=torch.int32).expand(tokens, 9))
    ops.check_status()


# ---- the served layer --------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("I,J", [(64, 48), (72, 40)])
def test_served_layer_after_casts_and_moves(cuda_device, dtype, I, J):
    torch.manual_seed(0)
    layer = RoutedExperts(8, I, J, 2, balance=True).cuda()
    x = randn(gen(1), 30, I)
    served, full = layer.quantized(), layer(x).detach()
    small = served(x)
    assert (small - full).norm() <= 0.04 * full.norm()
    moved = layer.quantized().cpu().cuda()
    assert torch.equal(moved(x), small)
    cast = layer.quantized().to(dtype)
    assert layer.router.W.dtype == torch.float32 and torch.equal(layer(x), full)
    out = cast(x.to(dtype))
    assert out.dtype == dtype and (out.float() - full).norm() <= 0.06 * full.norm()
    with torch.no_grad():
        layer.router.W.neg_()
    assert torch.equal(served(x), small)
    assert moved.up.stride(-2) % 16 == 0 and moved.down.stride(-2) % 16 == 0
    ops.check_status()


# ---- under autograd and torch.compile ----------------------------------------------------------------------

def test_second_derivatives_are_refused(cuda_device):
    """They are not implemented; a graph of first gradients may be made, and says so where it is differentiated."""
    g = gen(2)
    logits, X, W = (t.requires_grad_(True) for t in (randn(g, 20, 6), randn(g, 20, 8), randn(g, 6, 8, 4)))
    weights, ids = token_choice.route_tokens(logits, 2)
    plan = ops.plan_experts(ids, 6)
    Y = randn(g, 40, 4).requires_grad_(True)
    for out, leaf in ((weights, logits), (token_choice.expert_matmul(X, W, plan), X), (token_choice.combine(Y, weights.detach(), plan), Y)):
        first, = torch.autograd.grad(out.square().sum(), leaf, create_graph=True, retain_graph=True)
        plain, = torch.autograd.grad(out.square().sum(), leaf, retain_graph=True)
        assert torch.equal(first, plain) and not plain.requires_grad
        # (a penalty on the gradient beside another term of the leaf: without the refusal its part would be missing in silence)
        with pytest.raises(RuntimeError):
            (first.square().sum() + leaf.square().sum()).backward()


def test_compiled_layer(cuda_device):
    torch.manual_seed(0)
    layer = RoutedExperts(8, 64, 32, 2).cuda()
    x = randn(gen(3), 50, 64)
    ref = layer(x)
    ref.square().sum().backward()
    grads = [p.grad.clone() for p in layer.parameters()]
    layer.zero_grad()
    out = torch.compile(layer)(x)
    out.square().sum().backward()
    # (what lies between the operators, SiLU above all, may be rounded otherwise)
    assert torch.allclose(out, ref, rtol=1e-5, atol=1e-6)
    for p, g in zip(layer.parameters(), grads):
        assert torch.allclose(p.grad, g, rtol=1e-4, atol=1e-5)
    served = layer.quantized()
    assert torch.allclose(torch.compile(served)(x), served(x), rtol=0.02, atol=1e-3)
    ops.check_status()


# ---- the C entries -----------------------------------------------------------------------------------------

TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def shifted(t, by):
    """A copy that begins `by` elements into its storage."""
    store = torch.empty(t.numel() + by + 16, device="cuda", dtype=t.dtype)
    return store[by:by + t.numel()].view(t.shape).copy_(t)


# where a kernel stores several elements together it has to look at where the output begins: the first expert of these is cut into ranges,
# in the last one a range is a whole expert
@pytest.mark.parametrize("by", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("tokens,E,C,N", [(7000, 2, 64, 64), (7000, 2, 33, 36), (7000, 2, 35, 33), (60, 6, 64, 72)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_entries_take_outputs_that_begin_anywhere(cuda_device, by, tokens, E, C, N, dtype):
    lib, g, k = _lib.load(), gen(by + C), 2
    ids = torch.rand(tokens, E, device="cuda", generator=g).topk(k, -1).indices.int()
    plan = ops.plan_experts(ids, E)
    X, W, dY = randn(g, tokens, C, dtype=dtype), randn(g, E, C, N, dtype=dtype), randn(g, tokens * k, N, dtype=dtype)
    dims = ctypes.byref(_lib.Ragged(tokens, k, E, C, N))
    at = lambda t: ctypes.c_void_p(t.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    space = lambda n: (torch.empty(max(n, 16), device="cuda", dtype=torch.uint8), n)
    nan = lambda t: shifted(torch.full_like(t, float("nan")), by)

    Y = ops.expert_matmul(X, W, plan)
    got, (ws, n) = nan(Y), space(lib.egs_expert_matmul_workspace_bytes(dims, 0, 0, TYPES[dtype]))
    assert lib.egs_expert_matmul(at(X), at(W), at(plan.offsets), at(plan.slots), at(got), dims, 0, 0, TYPES[dtype], 0, at(ws), n, None, stream) == _lib.OK
    assert torch.equal(got, Y)
    dW = ops.expert_dweight(X, dY, plan)
    got, (ws, n) = nan(dW), space(lib.egs_expert_dweight_workspace_bytes(dims, 0, TYPES[dtype]))
    assert lib.egs_expert_dweight(at(X), at(dY), at(plan.offsets), at(plan.slots), at(got), dims, 0, TYPES[dtype], 0, at(ws), n, None, stream) == _lib.OK
    assert torch.equal(got, dW)
    w = torch.rand(tokens, k, device="cuda", generator=g)
    out = ops.combine(Y, w, plan)
    got = nan(out)
    assert lib.egs_combine(at(shifted(Y, by)), at(w), at(plan.position), at(got), tokens, k, N, TYPES[dtype], _lib.F32, stream) == _lib.OK
    # (the columns of a row are summed in the order of the choices whatever the vectors are)
    assert torch.equal(got, out)
    gY, gw = ops.combine_backward(out, Y, w, plan)
    got, got_w = nan(gY), torch.full_like(gw, float("nan"))
    assert lib.egs_combine_backward(at(shifted(out, by)), at(shifted(Y, by)), at(w), at(plan.position), at(got), at(got_w), tokens, k, N, TYPES[dtype],
                                    _lib.F32, stream) == _lib.OK
    assert torch.equal(got, gY)
    size = (out.double()[:, None] * Y.double()[plan.position.long()].view(tokens, k, N)).abs().sum(-1)
    assert ((got_w.double() - gw.double()).abs() <= 2 * (N + 2) * 2.0 ** -24 * size).all()         # (another order of a float32 sum)
    ops.check_status()


# ---- as many rows as there can be --------------------------------------------------------------------------

def test_rows_up_to_the_limit(cuda_device):
    """One expert of 2^31 - 4096 rows of one element."""
    n = (1 << 31) - 4096
    X = torch.ones(n, 1, device="cuda")
    slots = torch.zeros(n, device="cuda", dtype=torch.int32)                   # (sorted rows: nobody reads them)
    plan = ops.ExpertPlan(torch.tensor([0, n], device="cuda", dtype=torch.int32), slots, slots[:0], n, 1, 1)
    # sums of at most 3.7 million ones are exact; the ranges' (at most 592 + 1) are added one after the other
    dW = ops.expert_dweight(X, X, plan, rows="sorted")
    assert abs(dW.item() - n) <= 593 * 2.0 ** -24 * n
    Y = ops.expert_matmul(X, torch.full((1, 1, 1), 2.0, device="cuda"), plan, rows="sorted")
    assert Y[-5000:].eq(2).all() and Y[::4097].eq(2).all()
    ops.check_status()
    del X, Y, slots
    torch.cuda.empty_cache()


# a row for each of many experts, and more that are not routed: grids of more than 2^31 threads, which share the zeros among themselves
@pytest.mark.parametrize("dtype,E,N", [(torch.float32, 1024, 270000), (torch.bfloat16, 512, 1600000)])
def test_zeros_of_wide_rows(cuda_device, dtype, E, N):
    g = gen(N)
    tokens = E // 6 if dtype != torch.float32 else E
    ids = torch.stack([torch.randperm(E, device="cuda", generator=g)[:tokens], torch.full((tokens,), -1, device="cuda")], -1)
    ids[::5, 0] = -1
    plan = ops.plan_experts(ids, E)
    X, W = randn(g, tokens, 1, dtype=dtype), torch.rand(E, 1, N, device="cuda", generator=g).to(dtype)
    torch.full((tokens * 2, N), float("nan"), device="cuda", dtype=dtype)          # (what the output's memory held)
    for w, layout in ((W, "cn"), (W.view(E, N, 1), "nc")):
        Y = ops.expert_matmul(X, w, plan, w_layout=layout)
        routed = plan.offsets[E].item()
        assert not Y[routed:].any()
        # one product, rounded once
        slots = plan.slots[:routed].long()
        experts = ids.flatten()[slots]
        for r in range(0, routed, 64):
            part = slice(r, min(r + 64, routed))
            assert torch.equal(Y[part], (X[slots[part] // 2].float() * W[experts[part], 0].float()).to(dtype))
    ops.check_status()
    del X, W, Y
    torch.cuda.empty_cache()


# more column tiles than a grid's second dimension holds; few rows an expert, a block of 128 of them, tens
@pytest.mark.parametrize("tokens,E", [(40, 2), (200, 1), (2, 9)])
@pytest.mark.parametrize("dtype,path", [(torch.float32, "auto"), (torch.bfloat16, "generic"), (torch.bfloat16, "auto")])
def test_columns_beyond_65535_tiles(cuda_device, tokens, E, dtype, path):
    g, N = gen(tokens), 65535 * 64 + 72
    ids = torch.randint(0, E, (tokens, 1), device="cuda", generator=g)
    ids[1] = -1
    plan = ops.plan_experts(ids, E)
    X, W = randn(g, tokens, 1, dtype=dtype), torch.rand(E, 1, N, device="cuda", generator=g).to(dtype)
    for w, layout in ((W, "cn"), (W.view(E, N, 1), "nc")):
        Y = ops.expert_matmul(X, w, plan, w_layout=layout, path=path)
        assert not Y[-1].any()
        for r, slot in enumerate(plan.slots[:-1].tolist()):
            assert torch.equal(Y[r], (X[slot].float() * W[ids[slot, 0], 0].float()).to(dtype))
        del Y
    q = torch.ones(tokens, 16, device="cuda", dtype=torch.int8)
    Wq = torch.randint(-9, 9, (N, 16), device="cuda", generator=g).to(torch.int8)
    one = torch.ones(N, device="cuda")
    assert torch.equal(ops.matmul_int8(q, one[:tokens], Wq, one, out_dtype=torch.float32, path=path), Wq.sum(-1).float().expand(tokens, N))
    ops.check_status()
    torch.cuda.empty_cache()


def test_a_refused_launch_is_reported_once(cuda_device):
    """Columns of more tiles than a grid's second dimension holds: the launch is refused, and the next operator has nothing to do with it."""
    N = 1 << 24
    X, W = torch.ones(1, 4, 1, device="cuda"), torch.ones(1, 1, N, device="cuda")
    with pytest.raises(RuntimeError, match="invalid"):
        ops.gather_gemm(X, W, torch.zeros(1, 1, 1, device="cuda", dtype=torch.int32), path="generic")
    assert (X + 1).sum().item() == 8
    ops.check_status()


# ---- float32 rows of 16-bit tensors ------------------------------------------------------------------------

@pytest.mark.parametrize("tokens,k,E,C,N", MATMUL_SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_rows(cuda_device, tokens, k, E, C, N, dtype):
    """Products without a rounding, and their weighted sums with one."""
    g, k = gen(C + N), min(k, E)
    for kind in ("even", "holes"):
        ids = draw_experts(g, tokens, k, E, kind)
        plan = ops.plan_experts(ids, E)
        W = randn(g, E, C, N, dtype=dtype)
        for rows, x in (("tokens", randn(g, tokens, C, dtype=dtype)), ("sorted", randn(g, tokens * k, C, dtype=dtype))):
            ref, size = orc.matmul(x, W, ids, E, rows)
            for path in ("auto", "generic"):
                for layout, w in (("cn", W), ("nc", W.transpose(1, 2).contiguous())):
                    Y = ops.expert_matmul(x, w, plan, rows=rows, w_layout=layout, path=path, out_dtype=torch.float32)
                    assert Y.dtype == torch.float32
                    close(Y, ref, size, C)
            assert torch.equal(ops.expert_matmul(x, W, plan, rows=rows, out_dtype=dtype), ops.expert_matmul(x, W, plan, rows=rows))
            for weights in (None, torch.rand(tokens, k, device="cuda", generator=g), torch.rand(tokens, k, device="cuda", generator=g).to(dtype)):
                out = ops.combine(Y, weights, plan, out_dtype=dtype)
                assert out.dtype == dtype
                want, many = orc.combine(Y, weights, plan.position, tokens, k)
                close(out, want, many, k)
                # the chain: sums of k * C products, one rounding
                many, _ = orc.combine(size, None if weights is None else weights.abs(), plan.position, tokens, k)
                want, _ = orc.combine(ref, weights, plan.position, tokens, k)
                close(out, want, many, C + k)
    ops.check_status()


# rows of 1 to 40 vectors, many of them and few
@pytest.mark.parametrize("tokens,k,N", [(1, 1, 1), (1, 8, 512), (7, 3, 13), (300, 4, 200), (129, 32, 8), (1000, 2, 1032), (20000, 4, 8), (50001, 2, 3), (2000, 4, 2048)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_combine_of_float32_rows(cuda_device, tokens, k, N, dtype):
    g = gen(N)
    ids = draw_experts(g, tokens, k, max(40, k), "holes")
    plan = ops.plan_experts(ids, max(40, k))
    Y = randn(g, tokens * k, N)
    Y[plan.offsets[-1].item():] = float("nan")
    for weights in (None, torch.rand(tokens, k, device="cuda", generator=g), torch.rand(tokens, k, device="cuda", generator=g).to(dtype)):
        ref, size = orc.combine(Y, weights, plan.position, tokens, k)
        close(ops.combine(Y, weights, plan, out_dtype=dtype), ref, size, k)
    none = ops.ExpertPlan(plan.offsets * 0, plan.slots[:0], plan.position[:0], tokens, 0, max(40, k))
    out = ops.combine(Y[:0], None, none, out_dtype=dtype)
    assert out.dtype == dtype and out.shape == (tokens, N) and not out.any()


def test_float32_rows_are_refused_where_they_are_not_made(cuda_device):
    ids = draw_experts(gen(1), 10, 2, 4)
    plan = ops.plan_experts(ids, 4)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dtype)
    for out in (torch.float16, torch.float64, torch.int8):
        with pytest.raises(ValueError):
            ops.expert_matmul(z(10, 8), z(4, 8, 8), plan, out_dtype=out)
        with pytest.raises(ValueError):
            ops.combine(z(20, 8), None, plan, out_dtype=out)
    with pytest.raises(ValueError):
        ops.expert_matmul(z(10, 8, dtype=torch.float32), z(4, 8, 8, dtype=torch.float32), plan, out_dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.combine(z(20, 8), None, plan, out_dtype=torch.float32)
    with pytest.raises(ValueError):
        ops.combine(z(20, 8, dtype=torch.float32), z(10, 2, dtype=torch.float16), plan, out_dtype=torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_through_float32_rows(cuda_device, dtype):
    g = gen(5)
    tokens, k, E, C, N = 300, 4, 8, 72, 136
    ids = draw_experts(g, tokens, k, E)
    plan = ops.plan_experts(ids, E)
    X, W, w = (t.requires_grad_(True) for t in (randn(g, tokens, C, dtype=dtype), randn(g, E, C, N, dtype=dtype), torch.rand(tokens, k, device="cuda", generator=g).to(dtype)))
    dOut = randn(g, tokens, N, dtype=dtype)
    Y = token_choice.expert_matmul(X, W, plan, out_dtype=torch.float32)
    out = token_choice.combine(Y, w, plan, out_dtype=dtype)
    assert Y.dtype == torch.float32 and out.dtype == dtype
    out.backward(dOut)
    assert all(t.grad.dtype == dtype for t in (X, W, w))
    # dY is rounded to the tensors' type, once (a product of two of them: exact in float64), and multiplied as it is
    slots = plan.slots.long()
    dY = (dOut.double()[slots // k] * w.detach().double().flatten()[slots].unsqueeze(-1)).to(dtype)
    ref, size = orc.matmul(dY, W.detach().transpose(1, 2), ids, E, "sorted")
    ref, _ = orc.combine(ref, None, plan.position, tokens, k)
    size, _ = orc.combine(size, None, plan.position, tokens, k)
    close(X.grad, ref, size, N + k)
    ref, size = orc.dweight(X.detach(), dY, ids, E, "tokens")
    close(W.grad, ref, size, int(plan.counts().max()))
    rows = Y.detach().double()[plan.position.long()].view(tokens, k, N)
    ref = (rows * dOut.double().unsqueeze(1)).sum(-1)
    close(w.grad, ref, (rows * dOut.double().unsqueeze(1)).abs().sum(-1), N)
    # without the rounding of dY: the gradient of the token rows, gathered, times the weights, summed in float32, rounded once
    dX = ops.combine(ops.expert_matmul(dOut, W.detach(), plan, w_layout="nc", out_dtype=torch.float32), w.detach(), plan, out_dtype=dtype)
    ref, size = orc.matmul(dOut, W.detach().transpose(1, 2), ids, E, "tokens")
    ref, _ = orc.combine(ref, w.detach(), plan.position, tokens, k)
    size, _ = orc.combine(size, w.detach(), plan.position, tokens, k)
    close(dX, ref, size, N + k)
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_with_float32_rows(cuda_device, dtype):
    g = gen(6)
    errors = {}
    for wide in (False, True):
        torch.manual_seed(3)
        layer = RoutedExperts(16, 128, 96, 4, float32_rows=wide).cuda().to(dtype)
        x = randn(gen(7), 400, 128, dtype=dtype).requires_grad_(True)
        weights, ids = layer.router(x)
        out = layer(x)
        dOut = randn(gen(8), 400, 128, dtype=dtype)
        out.backward(dOut)
        xs = x.detach().double().requires_grad_(True)
        logits = xs @ layer.router.W.detach().double().t()
        p = torch.softmax(logits, -1).gather(1, ids.long())
        p = p / p.sum(-1, keepdim=True)
        ref = 0
        for j in range(4):
            h = torch.nn.functional.silu(torch.einsum("tc,tcn->tn", xs, layer.up.detach().double()[ids[:, j].long()]))
            ref = ref + p[:, j:j + 1] * torch.einsum("tc,tcn->tn", h, layer.down.detach().double()[ids[:, j].long()])
        ref.backward(dOut.double())
        errors[wide] = [((a.double() - b).norm() / b.norm()).item() for a, b in ((out, ref.detach()), (x.grad, xs.grad))]
        served = layer.quantized()
        assert served.float32_rows == wide and (served(x).double() - ref.detach()).norm() <= 0.05 * ref.norm()
    assert all(a < b for a, b in zip(errors[True], errors[False])), errors
    ops.check_status()


# ---- variants that sizes choose ----------------------------------------------------------------------------

def experts_of(counts, k, g):
    """Ids of sum(counts) slots in a random order, so many of each expert, -1 for the rest of the last token."""
    ids = torch.arange(len(counts), device="cuda").repeat_interleave(torch.tensor(counts, device="cuda"))
    ids = torch.cat([ids, ids.new_full((-len(ids) % k,), -1)])
    return ids[torch.randperm(len(ids), device="cuda", generator=g)].view(-1, k).int()


# rows of the experts; cut into ranges: those of more than 24 steps of 64 rows, on pairs where X has more than 128 features
LONG = {"one": [5000], "three": [1700, 2000, 4100], "even": [1601] * 40, "skewed": [9000, 1, 0, 700, 2600, 64], "empty first": [0, 0, 6401, 1537]}


@pytest.mark.parametrize("counts", LONG.values(), ids=LONG.keys())
@pytest.mark.parametrize("C,N", [(64, 64), (64, 200), (256, 64), (256, 200), (131, 67), (35, 33), (300, 520)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradients_of_long_experts(cuda_device, counts, C, N, dtype):
    g, k = gen(C + N), 2
    ids = experts_of(counts, k, g)
    E, tokens = len(counts), len(ids)
    plan = ops.plan_experts(ids, E)
    dY = randn(g, tokens * k, N, dtype=dtype)
    for rows, n in (("tokens", tokens), ("sorted", tokens * k)):
        X = randn(g, n, C, dtype=dtype)
        ref, size = orc.dweight(X, dY, ids, E, rows)
        for path in ("auto", "generic"):
            dW = ops.expert_dweight(X, dY, plan, rows=rows, path=path)
            close(dW, ref, size, max(counts))
            assert not any(dW[e].any() for e, c in enumerate(counts) if c == 0)
    ops.check_status()


# more experts than a CTA has threads: the tables of blocks and of ranges take two turns
@pytest.mark.parametrize("E", [513, 700, 1024])
@pytest.mark.parametrize("C,N", [(64, 72), (200, 264)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_products_of_many_experts(cuda_device, E, C, N, dtype):
    g, tokens, k = gen(E + C), 1500, 3
    ids = draw_experts(g, tokens, k, E, "skewed")
    ids[:, 2] = E - 1                                      # one of many rows, behind the first turn
    ids[ids[:, 0] == E - 1, 0] = -1
    ids[ids[:, 1] == E - 1, 1] = -1
    plan = ops.plan_experts(ids, E)
    X, W, dY = randn(g, tokens, C, dtype=dtype), randn(g, E, C, N, dtype=dtype), randn(g, tokens * k, N, dtype=dtype)
    ref, size = orc.matmul(X, W, ids, E, "tokens")
    for layout, w in (("cn", W), ("nc", W.transpose(1, 2).contiguous())):
        close(ops.expert_matmul(X, w, plan, w_layout=layout), ref, size, C)
    ref, size = orc.dweight(X, dY, ids, E, "tokens")
    close(ops.expert_dweight(X, dY, plan), ref, size, tokens)
    q = torch.randint(-127, 128, (tokens, C), device="cuda", generator=g).to(torch.int8)
    Wq = torch.randint(-127, 128, (E, N, C), device="cuda", generator=g).to(torch.int8)
    Y = ops.expert_matmul_int8(q, torch.ones(tokens, device="cuda"), Wq, torch.ones(E, N, device="cuda"), plan, out_dtype=torch.float32)
    ref, _ = orc.matmul(q, Wq.transpose(1, 2), ids, E, "tokens")
    assert torch.equal(Y.double(), ref)                    # sums below 2^24
    ops.check_status()


@pytest.mark.parametrize("tokens,k,E,C,N", [(300, 2, 6, 128, 192), (9, 2, 6, 128, 192), (301, 3, 5, 130, 67), (5000, 2, 3, 264, 136)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sorted_rows_of_an_expert_stay_with_it(cuda_device, tokens, k, E, C, N, dtype):
    """Infinities in the sorted rows of one expert, NaN in rows that are not routed: products and gradients of the others are the same bits."""
    g = gen(C)
    ids = draw_experts(g, tokens, k, E, "even")
    ids[::7, 0] = -1
    plan = ops.plan_experts(ids, E)
    X, W, dY = randn(g, tokens * k, C, dtype=dtype), randn(g, E, N, C, dtype=dtype), randn(g, tokens * k, N, dtype=dtype)
    bad = 1
    a, b, end = plan.offsets[bad].item(), plan.offsets[bad + 1].item(), plan.offsets[E].item()
    Xn, Yn = X.clone(), dY.clone()
    Xn[a:b], Xn[end:] = float("inf"), float("nan")
    Yn[a:b], Yn[end:] = float("-inf"), float("nan")
    rows = torch.ones(tokens * k, dtype=torch.bool, device="cuda")
    rows[a:b] = False
    others = torch.arange(E, device="cuda") != bad
    for path in ("auto", "generic"):
        ref, got = (ops.expert_matmul(x, W, plan, rows="sorted", w_layout="nc", path=path) for x in (X, Xn))
        assert torch.equal(ref[rows], got[rows]) and not got[end:].any() and not torch.isfinite(got[a:b]).any()
        ref, got = (ops.expert_dweight(x, y, plan, rows="sorted", path=path) for x, y in ((X, dY), (Xn, Yn)))
        assert torch.equal(ref[others], got[others]) and (a == b or not torch.isfinite(got[bad]).any())
    ops.check_status()
