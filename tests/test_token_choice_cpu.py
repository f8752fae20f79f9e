"""What the operators for tokens that choose experts check before they touch a GPU, and their oracle against plain loops."""
import ctypes

import pytest
import torch

import expertscattergather_b200 as egs
from expertscattergather_b200 import _lib, ops
from oracle import choice_oracle as orc

BAD, LARGE, WORKSPACE = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_TOO_LARGE, _lib.ERR_WORKSPACE
one = ctypes.c_void_p(16)          # a pointer that is never followed: every call here is refused or has nothing to do


def route(tokens=4, E=8, top_k=2, groups=1, top_groups=1, group_top=2, score=0, renormalize=1, scale=1.0):
    return ctypes.byref(_lib.Route(tokens, E, top_k, groups, top_groups, group_top, score, renormalize, scale))


@pytest.mark.parametrize("spec,code", [({"E": 0}, BAD), ({"top_k": 0}, BAD), ({"top_k": 9}, BAD), ({"groups": 3}, BAD), ({"groups": 4, "top_groups": 5}, BAD),
                                       ({"groups": 4, "top_groups": 0}, BAD), ({"groups": 4, "top_k": 3}, BAD), ({"group_top": 0}, BAD), ({"score": 2}, BAD),
                                       ({"tokens": -1}, BAD), ({"E": 1025}, LARGE), ({"E": 64, "top_k": 33}, LARGE), ({"E": 66, "groups": 33}, LARGE),
                                       ({"tokens": 1 << 31}, LARGE), ({"tokens": 0}, _lib.OK)])
def test_route_entry(spec, code):
    lib = _lib.load()
    assert lib.egs_route_tokens(one, None, one, one, route(**spec), 8, _lib.F32, None) == code


def test_route_entry_pointers_and_types():
    lib = _lib.load()
    assert lib.egs_route_tokens(one, None, one, one, None, 8, _lib.F32, None) == BAD
    assert lib.egs_route_tokens(one, None, one, one, route(), 8, 3, None) == BAD
    assert lib.egs_route_tokens(one, None, one, one, route(), -1, _lib.F32, None) == BAD
    for hole in range(3):
        args = [one, one, one]
        args[hole] = None
        assert lib.egs_route_tokens(args[0], None, args[1], args[2], route(), 8, _lib.F32, None) == BAD
        assert lib.egs_route_tokens_backward(one, args[0], args[1], args[2], route(), 8, _lib.F32, None) == BAD
    assert lib.egs_route_tokens_backward(one, one, one, one, route(tokens=0), 8, _lib.F32, None) == _lib.OK
    assert lib.egs_route_tokens_backward(one, one, one, one, route(top_k=33, E=64), 8, _lib.F32, None) == LARGE


def test_plan_entry_and_its_workspace():
    lib = _lib.load()
    assert lib.egs_plan_experts(one, 4, 0, one, one, one, None, 0, None, None) == BAD
    assert lib.egs_plan_experts(one, 4, 1025, one, one, one, None, 0, None, None) == LARGE
    assert lib.egs_plan_experts(one, 1 << 31, 4, one, one, one, None, 0, None, None) == LARGE
    assert lib.egs_plan_experts(None, 4, 4, one, one, one, None, 0, None, None) == BAD
    for n in (0, 2048, 2049, 65536):                       # (one launch: nothing between two)
        assert lib.egs_plan_workspace_bytes(n, 64) == 0
    need = lib.egs_plan_workspace_bytes(65537, 64)
    assert need == 33 * 65 * 4
    assert lib.egs_plan_experts(one, 65537, 64, one, one, one, one, need - 1, None, None) == WORKSPACE


def ragged(tokens=10, k=2, E=4, C=8, N=8):
    return ctypes.byref(_lib.Ragged(tokens, k, E, C, N))


@pytest.mark.parametrize("dims,code", [({"tokens": -1}, BAD), ({"E": 0}, BAD), ({"E": 1025}, LARGE), ({"tokens": 1 << 30, "k": 4}, LARGE), ({"C": (1 << 24) + 1}, LARGE),
                                       ({"N": (1 << 24) + 1}, LARGE), ({"tokens": 0}, _lib.OK), ({"N": 0}, _lib.OK)])
def test_product_entries(dims, code):
    lib = _lib.load()
    for dtype in (_lib.F32, _lib.BF16):
        assert lib.egs_expert_matmul(one, one, one, one, one, ragged(**dims), 0, 0, dtype, 0, None, 0, None, None) == code
    if dims.get("tokens") != 0:
        assert lib.egs_expert_dweight(one, one, one, one, one, ragged(**dims), 0, _lib.F32, 0, None, 0, None, None) == code
    assert lib.egs_expert_matmul_int8(one, one, 1 << 24, one, one, 1 << 24, one, one, one, ragged(**dims), 0, _lib.F32, 0, None, None) == (LARGE if dims.get("C", 0) > 8 else code)


def test_product_entries_enums_and_pointers():
    lib = _lib.load()
    for rows, layout, dtype, path in ((2, 0, 0, 0), (0, 2, 0, 0), (0, 0, 3, 0), (0, 0, 0, 3)):
        assert lib.egs_expert_matmul(one, one, one, one, one, ragged(), rows, layout, dtype, path, None, 0, None, None) == BAD
    for hole in range(5):
        a = [one] * 5
        a[hole] = None
        assert lib.egs_expert_matmul(*a, ragged(), 0, 0, 0, 0, None, 0, None, None) == BAD
    assert lib.egs_expert_matmul_int8(one, one, 7, one, one, 8, one, one, one, ragged(), 0, 0, 0, None, None) == BAD         # rows overlap
    assert lib.egs_expert_matmul_int8(one, one, 8, one, one, 8, None, one, one, ragged(), 0, 0, 0, None, None) == BAD        # one expert has one choice
    assert lib.egs_expert_matmul_int8(one, one, 1 << 17, one, one, 1 << 17, one, one, one, ragged(C=1 << 17), 0, 0, 0, None, None) == LARGE
    assert lib.egs_combine(one, one, one, one, 4, 2, 8, _lib.F16, _lib.BF16, None) == BAD
    assert lib.egs_combine(one, one, None, one, 4, 2, 8, _lib.F16, _lib.F32, None) == BAD
    assert lib.egs_combine_backward(one, None, one, one, one, one, 4, 2, 8, _lib.F16, _lib.F32, None) == BAD
    assert lib.egs_combine_backward(one, one, one, one, one, one, 0, 2, 8, _lib.F16, _lib.F32, None) == _lib.OK
    assert lib.egs_quantize_rows(one, one, one, 4, 8, 8, 7, _lib.F32, None) == BAD
    assert lib.egs_quantize_rows(one, one, one, 0, 8, 8, 8, _lib.F32, None) == _lib.OK


def test_workspaces_of_products():
    """Copies of 16-bit operands whose rows do not begin on 16 bytes; ranges of a weight gradient."""
    lib = _lib.load()
    q = lambda d, rows, layout, dtype: lib.egs_expert_matmul_workspace_bytes(d, rows, layout, dtype)
    assert q(ragged(C=64, N=72), 0, 0, _lib.BF16) == 0
    assert q(ragged(C=63, N=71), 0, 0, _lib.F32) == 0
    assert q(ragged(C=63, N=72), 0, 0, _lib.BF16) == 10 * 64 * 2
    assert q(ragged(C=63, N=72), 1, 0, _lib.BF16) == 20 * 64 * 2
    assert q(ragged(C=64, N=71), 0, 0, _lib.BF16) == 4 * 64 * 72 * 2
    assert q(ragged(C=63, N=71), 0, 1, _lib.BF16) == 10 * 64 * 2 + 4 * 71 * 64 * 2
    for dtype in (_lib.F32, _lib.BF16):
        big = lib.egs_expert_dweight_workspace_bytes(ragged(tokens=100000, k=4, C=256, N=256), 0, dtype)
        assert 0 < big < 256 << 20
        assert lib.egs_expert_dweight_workspace_bytes(ragged(tokens=0), 0, dtype) == 0


def test_python_refuses_cpu_tensors_and_bad_words():
    x = torch.zeros(4, 8)
    with pytest.raises((RuntimeError, ValueError)):
        ops.route_tokens(x, 2)
    with pytest.raises(ValueError):
        ops.route_tokens(x, 2, score="relu")
    with pytest.raises(ValueError):
        ops.plan_experts(torch.zeros(4, 0, dtype=torch.int32), 4)
    with pytest.raises(RuntimeError):
        egs.TokenRouter(4, 8, 2).adjust(None, 0.1)


def test_router_balance_stays_float32():
    router = egs.TokenRouter(4, 8, 2, balance=True).to(torch.bfloat16)
    assert router.W.dtype == torch.bfloat16 and router.balance.dtype == torch.float32
    assert "balance" in router.state_dict() and "balance" not in egs.TokenRouter(4, 8, 2).state_dict()


def test_oracle_against_loops():
    gen = torch.Generator().manual_seed(0)
    tokens, k, E, C, N = 13, 3, 5, 4, 6
    ids = torch.stack([torch.randperm(E, generator=gen)[:k] for _ in range(tokens)])
    ids[2, 1] = -1
    X, W, w = torch.randn(tokens, C, generator=gen), torch.randn(E, C, N, generator=gen), torch.rand(tokens, k, generator=gen)
    offsets, slots, position = orc.plan(ids, E)
    rows = [(t, j) for e in range(E) for t in range(tokens) for j in range(k) if ids[t, j] == e]
    assert [t * k + j for t, j in rows] == slots[:len(rows)].tolist() and slots[len(rows):].tolist() == [2 * k + 1]
    assert offsets.tolist() == [sum(ids.flatten().eq(f).sum().item() for f in range(e)) for e in range(E + 1)]
    Y, _ = orc.matmul(X, W, ids, E, "tokens")
    for r, (t, j) in enumerate(rows):
        assert torch.allclose(Y[r], X[t].double() @ W[ids[t, j]].double()) and position[t * k + j] == r
    out, _ = orc.combine(Y, w, position, tokens, k)
    ref = torch.zeros(tokens, N, dtype=torch.float64)
    for t in range(tokens):
        for j in range(k):
            if ids[t, j] >= 0:
                ref[t] += w[t, j].double() * (X[t].double() @ W[ids[t, j]].double())
    assert torch.allclose(out, ref)
    dW, _ = orc.dweight(X, Y, ids, E, "tokens")
    for e in range(E):
        assert torch.allclose(dW[e], sum((torch.outer(X[t].double(), Y[r]) for r, (t, j) in enumerate(rows) if ids[t, j] == e), torch.zeros(C, N, dtype=torch.float64)))


def test_served_layer_keeps_its_scales_its_rows_and_its_router(monkeypatch):
    """Casts, copies and moves of a layer on 8-bit weights, and of the layer it was made from."""
    import copy

    def quantize(x):                                       # (rows in 8 bits without a GPU, laid out as the operator's)
        scale = x.float().abs().amax(-1) / 127
        rows = torch.zeros(*x.shape[:-1], (x.shape[-1] + 15) // 16 * 16, dtype=torch.int8)[..., :x.shape[-1]]
        return rows.copy_((x.float() / scale.unsqueeze(-1)).round()), scale

    monkeypatch.setattr(ops, "quantize_rows", quantize)
    layer = egs.RoutedExperts(4, 24, 40, 2, balance=True)
    served = layer.quantized()
    before = {n: t.clone() for n, t in served.state_dict().items()}
    rows = lambda m: [(t.stride(-1), t.stride(-2) % 16) for t in (m.up, m.down)]
    assert rows(served) == [(1, 0)] * 2 and served.up.shape == (4, 40, 24)
    served.to(torch.bfloat16)
    assert served.up_scale.dtype == served.down_scale.dtype == served.router.balance.dtype == torch.float32
    assert served.router.W.dtype == torch.bfloat16 and layer.router.W.dtype == torch.float32
    for name in ("up", "down", "up_scale", "down_scale", "router.balance"):
        assert torch.equal(served.state_dict()[name], before[name])
    # training on does not move the served router
    with torch.no_grad():
        layer.router.W.add_(1.0)
        layer.router.balance.add_(1.0)
    assert torch.equal(served.router.W, before["router.W"].bfloat16()) and not served.router.balance.any()
    assert not any(p.requires_grad for p in served.parameters()) and all(p.requires_grad for p in layer.parameters())
    # copies that put rows together get their pitch back
    dense = served._apply(lambda t: t.contiguous().clone())
    assert dense is served and rows(served) == [(1, 0)] * 2 and torch.equal(served.up, before["up"])
    other = copy.deepcopy(served)
    other.load_state_dict(served.state_dict())
    assert rows(other) == [(1, 0)] * 2 and torch.equal(other.down, served.down)
    meta = copy.deepcopy(served).to("meta")
    assert meta.up_scale.dtype == torch.float32 and meta.up_scale.is_meta


def test_entries_refuse_rows_that_cannot_be_counted():
    """Up to 2^31 - 4096 rows a few tiles behind the last one can be counted in 32 bits; one more is refused, before a pointer is looked at."""
    lib, most = _lib.load(), (1 << 31) - 4096
    for n, code in ((most, BAD), (most + 1, LARGE), ((1 << 31) - 1, LARGE)):          # (BAD: the pointers that are missing)
        assert lib.egs_route_tokens(None, None, None, None, route(tokens=n), 8, _lib.F32, None) == code
        assert lib.egs_route_tokens_backward(None, None, None, None, route(tokens=n), 8, _lib.F32, None) == code
        assert lib.egs_plan_experts(None, n, 4, None, None, None, None, 0, None, None) == BAD
        assert lib.egs_plan_experts(one, n, 4, one, one, one, None, 0, None, None) == (WORKSPACE if code == BAD else LARGE)
        assert lib.egs_quantize_rows(None, None, None, n, 1, 1, 1, _lib.F32, None) == code
        for tokens, k in ((n, 1), (1, n)):
            d = ragged(tokens=tokens, k=k, E=2, C=1, N=1)
            for dtype in (_lib.F32, _lib.BF16):
                assert lib.egs_expert_matmul(None, None, None, None, None, d, 0, 0, dtype, 0, None, 0, None, None) == code
                assert lib.egs_expert_dweight(None, None, None, None, None, d, 0, dtype, 0, None, 0, None, None) == code
                assert lib.egs_combine(None, None, None, None, tokens, k, 1, dtype, dtype, None) == code
                assert lib.egs_combine_backward(None, None, None, None, None, None, tokens, k, 1, dtype, dtype, None) == code
            assert lib.egs_expert_matmul_int8(None, None, 1, None, None, 1, one, None, None, d, 0, _lib.F32, 0, None, None) == code
