"""Operators for tokens that choose experts, where a call is at the edge of what it takes: plans made by hand, plans that lie elsewhere,
groups whose values are almost equal, weight gradients in every variant, second derivatives, casts of the served layer.

Tolerances are those of the tests of the operators: float32 sums of n products are off by at most (n + 2) * 2 * u times the sum of the
products' magnitudes (u = 2^-24), a rounding to 16 bits by half a unit.
"""
import pytest
import torch

from expertscattergather_b200 import ops

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
