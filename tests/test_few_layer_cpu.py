"""What the whole layer for a few tokens checks before it touches a GPU, and the modules that call it."""
import copy
import ctypes

import pytest
import torch

import expertscattergather_b200 as egs
from expertscattergather_b200 import _lib, ops
from oracle import fp4_oracle as fp4

BAD, LARGE, WORKSPACE, OK = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_TOO_LARGE, _lib.ERR_WORKSPACE, _lib.OK
one, off = ctypes.c_void_p(16), ctypes.c_void_p(24)          # pointers that are never followed: every call here is refused or has nothing to do


def route(tokens=4, E=8, top_k=2, groups=1, top_groups=1, group_top=2, score=0, renormalize=1, scale=1.0):
    return ctypes.byref(_lib.Route(tokens, E, top_k, groups, top_groups, group_top, score, renormalize, scale))


def plain(spec=None, I=64, J=64, x_stride=64, dtype=0, ws=one, size=1 << 40, **hole):
    a = {n: hole.get(n, one) for n in ("X", "router", "up", "down", "out", "weights", "experts")}
    return _lib.load().egs_routed_experts_few(a["X"], a["router"], None, a["up"], a["down"], a["out"], a["weights"], a["experts"], spec if spec is not None else route(), I, J, x_stride,
                                              dtype, ws, size, None)


def fp4_call(spec=None, I=64, J=64, up=one, us=one, upp=32, upf=2048, usp=16, upl=_lib.W_NC, down=one, ds=one, dp=32, df=2048, dsp=16, dl=_lib.W_NC, ws=one, size=1 << 40):
    return _lib.load().egs_routed_experts_few_fp4(one, one, None, up, us, upp, upf, usp, upl, down, ds, dp, df, dsp, dl, one, one, one, spec if spec is not None else route(), I, J, 64, 0, ws, size, None)


@pytest.mark.parametrize("spec,code", [({"E": 0}, BAD), ({"top_k": 0}, BAD), ({"top_k": 9}, BAD), ({"groups": 3}, BAD), ({"groups": 4, "top_groups": 5}, BAD), ({"group_top": 3}, BAD), ({"score": 2}, BAD),
                                       ({"tokens": -1}, BAD), ({"tokens": 33}, LARGE), ({"tokens": 32, "E": 16, "top_k": 9}, LARGE), ({"E": 1025}, LARGE), ({"E": 64, "top_k": 33}, LARGE), ({"E": 66, "groups": 33}, LARGE),
                                       ({"tokens": 0}, OK)])
def test_entries(spec, code):
    assert plain(route(**spec)) == code and fp4_call(route(**spec)) == code


def test_entries_sizes_pointers_and_workspaces():
    for call in (plain, fp4_call):
        assert call(I=0) == BAD and call(J=0) == BAD and call(I=(1 << 24) + 1) == LARGE and call(J=(1 << 24) + 1) == LARGE
        need = _lib.load().egs_routed_experts_few_workspace_bytes(route(), 64, 64)
        assert need >= 4 * 8 * 4 + 4 * 2 * 64 * 4
        assert call(size=need - 1) == WORKSPACE and call(ws=None) == WORKSPACE and call(ws=off) == WORKSPACE
    assert plain(dtype=3) == BAD and plain(x_stride=-1) == BAD
    for name in ("X", "router", "up", "down", "out", "weights", "experts"):
        assert plain(**{name: None}) == BAD
    for bad in ({"upp": 24}, {"upp": 16}, {"usp": 1}, {"dp": 8}, {"dsp": 0}, {"us": None}, {"ds": None}, {"up": off}, {"down": off}, {"up": None}, {"upl": 2}, {"upf": 2000}, {"upf": 2040},
                {"df": 2008}, {"upl": _lib.W_CN}, {"upl": _lib.W_CN, "upp": 64, "upf": 2047}, {"upl": _lib.W_CN, "upp": 63}, {"dl": _lib.W_CN, "dp": 64, "df": 2047}, {"dl": _lib.W_CN, "dp": 64, "dsp": 1}):
        assert fp4_call(**bad) == BAD
    for good in ({"upl": _lib.W_CN, "upp": 64}, {"dl": _lib.W_CN, "dp": 64, "down": off}, {"upl": _lib.W_CN, "upp": 65, "upf": 31 * 65 + 64, "usp": 2}):
        assert fp4_call(**good, size=0) == WORKSPACE
    assert _lib.load().egs_routed_experts_few_workspace_bytes(route(tokens=33), 64, 64) == 0
    assert _lib.load().egs_routed_experts_few_workspace_bytes(route(tokens=0), 64, 64) == 0
    assert _lib.load().egs_routed_experts_few_workspace_bytes(None, 64, 64) == 0


def test_limits_are_the_librarys():
    assert plain(route(tokens=ops.FEW_TOKENS, E=64, top_k=ops.FEW_SLOTS // ops.FEW_TOKENS), size=0) == WORKSPACE
    assert plain(route(tokens=ops.FEW_TOKENS, E=64, top_k=ops.FEW_SLOTS // ops.FEW_TOKENS + 1), size=0) == LARGE
    assert plain(route(tokens=ops.FEW_TOKENS + 1, top_k=1), size=0) == LARGE


def test_python_refuses_cpu_tensors():
    x, router, up, down = torch.zeros(2, 16), torch.zeros(4, 16), torch.zeros(4, 16, 8), torch.zeros(4, 8, 16)
    with pytest.raises(RuntimeError):
        ops.routed_experts_few(x, router, up, down, 2)
    with pytest.raises(ValueError):
        ops.routed_experts_few(x, router, up, down, 2, up_scale=up)
    with pytest.raises(ValueError):
        ops.routed_experts_few(x, router, up[0], down, 2)
    with pytest.raises(ValueError):
        egs.RoutedExperts(4, 16, 8, 2).quantized(bits=5)


def rows4(x, **_):                                         # rows in 4 bits without a GPU, laid out as the operator's
    codes, byte = fp4.quantize(x.float())
    q = fp4.pack(codes)
    out = torch.zeros(*byte.shape[:-1], (byte.shape[-1] + 15) // 16 * 16, dtype=torch.uint8)
    out[..., :byte.shape[-1]] = byte
    return q[..., :(x.shape[-1] + 1) // 2], out[..., :byte.shape[-1]]


def test_served_layer_in_4_bits(monkeypatch):
    """Its weights, what casts, copies and moves leave of them, and which call it makes."""
    monkeypatch.setattr(ops, "quantize_rows_fp4", rows4)
    layer = egs.RoutedExperts(4, 24, 70, 2, balance=True, score="sigmoid", scale=2.0)
    served = layer.quantized(bits=4)
    assert isinstance(served, egs.RoutedExpertsFp4) and isinstance(layer.quantized.__func__(layer, 4), egs.RoutedExpertsFp4)
    assert served.up.shape == (4, 70, 12) and served.up_scale.shape == (4, 70, 1) and served.down.shape == (4, 24, 35) and served.down_scale.shape == (4, 24, 3)
    names = ("up", "down", "up_scale", "down_scale")
    pitches = lambda m: [getattr(m, n).stride(-2) % 16 for n in names]
    before = {n: getattr(served, n).clone() for n in names}
    assert pitches(served) == [0] * 4
    served.to(torch.bfloat16)
    other = copy.deepcopy(served)._apply(lambda t: t.contiguous().clone())
    for m in (served, other):
        assert pitches(m) == [0] * 4 and all(torch.equal(getattr(m, n), before[n]) for n in names)
        assert m.router.balance.dtype == torch.float32 and m.router.W.dtype == torch.bfloat16 and not any(p.requires_grad for p in m.parameters())
    assert set(names) <= set(served.state_dict())
    calls = []
    monkeypatch.setattr(ops, "routed_experts_few", lambda x, *a, **o: calls.append((x, a, o)) or (x, None, None))
    x = torch.zeros(ops.FEW_TOKENS, 1, 24, dtype=torch.bfloat16)
    assert served(x) is x
    _, a, o = calls[0]
    assert a[1] is served.up and a[3] == 2 and a[4] is served.router.balance and o["up_scale"] is served.up_scale and o["score"] == "sigmoid" and o["scale"] == 2.0
    layer.few(torch.zeros(2, 24))
    _, a, o = calls[1]
    assert a[1] is layer.up and a[2] is layer.down and "up_scale" not in o and o["scale"] == 2.0
    monkeypatch.setattr(ops, "plan_experts", lambda *a: (_ for _ in ()).throw(StopIteration))
    monkeypatch.setattr(egs.TokenRouter, "forward", lambda self, x: (None, None))
    with pytest.raises(StopIteration):
        served(torch.zeros(ops.FEW_TOKENS + 1, 24, dtype=torch.bfloat16))
    assert len(calls) == 2


def served_calls(monkeypatch, E, I, J, k, dtype=torch.float32):
    """A served layer in 4 bits without weights to speak of, and the list of the calls that it makes: 'few' or 'separate'."""
    monkeypatch.setattr(ops, "quantize_rows_fp4", lambda x, **_: (torch.zeros(*x.shape[:-1], 16 * ((x.shape[-1] + 31) // 32), dtype=torch.uint8)[..., :(x.shape[-1] + 1) // 2],
                                                                torch.zeros(*x.shape[:-1], (x.shape[-1] + 511) // 512 * 16, dtype=torch.uint8)[..., :(x.shape[-1] + 31) // 32]))
    served = egs.RoutedExperts(E, I, J, k).to(dtype).quantized(bits=4)
    calls = []
    monkeypatch.setattr(ops, "routed_experts_few", lambda x, *a, **o: calls.append("few") or (x, None, None))
    monkeypatch.setattr(egs.TokenRouter, "forward", lambda self, x: calls.append("separate") or (None, None))
    monkeypatch.setattr(ops, "plan_experts", lambda *a: None)
    monkeypatch.setattr(ops, "expert_matmul_fp4_rows", lambda *a, **o: (None, None))
    monkeypatch.setattr(ops, "expert_matmul_fp4", lambda *a, **o: None)
    monkeypatch.setattr(ops, "combine", lambda y, w, plan, out_dtype: torch.zeros(0))
    return lambda x: (calls.clear(), served(x), calls[:])[2]


def test_rows_of_another_type_go_through_the_router(monkeypatch):
    """As autocast hands them over: few tokens are taken as many are."""
    run = served_calls(monkeypatch, 4, 24, 70, 2)
    assert run(torch.zeros(3, 24)) == ["few"]
    monkeypatch.setattr(torch.Tensor, "view", lambda self, *a: self)
    assert run(torch.zeros(3, 24, dtype=torch.bfloat16)) == ["separate"] and run(torch.zeros(40, 24, dtype=torch.bfloat16)) == ["separate"]


@pytest.mark.parametrize("E,I,J,k,one,many", [(8, 24, 70, 2, (0, 1, 4, 5, 32), (33, 700)), (8, 24, 70, 8, (1, 32), (33,)), (64, 24, 70, 9, (1, 28), (29, 32)), (8, 512, 1000, 4, (1, 4, 32), (33,)),
                                              (8, 2048, 1024, 8, (1, 2, 4, 8, 11), (12, 16, 32)), (2, 4096, 4096, 2, (1, 3, 4), (6, 32)), (1, 4096, 4096, 1, (4, 11), (12, 32))])
def test_which_calls_the_served_layer_makes(monkeypatch, E, I, J, k, one, many):
    """Few tokens in one call; those whose experts' weights would be read over and over by the operators for many."""
    run = served_calls(monkeypatch, E, I, J, k)
    monkeypatch.setattr(torch.Tensor, "view", lambda self, *a: self)
    assert [run(torch.zeros(n, I)) for n in one] == [["few"]] * len(one)
    assert [run(torch.zeros(n, I)) for n in many] == [["separate"]] * len(many)
    assert run(torch.zeros(many[0], 1, I)) == ["separate"] and run(torch.zeros(1, one[1], I)) == ["few"]


def test_entries_refuse_addresses_inside_an_element():
    for name in ("X", "router", "up", "down", "out"):
        assert plain(**{name: ctypes.c_void_p(18)}) == BAD and plain(**{name: ctypes.c_void_p(17)}, dtype=1) == BAD
        assert plain(**{name: ctypes.c_void_p(20)}, size=0) == WORKSPACE and plain(**{name: ctypes.c_void_p(18)}, dtype=1, size=0) == WORKSPACE
