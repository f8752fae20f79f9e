"""What the operators in 4 bits check before they touch a GPU, and their oracle against plain loops."""
import ctypes
import math

import pytest
import torch

from expertscattergather_b200 import _lib, ops
from oracle import fp4_oracle as fp4

BAD, LARGE, WORKSPACE, OK = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_TOO_LARGE, _lib.ERR_WORKSPACE, _lib.OK
one, off = ctypes.c_void_p(16), ctypes.c_void_p(24)          # pointers that are never followed: every call here is refused or has nothing to do


def ragged(tokens=10, k=2, E=4, C=64, N=64):
    return ctypes.byref(_lib.Ragged(tokens, k, E, C, N))


def test_oracle_against_loops():
    gen = torch.Generator().manual_seed(0)
    X = torch.randn(6, 70, generator=gen) * torch.exp(2 * torch.randn(6, 1, generator=gen))
    X[0, :32] = torch.tensor([0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, -7, -5, -.25, -.75, .5, 1] * 2)
    codes, byte = fp4.quantize(X)
    for r in range(6):
        for b in range(3):
            x = [X[r, i].item() for i in range(32 * b, min(32 * b + 32, 70))]
            j = min(j for j in range(-127, 128) if max(map(abs, x)) <= 7 * 2.0 ** j)
            assert byte[r, b] == j + 127
            for i, v in enumerate(x):
                m = abs(v) / 2.0 ** j
                best = min(range(8), key=lambda c: (abs(fp4.LEVELS[c] - m), c % 2))      # (an even code has an even mantissa)
                assert codes[r, 32 * b + i] == best + 8 * (math.copysign(1, v) < 0)
    assert not codes[:, 70:].any()
    q = fp4.pack(codes)
    assert torch.equal(fp4.codes_of(q), codes)
    err = (fp4.values(codes, byte, 70) - X).norm() / X.norm()
    assert err < 0.2


@pytest.mark.parametrize("args,code", [((4, 64, 64, 32, 16, 0, 0), BAD), ((-1, 64, 64, 32, 16, 0, 0), BAD), ((4, -1, 64, 32, 16, 0, 0), BAD), ((4, 64, -1, 32, 16, 0, 0), BAD),
                                       ((4, 64, 64, 31, 16, 0, 0), BAD), ((4, 64, 64, 40, 16, 0, 0), BAD), ((4, 65, 65, 32, 16, 0, 0), BAD), ((4, 64, 64, 32, 8, 0, 0), BAD),
                                       ((4, 1024, 1024, 512, 16, 0, 0), BAD), ((4, 64, 64, 32, 16, 2, 0), BAD), ((4, 64, 64, 32, 16, 0, 3), BAD),
                                       (((1 << 31) - 4095, 64, 64, 32, 16, 0, 0), LARGE), ((4, (1 << 24) + 1, 1 << 25, 1 << 24, 1 << 20, 0, 0), LARGE),
                                       ((0, 64, 64, 32, 16, 0, 0), OK), ((4, 0, 0, 0, 0, 0, 0), OK)])
def test_rows_entries(args, code):
    lib = _lib.load()
    rows, C, x_stride, q_stride, s_stride, act, dtype = args
    X = None if code == BAD and args == (4, 64, 64, 32, 16, 0, 0) else one
    assert lib.egs_quantize_rows_fp4(X, one, one, rows, C, x_stride, q_stride, s_stride, act, dtype, None) == code
    if x_stride >= 0 and act < 2:
        assert lib.egs_dequantize_rows_fp4(one, one, X, rows, C, q_stride, s_stride, dtype, None) == code or q_stride == 32 and C == 65
    if code == OK:
        assert lib.egs_quantize_rows_fp4(None, None, None, rows, C, x_stride, q_stride, s_stride, act, dtype, None) == OK


def test_rows_entries_alignment():
    lib = _lib.load()
    assert lib.egs_quantize_rows_fp4(one, off, one, 4, 64, 64, 32, 16, 0, 0, None) == BAD
    assert lib.egs_dequantize_rows_fp4(off, one, one, 4, 64, 32, 16, 0, None) == BAD


def product(q=one, qs=one, qp=32, sp=16, w=one, ws=one, wp=32, wsp=16, offsets=one, slots=one, y=one, dims=None, rows=0, out=0, path=0, into4=False, yp=32, ysp=16, act=0,
            ws_mem=None, ws_bytes=0):
    lib = _lib.load()
    dims = dims if dims is not None else ragged()
    if into4:
        return lib.egs_expert_matmul_fp4_rows(q, qs, qp, sp, w, ws, wp, wsp, offsets, slots, y, y, yp, ysp, dims, rows, act, path, ws_mem, ws_bytes, None, None)
    return lib.egs_expert_matmul_fp4(q, qs, qp, sp, w, ws, wp, wsp, offsets, slots, y, dims, rows, out, path, None, None)


@pytest.mark.parametrize("into4", [False, True])
@pytest.mark.parametrize("change,code", [({"rows": 2}, BAD), ({"path": 3}, BAD), ({"qp": 24}, BAD), ({"qp": 16}, BAD), ({"sp": 8}, BAD), ({"sp": 0}, BAD), ({"wp": 40}, BAD), ({"wsp": 2}, BAD),
                                         ({"q": None}, BAD), ({"qs": None}, BAD), ({"w": None}, BAD), ({"ws": None}, BAD), ({"slots": None}, BAD), ({"y": None}, BAD), ({"offsets": None}, BAD),
                                         ({"q": off}, BAD), ({"qs": off}, BAD), ({"w": off}, BAD), ({"ws": off}, BAD), ({"dims": {"C": 63}}, BAD), ({"dims": {"tokens": -1}}, BAD), ({"dims": {"E": 0}}, BAD),
                                         ({"dims": {"E": 1025}}, LARGE), ({"dims": {"N": (1 << 24) + 1}}, LARGE), ({"dims": {"tokens": 1 << 30, "k": 4}}, LARGE), ({"dims": {"tokens": 0}}, OK), ({"dims": {"N": 0}}, OK)])
def test_product_entries(into4, change, code):
    change = dict(change)
    if "dims" in change:
        change["dims"] = ragged(**change["dims"])
    assert product(into4=into4, **change) == code


def test_product_entries_of_their_own():
    assert product(out=3) == BAD
    assert product(into4=True, act=2) == BAD
    for bad in ({"yp": 24}, {"yp": 16}, {"ysp": 1}, {"y": off}):
        assert product(into4=True, **bad) == BAD
    lib = _lib.load()
    need = lib.egs_expert_matmul_fp4_rows_workspace_bytes(ragged(), _lib.PATH_GENERIC)
    assert need == 20 * 64 * 4
    assert product(into4=True, path=_lib.PATH_GENERIC, ws_mem=one, ws_bytes=need - 1) == WORKSPACE
    assert product(into4=True, path=_lib.PATH_GENERIC) == WORKSPACE
    assert product(into4=True, path=_lib.PATH_GENERIC, ws_mem=off, ws_bytes=need) == WORKSPACE
    assert lib.egs_expert_matmul_fp4_rows_workspace_bytes(ragged(tokens=0), 0) == 0
    assert lib.egs_expert_matmul_fp4_rows_workspace_bytes(ragged(C=63), 0) == 0


def test_python_refuses():
    x = torch.zeros(4, 64)
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    with pytest.raises((RuntimeError, ValueError)):
        ops.quantize_rows_fp4(x)
    with pytest.raises(ValueError):
        ops.quantize_rows_fp4(x, activation="relu")
    with pytest.raises(ValueError):
        ops.quantize_rows_fp4(torch.tensor(1.0))
    with pytest.raises((RuntimeError, ValueError)):
        ops.matmul_fp4(q, s, q, s)
    with pytest.raises((RuntimeError, ValueError)):
        ops.dequantize_rows_fp4(q, s, dtype=torch.int32)
