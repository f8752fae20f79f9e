"""Rows in 4 bits and their products on the GPU, against the definitions in float64."""
import pytest
import torch

from expertscattergather_b200 import ops
from oracle import choice_oracle as orc
from oracle import fp4_oracle as fp4

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def randn(*shape, seed=0, dtype=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=gen).to(dtype)


def same(a, b):
    """Equal values, NaN where the other is NaN."""
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def check_rows(X, q, scale):
    C = X.shape[-1]
    codes, byte = fp4.quantize(X)
    assert q.dtype == scale.dtype == torch.uint8
    assert q.shape == (*X.shape[:-1], (C + 1) // 2) and scale.shape == (*X.shape[:-1], (C + 31) // 32)
    assert torch.equal(scale.int(), byte.int())
    assert torch.equal(q, fp4.pack(codes)[..., :q.shape[-1]])


# ---- rows ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 2), (5, 31), (1, 32), (7, 33), (130, 64), (33, 330), (9, 1030), (600, 2048), (2, 8200), (4097, 40)])
def test_quantize(dtype, rows, C):
    X = (randn(rows, C, seed=C) * torch.exp(3 * randn(rows, 1, seed=1))).to(TYPES[dtype])
    q, scale = ops.quantize_rows_fp4(X)
    check_rows(X, q, scale)
    assert (rows == 1 or q.stride(0) % 16 == 0) and (rows == 1 or scale.stride(0) % 16 == 0)
    for out in TYPES.values():
        back = ops.dequantize_rows_fp4(q, scale, C, dtype=out)
        assert back.dtype == out and same(back.double(), fp4.values(*fp4.quantize(X), C).to(out).double())     # (rows beyond f16 have infinities)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_borders(dtype):
    """Every border between two values, its neighbours on both sides, at many scales, both signs."""
    t = TYPES[dtype]
    base = torch.tensor([0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, .5, 1, 1.5, 2, 3, 4], device="cuda")
    e = torch.arange(-12 if dtype == "f16" else -120, 12 if dtype == "f16" else 120, device="cuda").float()
    at = (base * torch.exp2(e).unsqueeze(-1)).to(t)
    up, down = (torch.nextafter(at, torch.full_like(at, s)) for s in (float("inf"), 0.0))
    X = torch.stack([torch.cat((v, -v), -1) for v in (at, up, down)], 1)          # [e, 3, 32]: a border is the block's largest, or not
    small = X.clone()
    small[..., 8:10] = 0
    small[..., 24:26] = 0
    for x in (X, small, X.flatten(1)):
        check_rows(x, *ops.quantize_rows_fp4(x))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_specials(dtype):
    t = TYPES[dtype]
    inf, nan, top, tiny = float("inf"), float("nan"), torch.finfo(t).max, torch.finfo(t).smallest_normal
    X = randn(9, 96, seed=3).to(t)
    X[0] = 0
    X[1] = -0.0
    X[2, 40] = inf
    X[3, 95] = -inf
    X[4, 0] = nan
    X[5] = top
    X[6] = torch.linspace(-1, 1, 96, device="cuda").to(t) * tiny
    X[7, 5:] = 0
    X[8] = torch.linspace(-1, 1, 96, device="cuda").to(t) * top
    q, scale = ops.quantize_rows_fp4(X)
    check_rows(X, q, scale)
    back = ops.dequantize_rows_fp4(q, scale)
    assert back[2, 32:64].isnan().all() and not back[2, :32].isnan().any() and back[4, :32].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strides(dtype):
    t = TYPES[dtype]
    big = randn(40, 7, 200, seed=5).to(t)
    for X in (big[:, 1], big[:, :, 3:99], big[::2, 2, 1:], big.transpose(0, 2), big[3, 4], big[:, 2, ::2], big[:0], big[:, :, :0], big[:1, :1, 5:38], big[0, 0, 7]):
        if X.dim() == 0:
            with pytest.raises(ValueError):
                ops.quantize_rows_fp4(X)
            continue
        q, scale = ops.quantize_rows_fp4(X)
        check_rows(X, q, scale)
        assert torch.equal(ops.dequantize_rows_fp4(q, scale, X.shape[-1]).double(), fp4.values(*fp4.quantize(X), X.shape[-1]))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_silu_is_torchs(dtype):
    X = (3 * randn(700, 1030, seed=2)).to(TYPES[dtype])
    X[0, :8] = torch.tensor([-200.0, -104, -88, -87, 0, 88, 200, -1e-6], device="cuda").to(X.dtype)
    x = X.float()
    check_rows(x / (1 + torch.exp(-x)), *ops.quantize_rows_fp4(X, activation="silu"))


def test_quantize_many_rows_and_far_ones():
    """More rows than a dimension of a grid has CTAs for, and elements beyond 2^31."""
    X = randn(600011, 2, seed=7, dtype=torch.bfloat16)
    check_rows(X, *ops.quantize_rows_fp4(X))
    X = torch.zeros(2 ** 21 + 5, 1056, device="cuda", dtype=torch.bfloat16)
    X[-3:] = randn(3, 1056, seed=8)
    q, scale = ops.quantize_rows_fp4(X)
    check_rows(X[-5:], q[-5:], scale[-5:])
    assert torch.equal(ops.dequantize_rows_fp4(q, scale, dtype=torch.bfloat16)[-5:].double(), fp4.rows(q[-5:], scale[-5:]))


# ---- products -----------------------------------------------------------------------------------------

def product_bound(size, Y, C, out):
    """A block's 32 products are exact and so is their sum; sums of blocks are float32: four truncations for two blocks at most, each by 2^-23 of what has
    been summed, and the result is rounded once."""
    return size * ((C / 64 + 2) * 4 * 2.0 ** -23) + Y.abs() * (torch.finfo(out).eps / 2 if out != torch.float32 else 0) + 1e-30


def operands(rows, E, C, N, seed=0):
    X = randn(rows, C, seed=seed) * torch.exp(randn(rows, 1, seed=seed + 1))
    W = randn(E, N, C, seed=seed + 2) / C ** 0.5
    return ops.quantize_rows_fp4(X), ops.quantize_rows_fp4(W)


def even(C):
    return (C + 1) // 2 * 2


SHAPES = [(1, 32, 32), (5, 64, 33), (130, 256, 224), (128, 2048, 512), (700, 330, 201), (300, 1030, 777), (257, 96, 450), (64, 4100, 64), (1500, 512, 1000), (3, 1, 1)]


@pytest.mark.parametrize("path", ["tensor", "generic"])
@pytest.mark.parametrize("rows,C,N", SHAPES)
def test_matmul(path, rows, C, N):
    (q, s), (wq, ws) = operands(rows, 1, C, N)
    x, w = fp4.rows(q, s), fp4.rows(wq[0], ws[0])
    Y, size = x @ w.t(), x.abs() @ w.abs().t()
    for out in TYPES.values():
        got = ops.matmul_fp4(q, s, wq[0], ws[0], out_dtype=out, path=path)
        assert got.shape == (rows, N) and got.dtype == out
        worst = ((got.double() - Y).abs() - product_bound(size, Y, C, out)).max().item()
        assert worst <= 0, (out, worst, (got.double() - Y).abs().max().item())


def choose(tokens, E, k, seed, skew=0.5, idle=0, lost=0.0):
    popular = skew * randn(E, seed=seed)
    if idle:
        popular[:idle] = -1e4
    ids = (randn(tokens, E, seed=seed + 1) + popular).topk(k, -1).indices.int()
    if lost:
        ids[randn(tokens, k, seed=seed + 2).abs() < lost] = -1
    return ids


ROUTED = [(1, 64, 8, 256, 64, 0), (3, 64, 8, 2048, 512, 0), (200, 13, 3, 330, 201, 0.3), (1000, 8, 2, 512, 480, 0.1), (4000, 16, 4, 288, 512, 0), (50, 1, 1, 64, 32, 0.5), (6, 4, 2, 64, 64, 9.0), (900, 200, 2, 128, 96, 0)]


@pytest.mark.parametrize("path", ["auto", "tensor", "generic"])
@pytest.mark.parametrize("tokens,E,k,C,N,lost", ROUTED)
def test_expert_matmul(path, tokens, E, k, C, N, lost):
    ids = choose(tokens, E, k, seed=tokens, lost=lost, idle=E // 8)
    plan = ops.plan_experts(ids, E)
    for rows in ("tokens", "sorted"):
        (q, s), (wq, ws) = operands(tokens if rows == "tokens" else tokens * k, E, C, N, seed=3)
        Y, size = orc.matmul(fp4.rows(q, s), fp4.rows(wq, ws).transpose(1, 2), ids, E, rows)
        for out in TYPES.values():
            got = ops.expert_matmul_fp4(q, s, wq, ws, plan, rows=rows, out_dtype=out, path=path)
            worst = ((got.double() - Y).abs() - product_bound(size, Y, C, out)).max().item()
            assert worst <= 0, (rows, out, worst)
    ops.check_status()


@pytest.mark.parametrize("path", ["tensor", "generic"])
@pytest.mark.parametrize("tokens,E,k,C,N,lost", ROUTED)
def test_expert_matmul_into_4_bits(path, tokens, E, k, C, N, lost):
    """The rows that leave in 4 bits are those of the product in float32."""
    ids = choose(tokens, E, k, seed=tokens, lost=lost)
    plan = ops.plan_experts(ids, E)
    (q, s), (wq, ws) = operands(tokens, E, C, N, seed=4)
    full = ops.expert_matmul_fp4(q, s, wq, ws, plan, out_dtype=torch.float32, path=path)
    check_rows(full, *ops.expert_matmul_fp4_rows(q, s, wq, ws, plan, path=path))
    y, ys = ops.expert_matmul_fp4_rows(q, s, wq, ws, plan, activation="silu", path=path)
    got = fp4.values(fp4.codes_of(y), ys, N)
    want = fp4.values(*fp4.quantize(full / (1 + torch.exp(-full))), N)
    # the tensor cores' read-out forms the activation within 2^-20: a value that lies so near a border may go the other way, one step, or its block's scale
    off = got != want
    assert off.double().mean().item() <= (0 if path == "generic" else 2e-4)
    step = torch.exp2(torch.maximum(ys.double(), fp4.quantize(full / (1 + torch.exp(-full)))[1].double()) - 127).repeat_interleave(32, -1)[..., :N]
    assert ((got - want).abs() <= 2 * step).all()
    ops.check_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_smallest_numbers_and_no_numbers(dtype):
    """Blocks of subnormal numbers, zeros, infinities and NaN beside ordinary ones, in rows of all three forms of the kernels."""
    t = TYPES[dtype]
    small = torch.finfo(t).smallest_normal if dtype != "f16" else 2.0 ** -14
    for C in (32, 31, 40, 264, 1030, 1056):
        X = randn(12, C, seed=C).to(t)
        X[0] = (X[0].float() * small).to(t)
        X[1] = (X[1].float() * small / 8).to(t)
        X[2] = 0
        X[3, C // 2] = float("inf")
        X[4, 0] = float("-inf")
        X[5, C - 1] = float("nan")
        X[6] = torch.finfo(t).max
        q, scale = ops.quantize_rows_fp4(X)
        check_rows(X, q, scale)
        back = ops.dequantize_rows_fp4(q, scale, C, dtype=torch.float32)
        want = fp4.values(*fp4.quantize(X), C).to(torch.float32)             # (6 * 2^126, what float32's largest number becomes, is beyond it)
        assert bool(same(back, want))


# ---- sums over a token's experts ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,E,k,C,N", [(40, 8, 2, 256, 96), (300, 16, 4, 520, 330)])
def test_projection_of_experts_is_rounded_once(dtype, tokens, E, k, C, N):
    """A token's sum over its experts as a workload forms it: off by half a step of its type, and by float32 sums."""
    from perf import more_operators as workloads
    case = workloads._product("", tokens, E, k, C, N, dtype)
    state = workloads.prepare(case, 5)
    out, = workloads._run_own(state)
    up, w, ids = fp4.rows(state["up"], state["up_scale"])[..., :C], state["weights"].double(), state["experts"].long()
    xq = fp4.values(*fp4.quantize(state["X"]), C)
    want, size = (torch.zeros(tokens, N, dtype=torch.float64, device="cuda") for _ in range(2))
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        want.index_put_((t,), w[t, j].unsqueeze(-1) * (xq[t] @ up[e].t()), accumulate=True)
        size.index_put_((t,), w[t, j].unsqueeze(-1) * (xq[t].abs() @ up[e].abs().t()), accumulate=True)
    # a product's float32 sums (product_bound), then k products with weights and their sums, 2^-24 of what has been summed each
    off = product_bound(size, want, C, TYPES[dtype]) + size * (2 * k * 2.0 ** -24) + (2.0 ** -25 if dtype == "f16" else 0)
    assert ((out.double() - want).abs() - off).max().item() <= 0


@pytest.mark.parametrize("tokens", [1, 3, 300])
def test_weights_beyond_32_bits(tokens):
    """Experts whose weights lie more than 2^32 bytes behind the first one's; their last channels."""
    E, N, C = 18, 16384, 32768
    wq, ws = (torch.empty(E, N, n, device="cuda", dtype=torch.uint8) for n in (C // 2, C // 32))
    last = 96
    wq[E - 1], ws[E - 1] = 0, 127
    wq[E - 1, -last:], ws[E - 1, -last:] = ops.quantize_rows_fp4(randn(last, C, seed=1))
    q, s = ops.quantize_rows_fp4(randn(tokens, C, seed=2))
    plan = ops.plan_experts(torch.full((tokens, 1), E - 1, dtype=torch.int32, device="cuda"), E)
    x, w = fp4.rows(q, s), fp4.rows(wq[E - 1, -last:], ws[E - 1, -last:])
    Y, size = x @ w.t(), x.abs() @ w.abs().t()
    got = ops.expert_matmul_fp4(q, s, wq, ws, plan, out_dtype=torch.float32)
    assert not got[:, :-last].any()
    assert ((got[:, -last:].double() - Y).abs() - product_bound(size, Y, C, torch.float32)).max().item() <= 0
    ops.check_status()


# ---- far scales ---------------------------------------------------------------------------------------

FAR = [(123, -20), (-20, 123), (124, -130), (-130, 124), (110, 8), (8, 110), (-100, 20), (20, -100), (100, -100), (-149, 110)]


@pytest.mark.parametrize("path", ["auto", "tensor", "generic"])
@pytest.mark.parametrize("up,down", FAR)
@pytest.mark.parametrize("rows,C,N", [(1, 4096, 64), (1, 70, 33), (130, 512, 96)])
def test_products_of_far_scales(path, up, down, rows, C, N):
    """Rows and weights of magnitudes at the ends of float32 whose products are ordinary numbers."""
    X, W = torch.ldexp(randn(rows, C, seed=1), torch.tensor(up, device="cuda")), torch.ldexp(randn(N, C, seed=2), torch.tensor(down, device="cuda"))
    (q, s), (wq, ws) = ops.quantize_rows_fp4(X), ops.quantize_rows_fp4(W)
    x, w = fp4.rows(q, s), fp4.rows(wq, ws)
    Y, size = x @ w.t(), x.abs() @ w.abs().t()
    plan = ops.plan_experts(torch.zeros(rows, 1, dtype=torch.int32, device="cuda"), 1)
    for out in (torch.float32, torch.bfloat16):
        for got in (ops.matmul_fp4(q, s, wq, ws, out_dtype=out, path=path), ops.expert_matmul_fp4(q, s, wq[None], ws[None], plan, out_dtype=out, path=path)):
            # relative to the magnitudes, which product_bound's smallest term would hide: 2^-149 is float32's
            off = product_bound(size, Y, C, out) - 1e-30 + 2.0 ** -148
            assert ((got.double() - Y).abs() - off).max().item() <= 0


# ---- activations ahead of 4 bits ----------------------------------------------------------------------

@pytest.mark.parametrize("path", ["auto", "tensor", "generic"])
@pytest.mark.parametrize("tokens,E,k,C,N", [(1, 8, 2, 96, 70), (300, 6, 2, 128, 256), (2000, 4, 1, 64, 224)])
@pytest.mark.parametrize("low,high", [(-110, -86), (-90, -60), (-70, -10), (-12, 0), (-1, 1), (0, 100)])
def test_activations_ahead_of_4_bits_are_the_exact_ones(path, tokens, E, k, C, N, low, high):
    """Rows that leave activated are those of the same product in float32, activated and brought into 4 bits by themselves, whatever kernel has them: whole
    blocks of sums between `low` and `high`.  The tensor cores' read-out forms activations within 2^-20 of the elementary form (relative; infinite
    exponentials give 0 in both), so there a value may go the other way where a border between two lies as near."""
    plan = ops.plan_experts(choose(tokens, E, k, seed=7), E)
    q, s = ops.quantize_rows_fp4(1 + 0.2 * randn(tokens, C, seed=1))
    wq, ws = ops.quantize_rows_fp4((low + (high - low) * torch.rand(E, N, 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))) * (1 + 0.1 * randn(E, N, C, seed=3)) / C)
    full = ops.expert_matmul_fp4(q, s, wq, ws, plan, out_dtype=torch.float32, path=path)
    y, ys = ops.expert_matmul_fp4_rows(q, s, wq, ws, plan, activation="silu", path=path)
    elementary = full / (1 + torch.exp(-full))
    if path == "generic" or tokens == 1 and path == "auto":
        check_rows(elementary, y, ys)
    v = elementary.double()
    (_, least), (_, most) = (fp4.quantize(v * f) for f in (1 - 2.0 ** -20, 1 + 2.0 ** -20))
    assert ((ys >= least) & (ys <= most)).all()
    power = torch.exp2(ys.double() - 127).repeat_interleave(32, -1)[..., :N]
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5], dtype=torch.float64, device="cuda")
    level = torch.tensor(fp4.LEVELS, dtype=torch.float64, device="cuda")
    size, got = v.abs() / power, fp4.values(fp4.codes_of(y), ys, N) / power
    low_level, high_level = (level[torch.bucketize(size * f, edges)] for f in (1 - 2.0 ** -20, 1 + 2.0 ** -20))
    assert ((got.abs() >= low_level) & (got.abs() <= high_level) & ((got == 0) | (torch.sign(got) == torch.sign(v)))).all()


def test_activations_where_the_exponential_ends():
    """Sums on both sides of the first float whose exponential is infinite: 0 or a number as in the elementary form."""
    N, edge = 256, int(88.72283935546875 * 2 ** 17)
    sums = edge + torch.randint(-8, 9, (N,), generator=torch.Generator().manual_seed(1))
    codes, C = torch.zeros(N, 192, dtype=torch.int32), 192
    for n, total in enumerate(sums.tolist()):
        for digit in range(6):                               # four bits of a sum to each block
            left, at = total >> 4 * digit & 15, 32 * digit
            for code in (7, 6, 5, 4, 2):                     # 6, 4, 3, 2, 1
                while left >= fp4.LEVELS[code]:
                    codes[n, at], left, at = code + 8, left - int(fp4.LEVELS[code]), at + 1
    wq, ws = fp4.pack(codes)[None].cuda(), torch.zeros(1, N, 16, dtype=torch.uint8, device="cuda")
    ws[..., :6] = torch.tensor([127 - 17 + 4 * digit for digit in range(6)], dtype=torch.uint8)
    ws = ws[..., :6]
    q, s = ops.quantize_rows_fp4(torch.ones(130, C, device="cuda"))
    plan = ops.plan_experts(torch.zeros(130, 1, dtype=torch.int32, device="cuda"), 1)
    for path in ("tensor", "generic"):
        full = ops.expert_matmul_fp4(q, s, wq, ws, plan, out_dtype=torch.float32, path=path)
        assert (full.double() * 2 ** 17 + sums.cuda()).abs().max() <= 2
        elementary = full / (1 + torch.exp(-full))
        got = fp4.rows(*ops.expert_matmul_fp4_rows(q, s, wq, ws, plan, activation="silu", path=path))
        assert torch.equal(got == 0, elementary == 0) and (elementary == 0).any() and (elementary != 0).any()
