"""The whole routed layer for a few tokens, against its definition in float64."""
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


def check_choice(x, router, bias, k, weights, experts, score="softmax", groups=1, top_groups=1, group_top=2, renormalize=True, scale=1.0):
    """The choice is right within what float32 logits and keys are off by; the weights are those of the choice."""
    logits = x.double() @ router.double().t()
    off = 2e-7 * (x.double().abs() @ router.double().abs().t()).max().item() * (x.shape[1] / 256 + 4) + 1e-6       # 3 units a step of a lane, and of the keys
    s = orc.scores(logits, score)
    E = s.shape[1]
    by_logit = bias is None
    key = logits if by_logit else s + bias.double()
    ids = experts.long()
    assert ((ids >= 0) & (ids < E)).all() and all(len(set(r)) == k for r in ids.tolist())
    if groups > 1:
        gkey = s + (0 if bias is None else bias.double())
        value = orc.group_values(gkey, groups, min(group_top, E // groups))
        used = torch.zeros_like(value, dtype=torch.bool).scatter_(1, ids // (E // groups), True)
        cut = value.sort(-1, descending=True).values[:, top_groups - 1:top_groups]
        assert (value >= cut - 4 * off)[used].all() and (used.sum(-1) <= top_groups).all()
        left = torch.where(value > cut + 4 * off, True, used)                              # groups that have to be there, or are
        key = key.masked_fill(~left.repeat_interleave(E // groups, 1), -float("inf"))
    chosen = key.gather(1, ids)
    best = key.sort(-1, descending=True).values[:, :k]
    assert ((best - chosen).abs() <= 4 * off).all()
    want = orc.weights_of(s, ids, renormalize, scale)
    assert ((weights.double() - want).abs() <= scale * (8 * off * want.abs() / scale + 1e-6)).all()


def layer64(x, w, ids, up, down):
    """out and a bound of its error before it is rounded, from the definition; up [E, I, J], down [E, J, I], float64."""
    out, off = torch.zeros(x.shape[0], down.shape[2], dtype=torch.float64, device=x.device), None
    off = torch.zeros_like(out)
    I, J, k = up.shape[1], up.shape[2], ids.shape[1]
    u = 2.0 ** -24
    for e in range(up.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        h = x[t] @ up[e]
        h_off = (x[t].abs() @ up[e].abs()) * ((I / 8 + 24) * u)            # a lane's longest chain, and the joins
        a = h * torch.sigmoid(h)
        a_off = 1.1 * h_off + 8 * u * a.abs()                             # |silu'| < 1.1; exponential, sum, division, weight
        we = w[t, j].unsqueeze(-1)
        out.index_put_((t,), we * (a @ down[e]), accumulate=True)
        off.index_put_((t,), we.abs() * (a_off @ down[e].abs() + a.abs() @ down[e].abs() * ((J + k + 24) * u)), accumulate=True)
    return out, off


SHAPES = [(1, 64, 8, 256, 128), (2, 32, 2, 128, 64), (5, 13, 3, 330, 201), (16, 64, 4, 1024, 256), (32, 8, 8, 64, 96), (32, 4, 1, 40, 8), (7, 1, 1, 33, 1), (3, 5, 2, 1, 7), (1, 300, 32, 72, 520), (8, 16, 4, 2056, 1032), (11, 2, 2, 3000, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,E,k,I,J", SHAPES)
def test_layer(dtype, tokens, E, k, I, J):
    t = TYPES[dtype]
    x, router = randn(tokens, I, seed=1, dtype=t), (randn(E, I, seed=2) * 1.5 / I ** 0.5).to(t)
    up, down = (randn(E, I, J, seed=3) * 2 / I ** 0.5).to(t), (randn(E, J, I, seed=4) / J ** 0.5).to(t)
    out, w, ids = ops.routed_experts_few(x, router, up, down, k)
    assert out.dtype == t and out.shape == x.shape and w.dtype == torch.float32 and ids.dtype == torch.int32
    check_choice(x, router, None, k, w, ids)
    want, off = layer64(x.double(), w.double(), ids.long(), up.double(), down.double())
    worst = ((out.double() - want).abs() - off - want.abs() * (torch.finfo(t).eps / 2) - (2.0 ** -25 if dtype == "f16" else 0)).max().item()
    assert worst <= 0, (worst, (out.double() - want).abs().max().item())
    again = ops.routed_experts_few(x, router, up, down, k)
    assert torch.equal(out, again[0]) and torch.equal(w, again[1]) and torch.equal(ids, again[2])


@pytest.mark.parametrize("options", [dict(score="sigmoid"), dict(renormalize=False), dict(score="sigmoid", renormalize=False, scale=2.5), dict(groups=4, top_groups=2), dict(groups=8, top_groups=3, group_top=1),
                                     dict(groups=4, top_groups=4, score="sigmoid", scale=0.5)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_choices(options, with_bias):
    tokens, E, k, I, J = 9, 24, 3, 96, 64
    x, router = randn(tokens, I, seed=1), randn(E, I, seed=2) * 1.5 / I ** 0.5
    up, down = randn(E, I, J, seed=3) * 2 / I ** 0.5, randn(E, J, I, seed=4) / J ** 0.5
    bias = 0.2 * randn(E, seed=5) if with_bias else None
    out, w, ids = ops.routed_experts_few(x, router, up, down, k, bias, **options)
    check_choice(x, router, bias, k, w, ids, **options)
    want, off = layer64(x.double(), w.double(), ids.long(), up.double(), down.double())
    assert ((out.double() - want).abs() <= off + want.abs() * 2.0 ** -24).all()


def test_equal_logits_and_extremes():
    """Equal keys: lower experts first; a token of zeros; one whose logits are not finite."""
    E, I, J, k = 40, 64, 32, 5
    up, down = randn(E, I, J, seed=3), randn(E, J, I, seed=4)
    x, router = randn(4, I, seed=1), randn(E, I, seed=2)
    x[1] = 0
    x[2] = float("nan")
    x[3] *= 1e30
    out, w, ids = ops.routed_experts_few(x, router, up, down, k)
    assert ids[1].tolist() == list(range(k)) and torch.equal(w[1], torch.full((k,), 0.2, device="cuda")) and not out[1].any()
    assert out[2].isnan().all()
    check_choice(x[:1], router, None, k, w[:1], ids[:1])
    same = torch.zeros_like(router)
    _, w, ids = ops.routed_experts_few(x[:1], same, up, down, k)
    assert ids[0].tolist() == list(range(k))


def grid4(*shape, seed, low=125, high=129):
    """Random values of 4 bits and scales of a few sizes: sums of their products are exact in float32."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    C = shape[-1]
    q = torch.randint(0, 256, (*shape[:-1], (C + 1) // 2), device="cuda", generator=gen, dtype=torch.int32).to(torch.uint8)
    if C % 2:
        q[..., -1] &= 15
    return q, torch.randint(low, high, (*shape[:-1], (C + 31) // 32), device="cuda", generator=gen, dtype=torch.int32).to(torch.uint8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,E,k,I,J", SHAPES)
def test_layer_on_4_bits(dtype, tokens, E, k, I, J):
    t = TYPES[dtype]
    (u, us), (d, ds) = grid4(E, J, I, seed=3, low=120, high=124), grid4(E, I, J, seed=4)
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.randint(-6, 7, (tokens, I), device="cuda", generator=gen).float() * 0.5).to(t)
    router = (randn(E, I, seed=2) * 1.5 / I ** 0.5).to(t)
    others = []
    out, w, ids = ops.routed_experts_few(x, router, u, d, k, up_scale=us, down_scale=ds)
    check_choice(x, router, None, k, w, ids)
    across = [q.transpose(1, 2).contiguous().transpose(1, 2) for q in (u, d)]             # the bytes of all channels together
    spare = torch.nn.functional.pad(across[1].transpose(1, 2), (0, 3, 0, 2))[:, :d.shape[2], :I].transpose(1, 2)      # ... experts and rows apart, rows that begin anywhere
    for uu, dd in ((across[0], d), (u, across[1]), (across[0], across[1]), (u, spare)):
        other = ops.routed_experts_few(x, router, uu, dd, k, up_scale=us, down_scale=ds)
        assert torch.equal(other[1], w) and torch.equal(other[2], ids)
        others.append(other[0])
    xq = fp4.values(*fp4.quantize(x), I)
    up, down = fp4.rows(u, us)[..., :I].transpose(1, 2), fp4.rows(d, ds)[..., :J].transpose(1, 2)
    want = torch.zeros(tokens, I, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for e in range(E):
        tt, j = (ids.long() == e).nonzero(as_tuple=True)
        if tt.numel():
            h = (xq[tt] @ up[e]).float()                     # exact: see grid4
            a = fp4.values(*fp4.quantize(h / (1 + torch.exp(-h))), J)
            we = w[tt, j].double().unsqueeze(-1)
            want.index_put_((tt,), we * (a @ down[e]), accumulate=True)
            size.index_put_((tt,), we * (a.abs() @ down[e].abs()), accumulate=True)
    # a block's products are exact; chains of at most J / 32 blocks, the joins, the CTAs and the choices
    off = size * ((J / 32 + k + 24) * 2.0 ** -24) + want.abs() * (torch.finfo(t).eps / 2) + (2.0 ** -25 if dtype == "f16" else 0)
    for got in (out, *others):
        worst = ((got.double() - want).abs() - off).max().item()
        assert worst <= 0, (worst, (got.double() - want).abs().max().item())


def test_strides_and_shapes():
    E, k, I, J = 6, 2, 48, 40
    big = randn(3, 2, 100, seed=1)
    router, up, down = randn(E, I, seed=2), randn(E, I, J, seed=3), randn(E, J, I, seed=4)
    for x in (big[:, 0, 3:51], big[..., 7:55], big[:, :, ::2][..., :48], big[0, 0, :48], big[:0, 0, :48]):
        out, w, ids = ops.routed_experts_few(x, router, up, down, k)
        ref = ops.routed_experts_few(x.contiguous().view(-1, I), router, up, down, k)
        assert out.shape == x.shape and ids.shape == (*x.shape[:-1], k)
        # logits are summed in another order where rows begin anywhere: sums of 48 products, at most 14 units of 2^-24 of sum |x r| < 100 off, 8e-5,
        # and weights by twice that
        assert ((out.view(-1, I) - ref[0]).abs() <= 2e-4 * ref[0].abs().sum(-1, keepdim=True)).all() and torch.equal(ids.view(-1, k), ref[2])
    x = randn(4, I, seed=9)
    want = ops.routed_experts_few(x, router, up, down, k)
    buf = torch.empty(E * I * J + 3, device="cuda")
    odd = buf[3:].view(E, I, J).copy_(up)                    # begins on 12 bytes
    for u, d in ((odd, down), (up.transpose(1, 2).contiguous().transpose(1, 2), down.transpose(0, 1).contiguous().transpose(0, 1))):
        assert torch.equal(ops.routed_experts_few(x, router, u, d, k)[0], want[0])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,E,k,I,J", [(1, 3, 3, 2047, 511), (9, 5, 3, 515, 771), (4, 6, 2, 1031, 257), (32, 3, 2, 266, 1001), (2, 2, 2, 37, 7001), (3, 4, 1, 9000, 15)])
@pytest.mark.parametrize("begin", [8, 3])
def test_wide_rows_that_begin_anywhere(dtype, tokens, E, k, I, J, begin):
    """Rows of no whole vectors, all experts among the chosen ones, NaN before and behind the weights; weights that begin on 16 bytes, or not."""
    t = TYPES[dtype]
    x, router = randn(tokens, I, seed=1, dtype=t), (randn(E, I, seed=2) * 1.5 / I ** 0.5).to(t)
    up, down = (torch.full((begin + E * I * J + 9,), float("nan"), device="cuda", dtype=t)[begin:begin + E * I * J] for _ in range(2))
    up, down = up.view(E, I, J).copy_(randn(E, I, J, seed=3) * 2 / I ** 0.5), down.view(E, J, I).copy_(randn(E, J, I, seed=4) / J ** 0.5)
    out, w, ids = ops.routed_experts_few(x, router, up, down, k)
    want, off = layer64(x.double(), w.double(), ids.long(), up.double(), down.double())
    worst = ((out.double() - want).abs() - off - want.abs() * (torch.finfo(t).eps / 2) - (2.0 ** -25 if dtype == "f16" else 0)).max().item()
    assert worst <= 0, (worst, (out.double() - want).abs().max().item())


@pytest.mark.parametrize("tokens,k", [(8, 32), (32, 8), (1, 32)])
@pytest.mark.parametrize("dtype,I,J", [("bf16", 96, 64), ("f16", 2049, 67), ("f32", 33, 20)])
def test_most_slots_and_experts(tokens, k, dtype, I, J):
    """1024 experts, 256 of tokens * top_k, in 16 and 32 bits and on weights in 4."""
    t, E = TYPES[dtype], 1024
    x, router = randn(tokens, I, seed=1, dtype=t), (randn(E, I, seed=2) * 1.5 / I ** 0.5).to(t)
    up, down = (randn(E, I, J, seed=3) * 2 / I ** 0.5).to(t), (randn(E, J, I, seed=4) / J ** 0.5).to(t)
    out, w, ids = ops.routed_experts_few(x, router, up, down, k)
    check_choice(x, router, None, k, w, ids)
    want, off = layer64(x.double(), w.double(), ids.long(), up.double(), down.double())
    assert ((out.double() - want).abs() - off - want.abs() * (torch.finfo(t).eps / 2) - (2.0 ** -25 if dtype == "f16" else 0)).max().item() <= 0
    (u, us), (d, ds) = grid4(E, J, I, seed=3, low=120, high=124), grid4(E, I, J, seed=4)
    out, w4, ids4 = ops.routed_experts_few(x, router, u, d, k, up_scale=us, down_scale=ds)
    assert torch.equal(w4, w) and torch.equal(ids4, ids)
    # the experts that were chosen alone, in another order: the same products, sums over the choices in their order
    used, place = ids.long().unique(return_inverse=True)
    again = torch.zeros(tokens, I, dtype=torch.float64, device="cuda")
    xq = fp4.values(*fp4.quantize(x), I)
    upq, downq = fp4.rows(u[used], us[used])[..., :I].transpose(1, 2), fp4.rows(d[used], ds[used])[..., :J].transpose(1, 2)
    size = torch.zeros_like(again)
    for e in range(used.numel()):
        tt, j = (place == e).nonzero(as_tuple=True)
        h = (xq[tt] @ upq[e]).float()                        # sums of 2049 products of multiples of 2^-9 below 2^4 * 2^-4 * 2049 < 2^12: below 2^24 steps of float32, to 2^-12
        a = fp4.values(*fp4.quantize(h / (1 + torch.exp(-h))), J)
        we = w[tt, j].double().unsqueeze(-1)
        again.index_put_((tt,), we * (a @ downq[e]), accumulate=True)
        size.index_put_((tt,), we * (a.abs() @ downq[e].abs()), accumulate=True)
    # where a value lies on a border between two of 4 bits up to the float32 sums' last bits the other one may be taken: a step of it, at most a third of the largest
    off = size * ((J / 32 + k + 24) * 2.0 ** -24) + again.abs() * (torch.finfo(t).eps / 2) + (2.0 ** -25 if dtype == "f16" else 0)
    wrong = (out.double() - again).abs() > off
    assert wrong.double().mean().item() <= (0.02 if I > 1000 else 0.0), wrong.double().mean().item()
    assert ((out.double() - again).abs() <= off + size / 3).all()


def test_blocks_that_are_not_numbers():
    """A block with the scale 255 makes NaN of what uses it and of nothing else; so does a row with a NaN."""
    tokens, E, k, I, J = 5, 4, 2, 160, 96
    (u, us), (d, ds) = grid4(E, J, I, seed=3, low=120, high=124), grid4(E, I, J, seed=4)
    x, router = randn(tokens, I, seed=1, dtype=torch.bfloat16), randn(E, I, seed=2, dtype=torch.bfloat16)
    good, _, ids = ops.routed_experts_few(x, router, u, d, k, up_scale=us, down_scale=ds)
    e = int(ids[0, 0])
    bad = ds.clone()
    bad[e, 7, 1] = 255
    bad[e, 133, 2] = 255
    out = ops.routed_experts_few(x, router, u, d, k, up_scale=us, down_scale=bad)[0]
    users = (ids == e).any(-1)
    gone = users.unsqueeze(-1) & torch.isin(torch.arange(I, device="cuda"), torch.tensor([7, 133], device="cuda"))
    assert torch.equal(out.isnan(), gone) and torch.equal(out[~gone], good[~gone])
    bad = us.clone()
    bad[e, 40, 0] = 255                                     # one activation, so a block of them, so all outputs
    out = ops.routed_experts_few(x, router, u, d, k, up_scale=bad, down_scale=ds)[0]
    assert torch.equal(out.isnan().all(-1), users) and torch.equal(out[~users], good[~users])
    y = x.clone()
    y[2, 50] = float("nan")
    out, _, other = ops.routed_experts_few(y, router, u, d, k, up_scale=us, down_scale=ds)
    rest = torch.arange(tokens, device="cuda") != 2
    assert out[2].isnan().all() and torch.equal(out[rest], good[rest]) and torch.equal(other[rest], ids[rest])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,E,k,I,J", [(19, 10, 3, 256, 1792), (19, 10, 3, 250, 1793), (2, 4, 4, 64, 9000), (32, 3, 1, 40, 20000), (8, 16, 4, 520, 2048)])
def test_wide_contraction_of_the_last_product(dtype, tokens, E, k, I, J):
    """Few columns and a long contraction: several clusters for a tile of columns."""
    t = TYPES[dtype]
    x, router = randn(tokens, I, seed=1, dtype=t), (randn(E, I, seed=2) * 1.5 / I ** 0.5).to(t)
    up, down = (randn(E, I, J, seed=3) * 2 / I ** 0.5).to(t), (randn(E, J, I, seed=4) / J ** 0.5).to(t)
    out, w, ids = ops.routed_experts_few(x, router, up, down, k)
    want, off = layer64(x.double(), w.double(), ids.long(), up.double(), down.double())
    worst = ((out.double() - want).abs() - off - want.abs() * (torch.finfo(t).eps / 2) - (2.0 ** -25 if dtype == "f16" else 0)).max().item()
    assert worst <= 0, (worst, (out.double() - want).abs().max().item())
    assert torch.equal(out, ops.routed_experts_few(x, router, up, down, k)[0])


def test_two_streams_and_two_graphs_at_once():
    """Calls on two streams, and replays of two graphs on them, that run beside each other: each has a workspace of its own."""
    E, k, I, J = 24, 3, 512, 320
    router, up, down = randn(E, I, seed=2, dtype=torch.bfloat16), randn(E, I, J, seed=3, dtype=torch.bfloat16), randn(E, J, I, seed=4, dtype=torch.bfloat16)
    (u, us), (d, ds) = grid4(E, J, I, seed=3, low=120, high=124), grid4(E, I, J, seed=4)
    xs = [randn(t, I, seed=10 + t, dtype=torch.bfloat16) for t in (1, 5, 16, 32)]

    def both(x):
        return ops.routed_experts_few(x, router, up, down, k)[0], ops.routed_experts_few(x, router, u, d, k, up_scale=us, down_scale=ds)[0]

    want = [both(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for n in range(12):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[s].append(both(xs[(n + s) % 4]))
    graphs = []
    for s in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[s]):
            graphs.append((g, [both(x) for x in xs]))
    torch.cuda.synchronize()
    for n in range(6):
        for (g, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for s in range(2):
        for n in range(12):
            assert all(torch.equal(a, b) for a, b in zip(got[s][n], want[(n + s) % 4]))
        for out, ref in zip(graphs[s][1], want):
            assert all(torch.equal(a, b) for a, b in zip(out, ref))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k", [(2, 1), (3, 2), (32, 1)])
@pytest.mark.parametrize("I,J", [(3, 1), (32, 32), (65, 31)])
def test_many_experts_of_a_small_layer(dtype, tokens, k, I, J):
    """1024 experts and next to no products: the list of the items needs more room than they do."""
    t, E = TYPES[dtype], 1024
    x, router = randn(tokens, I, seed=1, dtype=t), (randn(E, I, seed=2) * 1.5 / I ** 0.5).to(t)
    up, down = (randn(E, I, J, seed=3) * 2 / I ** 0.5).to(t), (randn(E, J, I, seed=4) / J ** 0.5).to(t)
    out, w, ids = ops.routed_experts_few(x, router, up, down, k)
    want, off = layer64(x.double(), w.double(), ids.long(), up.double(), down.double())
    assert ((out.double() - want).abs() - off - want.abs() * (torch.finfo(t).eps / 2) - (2.0 ** -25 if dtype == "f16" else 0)).max().item() <= 0


@pytest.mark.parametrize("E", [905, 1024])
@pytest.mark.parametrize("dtype,tokens,k,I,J", [("f32", 2, 1, 33, 70), ("f32", 3, 1, 65, 130), ("bf16", 2, 2, 31, 259), ("f16", 1, 3, 97, 65)])
def test_clusters_of_a_layer_with_many_experts(E, dtype, tokens, k, I, J):
    """Several CTAs to a tile and a list of items that is longer than all they add up: the sums that they hand to each other lie behind it."""
    t = TYPES[dtype]
    x, router = randn(tokens, I, seed=1, dtype=t), (randn(E, I, seed=2) * 1.5 / I ** 0.5).to(t)
    up, down = (randn(E, I, J, seed=3) * 2 / I ** 0.5).to(t), (randn(E, J, I, seed=4) / J ** 0.5).to(t)
    out, w, ids = ops.routed_experts_few(x, router, up, down, k)
    want, off = layer64(x.double(), w.double(), ids.long(), up.double(), down.double())
    off = off + want.abs() * (torch.finfo(t).eps / 2) + (2.0 ** -25 if dtype == "f16" else 0)
    for _ in range(8):
        assert ((out.double() - want).abs() - off).max().item() <= 0
        out = ops.routed_experts_few(x, router, up, down, k)[0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,E,k,I,J", [(1, 5, 3, 2048, 512), (9, 6, 2, 264, 520), (4, 3, 2, 48, 40), (20, 2, 1, 8, 4096), (3, 33, 4, 512, 8)])
@pytest.mark.parametrize("up_begin,down_begin", [(1, 0), (0, 3), (2, 1), (5, 7)])
def test_weights_that_begin_anywhere(dtype, tokens, E, k, I, J, up_begin, down_begin):
    """Slices of a larger buffer, NaN right before and behind them: the bits that weights on 16 bytes give, and no copy of them."""
    t = TYPES[dtype]
    x, router = randn(tokens, I, seed=1, dtype=t), (randn(E, I, seed=2) * 1.5 / I ** 0.5).to(t)
    whole = [(randn(E, I, J, seed=3) * 2 / I ** 0.5).to(t), (randn(E, J, I, seed=4) / J ** 0.5).to(t)]
    up, down = (torch.full((n + w.numel() + 9,), float("nan"), device="cuda", dtype=t)[n:n + w.numel()].view(w.shape).copy_(w) for n, w in zip((up_begin, down_begin), whole))
    want = ops.routed_experts_few(x, router, *whole, k)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = ops.routed_experts_few(x, router, up, down, k)
    grown = torch.cuda.max_memory_allocated() - before
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if I * J > 100000:                                       # (the workspace is eight parts of the first product, the sums of the second, logits and outputs)
        assert grown < up.numel() * t.itemsize


@pytest.mark.parametrize("fp4_weights", [False, True])
def test_padded_tokens_that_are_no_numbers(fp4_weights):
    """Rows of a padded batch that hold anything: valid choices, each expert once, and not a bit of the other rows' results."""
    tokens, E, k, I, J = 12, 9, 4, 136, 72
    x, router = randn(tokens, I, seed=1, dtype=torch.bfloat16), randn(E, I, seed=2, dtype=torch.bfloat16)
    if fp4_weights:
        (u, us), (d, ds) = grid4(E, J, I, seed=3, low=120, high=124), grid4(E, I, J, seed=4)
        run = lambda x: ops.routed_experts_few(x, router, u, d, k, up_scale=us, down_scale=ds)
    else:
        up, down = randn(E, I, J, seed=3, dtype=torch.bfloat16), randn(E, J, I, seed=4, dtype=torch.bfloat16)
        run = lambda x: ops.routed_experts_few(x, router, up, down, k)
    want = run(x)
    y = x.clone()
    y[1], y[4], y[5], y[11] = float("nan"), float("inf"), -float("inf"), 3e38
    y[7, 3], y[8, 100] = float("nan"), -float("inf")
    rest = torch.tensor([0, 2, 3, 6, 9, 10], device="cuda")
    first = run(y)
    for _ in range(3):
        out, w, ids = run(y)
        assert ((ids >= 0) & (ids < E)).all() and all(len(set(r)) == k for r in ids.tolist())
        # (experts' tokens are read in fours: which ones share a read is no matter of their sums)
        assert torch.equal(out[rest], want[0][rest]) and torch.equal(w[rest], want[1][rest]) and torch.equal(ids[rest], want[2][rest])
        assert torch.equal(ids, first[2]) and torch.equal(out.isnan(), first[0].isnan()) and out[1].isnan().all()


def test_weights_beyond_32_bits():
    """Experts that lie more than 2^31 elements, and 2^32 bytes, behind the first one."""
    E, I, J = 33, 8192, 8192
    x = randn(3, I, seed=1, dtype=torch.bfloat16).abs()
    router = torch.zeros(E, I, device="cuda", dtype=torch.bfloat16)
    router[E - 1] = 1                                        # all tokens choose the last one
    up, down = (torch.empty(E, a, b, device="cuda", dtype=torch.bfloat16) for a, b in ((I, J), (J, I)))
    up[E - 1], down[E - 1] = randn(I, J, seed=2) * 2 / I ** 0.5, randn(J, I, seed=3) / J ** 0.5
    out, w, ids = ops.routed_experts_few(x, router, up, down, 1)
    assert (ids == E - 1).all()
    want, off = layer64(x.double(), w.double(), torch.zeros_like(ids).long(), up[E - 1:].double(), down[E - 1:].double())
    assert ((out.double() - want).abs() - off - want.abs() * 2.0 ** -8).max().item() <= 0
    del up, down
    E = 129                                                  # in 4 bits an expert's matrix is 2^25 bytes
    router = torch.zeros(E, I, device="cuda", dtype=torch.bfloat16)
    router[E - 1] = 1
    up, down = (torch.empty(E, I, I // 2, device="cuda", dtype=torch.uint8) for _ in range(2))
    us, ds = (torch.empty(E, I, I // 32, device="cuda", dtype=torch.uint8) for _ in range(2))
    (up[E - 1], us[E - 1]), (down[E - 1], ds[E - 1]) = grid4(J, I, seed=3, low=120, high=124), grid4(I, J, seed=4)
    out, w, ids = ops.routed_experts_few(x, router, up, down, 1, up_scale=us, down_scale=ds)
    assert (ids == E - 1).all() and not out.isnan().any()
    again = ops.routed_experts_few(x, router[E - 1:], up[E - 1:], down[E - 1:], 1, up_scale=us[E - 1:], down_scale=ds[E - 1:])[0]
    assert torch.equal(out, again)


def test_refusals():
    E, I, J = 4, 16, 8
    x, router, up, down = randn(3, I), randn(E, I), randn(E, I, J), randn(E, J, I)
    few = ops.routed_experts_few
    for bad in (lambda: few(x, router, up, down, 0), lambda: few(x, router, up, down, 5), lambda: few(x.half(), router, up, down, 2), lambda: few(x, router, up.half(), down, 2), lambda: few(x, router[:, :8], up, down, 2),
                lambda: few(x, router, up[:3], down, 2), lambda: few(x, router, down, up, 2), lambda: few(randn(33, I), router, up, down, 2), lambda: few(x, router, up, down, 2, score="relu"),
                lambda: few(x, router, up, down, 2, groups=3), lambda: few(x, router, up, down, 2, torch.zeros(3, device="cuda")), lambda: few(x, router, up, down, 2, up_scale=x),
                lambda: few(randn(32, I), randn(64, I), randn(64, I, J), randn(64, J, I), 9)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: few(x.cpu(), router, up, down, 2), lambda: few(x, router, up, down.cpu(), 2), lambda: few(x, router, up, down, 2, torch.zeros(E))):
        with pytest.raises(RuntimeError):
            bad()


def test_captured_and_replayed():
    """Two graphs of the same weights, replayed on two streams at once with other inputs."""
    E, k, I, J = 16, 4, 256, 128
    router, up, down = (randn(E, I, seed=2) / 16).bfloat16(), randn(E, I, J, seed=3).bfloat16() / 8, randn(E, J, I, seed=4).bfloat16() / 8
    xs = [randn(n, I, seed=n).bfloat16() for n in (1, 6)]
    want = [[ops.routed_experts_few(x * f, router, up, down, k)[0] for f in (1, 2)] for x in xs]
    graphs, ins, outs = [], [], []
    for x in xs:
        ins.append(x.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.routed_experts_few(ins[-1], router, up, down, k)[0])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for i, f in enumerate((1, 2, 1)):
        for x, to in zip(xs, ins):
            to.copy_(x * f)
        torch.cuda.synchronize()
        for _ in range(20):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w[f - 1])


# ---- modules ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_few_is_the_layer(dtype):
    import expertscattergather_b200 as egs
    torch.manual_seed(3)
    layer = egs.RoutedExperts(16, 256, 192, 4, balance=True, groups=4, top_groups=2).cuda().to(TYPES[dtype])
    layer.router.balance.copy_(0.05 * randn(16, seed=1))
    x = randn(3, 5, 256, seed=2, dtype=TYPES[dtype])
    y, full = layer.few(x), layer(x)
    assert y.shape == x.shape and y.dtype == x.dtype and not y.requires_grad and full.requires_grad
    # float32: sums in another order.  bf16: forward rounds logits, h, silu(h) and rows, 2^-9 each in the mean of the squares, and logits move the weights
    assert (y - full).norm() <= (1e-5 if dtype == "f32" else 2e-2) * full.norm()


@pytest.mark.parametrize("tokens", [1, 32, 33, 700])
@pytest.mark.parametrize("float32_rows", [False, True])
def test_served_in_4_bits(tokens, float32_rows):
    """The served layer against the definition on the values that its weights stand for, few tokens and many."""
    import expertscattergather_b200 as egs
    torch.manual_seed(4)
    E, I, J, k = 12, 320, 200, 3
    layer = egs.RoutedExperts(E, I, J, k, float32_rows=float32_rows).cuda().bfloat16()
    served = layer.quantized(bits=4)
    x = randn(tokens, I, seed=tokens, dtype=torch.bfloat16)
    y = served(x)
    assert y.shape == x.shape and y.dtype == x.dtype
    if tokens <= ops.FEW_TOKENS:
        _, w, ids = ops.routed_experts_few(x, served.router.W, served.up, served.down, k, up_scale=served.up_scale, down_scale=served.down_scale)
    else:
        w, ids = served.router(x)
    up, down = fp4.rows(served.up, served.up_scale).transpose(1, 2), fp4.rows(served.down, served.down_scale).transpose(1, 2)
    xq = fp4.values(*fp4.quantize(x), I)
    want = torch.zeros(tokens, I, dtype=torch.float64, device="cuda")
    for e in range(E):
        t, j = (ids.long() == e).nonzero(as_tuple=True)
        h = (xq[t] @ up[e]).float()
        a = fp4.values(*fp4.quantize(h / (1 + torch.exp(-h))), J)
        want.index_put_((t,), w[t, j].double().unsqueeze(-1) * (a @ down[e]), accumulate=True)
    # rows and the output are rounded to bf16, 0.0017 each in the 2-norm; a value of h that falls the other way at a border is a third of itself off, and
    # fewer than 2^-17 of them lie so near
    assert (y.double() - want).norm() <= 4e-3 * want.norm()


def test_served_in_4_bits_on_another_stream():
    import expertscattergather_b200 as egs
    torch.manual_seed(5)
    served = egs.RoutedExperts(8, 128, 96, 2).cuda().bfloat16().quantized(bits=4)
    xs = [randn(n, 128, seed=n, dtype=torch.bfloat16) for n in (4, 200)]
    want = [served(x) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [served(x) for x in xs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,E,k,I,J", [(1, 8, 2, 256, 96), (7, 5, 3, 330, 201), (32, 4, 2, 96, 1032)])
@pytest.mark.parametrize("x_far,up_far,down_far", [(120, -118, 0), (-118, 120, 0), (0, 118, -118), (0, 60, 40), (100, -40, -60), (-110, 118, 90)])
def test_layer_on_4_bits_of_far_scales(dtype, tokens, E, k, I, J, x_far, up_far, down_far):
    """Rows, weights and activations of magnitudes at the ends of float32 whose products are ordinary numbers."""
    t = TYPES[dtype]
    (u, us), (d, ds) = grid4(E, J, I, seed=3, low=124 + up_far, high=128 + up_far), grid4(E, I, J, seed=4, low=125 + down_far, high=129 + down_far)
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.ldexp(torch.randint(-6, 7, (tokens, I), device="cuda", generator=gen).float() * 0.5, torch.tensor(x_far, device="cuda")).to(t)
    router = torch.ldexp(randn(E, I, seed=2) * 1.5 / I ** 0.5, torch.tensor(-x_far, device="cuda")).to(t)
    xq = fp4.values(*fp4.quantize(x), I)
    up, down = fp4.rows(u, us)[..., :I].transpose(1, 2), fp4.rows(d, ds)[..., :J].transpose(1, 2)
    for uu, dd in ((u, d), tuple(q.transpose(1, 2).contiguous().transpose(1, 2) for q in (u, d))):
        out, w, ids = ops.routed_experts_few(x, router, uu, dd, k, up_scale=us, down_scale=ds)
        want = torch.zeros(tokens, I, dtype=torch.float64, device="cuda")
        size = torch.zeros_like(want)
        for e in range(E):
            tt, j = (ids.long() == e).nonzero(as_tuple=True)
            if tt.numel():
                h = (xq[tt] @ up[e]).float()                 # exact: see grid4
                a = fp4.values(*fp4.quantize(h / (1 + torch.exp(-h))), J)
                we = w[tt, j].double().unsqueeze(-1)
                want.index_put_((tt,), we * (a @ down[e]), accumulate=True)
                size.index_put_((tt,), we * (a.abs() @ down[e].abs()), accumulate=True)
        assert want.isfinite().all() and want.abs().max() < 2.0 ** 126
        off = size * ((J / 32 + k + 24) * 2.0 ** -24) + want.abs() * (torch.finfo(t).eps / 2)      # (as test_layer_on_4_bits)
        assert ((out.double() - want).abs() - off).max().item() <= 0


def test_served_in_4_bits_under_autocast():
    """A float32 layer whose rows come in 16 bits: few tokens give what they give among many."""
    import expertscattergather_b200 as egs
    torch.manual_seed(6)
    served = egs.RoutedExperts(8, 128, 96, 2).cuda().quantized(bits=4)
    x = randn(40, 128, seed=2, dtype=torch.bfloat16)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        many, few = served(x), served(x[:5])
    assert few.dtype == many.dtype == torch.bfloat16
    # the router's product may be summed in another order: logits are off by a step of bf16 at most, 2^-8 of themselves (which are below 2), weights by as much
    assert (few.float() - many[:5].float()).norm() <= 2e-2 * many[:5].float().norm()


@pytest.mark.parametrize("tokens,E,I,J,k", [(4, 4, 1024, 3000, 4), (32, 4, 1024, 3000, 4), (12, 8, 2048, 1030, 8), (33, 8, 2048, 1030, 8)])
def test_served_large_layer_in_4_bits(tokens, E, I, J, k):
    """Few tokens of a large layer go through the operators for many, with float32 rows ahead of the sum."""
    import expertscattergather_b200 as egs
    torch.manual_seed(8)
    served = egs.RoutedExperts(E, I, J, k).cuda().bfloat16().quantized(bits=4)
    x = randn(tokens, I, seed=tokens, dtype=torch.bfloat16)
    ops.check_status()
    y = served(x)
    one_call = tokens <= 4
    w, ids = ops.routed_experts_few(x, served.router.W, served.up, served.down, k, up_scale=served.up_scale, down_scale=served.down_scale)[1:] if one_call else served.router(x)
    up, down = fp4.rows(served.up, served.up_scale).transpose(1, 2), fp4.rows(served.down, served.down_scale).transpose(1, 2)
    xq = fp4.values(*fp4.quantize(x), I)
    want = torch.zeros(tokens, I, dtype=torch.float64, device="cuda")
    for e in range(E):
        t, j = (ids.long() == e).nonzero(as_tuple=True)
        h = (xq[t] @ up[e]).float()
        a = fp4.values(*fp4.quantize(h / (1 + torch.exp(-h))), J)[:, :J]
        want.index_put_((t,), w[t, j].double().unsqueeze(-1) * (a @ down[e][:J]), accumulate=True)
    # (as test_served_in_4_bits; one rounding to bf16 where rows are float32)
    assert (y.double() - want).norm() <= (2.5e-3 if tokens <= ops.FEW_TOKENS else 4e-3) * want.norm()
    ops.check_status()
