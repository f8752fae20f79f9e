"""Rows in 4 bits, from their definition in float64 (torch, any device)."""
import torch

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize(X):
    """X [..., C] -> codes [..., blocks * 32] and scale bytes [..., blocks], zeros behind the row's end."""
    x = X.double()
    C = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -C % 32)).unflatten(-1, ((C + 31) // 32, 32))
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    mantissa, exponent = torch.frexp(torch.where(bad, torch.ones_like(top), top))         # top = mantissa 2^exponent, mantissa in [.5, 1)
    exponent = (exponent - 3 + (mantissa > 0.875)).clamp(min=-127)                        # the smallest j with top <= 7 2^j
    exponent = torch.where(top == 0, torch.full_like(exponent, -127), exponent)
    x = torch.where(bad.unsqueeze(-1), torch.zeros_like(x), x)
    m = torch.ldexp(x.abs(), -exponent.unsqueeze(-1))
    code = sum((m > b).int() for b in (0.25, 1.25, 2.5, 5.0)) + sum((m >= b).int() for b in (0.75, 1.75, 3.5))
    code = code + 8 * torch.signbit(x).int()
    return code.flatten(-2), torch.where(bad, torch.full_like(exponent, 255), exponent + 127)


def pack(codes):
    return (codes[..., ::2] + 16 * codes[..., 1::2]).to(torch.uint8)


def codes_of(q):
    return torch.stack((q % 16, q // 16), -1).flatten(-2).int()


def values(codes, scale, C):
    """What codes [..., >= C] stand for, float64."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64, device=codes.device)
    s = scale.double()
    power = torch.where(s == 255, torch.full_like(s, float("nan")), torch.exp2(s - 127))
    return level[codes[..., :C].long()] * power.repeat_interleave(32, -1)[..., :C]


def rows(q, scale):
    return values(codes_of(q), scale, 2 * q.shape[-1])
