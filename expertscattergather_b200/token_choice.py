"""Layers whose tokens choose their experts: the router, the experts' products with their gradients, and the layer made of them, for
training and, with weights in 8 or 4 bits, for serving.

    layer = RoutedExperts(E, I, J, top_k).cuda()        # x [..., I] -> [..., I]
    served = layer.quantized()                          # the same layer on int8 weights, no gradients
    served = layer.quantized(bits=4)                    # ... on weights in 4 bits
    y = layer.few(x)                                    # a decoding step's few tokens, no gradients

No counterpart in the reference, whose experts choose their tokens (``ExpertGather`` / ``ExpertScatter``).  The operators are those of
``ops``; here they have gradients, first ones alone: a second derivative through them raises.  ``torch.compile`` runs the operators as they
are, between the graphs that it makes of what lies around them; with ``fullgraph=True`` it refuses these layers.
"""
from __future__ import annotations

import copy
import math

import torch
from torch import nn
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from . import ops

__all__ = ["RouteTokensFunction", "ExpertMatmulFunction", "CombineFunction", "route_tokens", "expert_matmul", "combine", "TokenRouter",
           "RoutedExperts", "RoutedExpertsInt8", "RoutedExpertsFp4"]


class RouteTokensFunction(torch.autograd.Function):
    """``apply(logits, bias, top_k, options) -> (weights, experts)``; options as ``ops.route_tokens`` takes them, as a dict."""

    @staticmethod
    def forward(ctx, logits, bias, top_k, options):
        weights, experts = ops.route_tokens(logits, top_k, bias, **options)
        ctx.save_for_backward(logits, experts)
        ctx.options = {n: options[n] for n in ("score", "renormalize", "scale") if n in options}
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _):
        logits, experts = ctx.saved_tensors
        return ops.route_tokens_backward(dweights, logits, experts, **ctx.options), None, None, None


class ExpertMatmulFunction(torch.autograd.Function):
    """``apply(X, W, plan, rows, out_dtype=None) -> Y`` (``ops.expert_matmul``, W [E, C, N]).  With float32 rows of 16-bit tensors the rows of
    dX are float32 too until they have been summed; dY is rounded to the tensors' type, as what the tensor cores multiply."""

    @staticmethod
    def forward(ctx, X, W, plan, rows, out_dtype=None):
        ctx.save_for_backward(X, W)
        ctx.plan, ctx.rows, ctx.out_dtype = plan, rows, out_dtype
        return ops.expert_matmul(X, W, plan, rows=rows, out_dtype=out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dY):
        X, W = ctx.saved_tensors
        dY = dY.to(X.dtype)
        dX = dW = None
        if ctx.needs_input_grad[0]:
            if ctx.rows == "tokens":                       # a token's row went to each of its experts
                dX = ops.combine(ops.expert_matmul(dY, W, ctx.plan, rows="sorted", w_layout="nc", out_dtype=ctx.out_dtype), None, ctx.plan, out_dtype=X.dtype)
            else:
                dX = ops.expert_matmul(dY, W, ctx.plan, rows="sorted", w_layout="nc")
            dX = dX.view(X.shape)
        if ctx.needs_input_grad[1]:
            dW = ops.expert_dweight(X, dY, ctx.plan, rows=ctx.rows)
        return dX, dW, None, None, None


class CombineFunction(torch.autograd.Function):
    """``apply(Y, weights, plan, out_dtype=None) -> out`` (``ops.combine``)."""

    @staticmethod
    def forward(ctx, Y, weights, plan, out_dtype=None):
        ctx.save_for_backward(Y, weights)
        ctx.plan = plan
        return ops.combine(Y, weights, plan, out_dtype=out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dOut):
        Y, weights = ctx.saved_tensors
        if weights is None or weights.dtype in (torch.float32, Y.dtype):
            return (*ops.combine_backward(dOut.to(Y.dtype), Y, weights, ctx.plan), None, None)
        dY, dweights = ops.combine_backward(dOut.to(Y.dtype), Y, weights.to(Y.dtype), ctx.plan)
        return dY, dweights.to(weights.dtype), None, None


def route_tokens(logits, top_k, bias=None, **options):
    """``ops.route_tokens`` with a gradient for the logits."""
    return RouteTokensFunction.apply(logits, bias, top_k, options)


def expert_matmul(X, W, plan, *, rows="tokens", out_dtype=None):
    """``ops.expert_matmul`` (W [E, C, N]) with gradients for X and W."""
    return ExpertMatmulFunction.apply(X, W, plan, rows, out_dtype)


def combine(Y, weights, plan, *, out_dtype=None):
    """``ops.combine`` with gradients for Y and the weights."""
    return CombineFunction.apply(Y, weights, plan, out_dtype)


class TokenRouter(nn.Module):
    """``forward(x [..., I]) -> (weights [..., top_k], experts [..., top_k])``: the logits are ``x @ W.T`` (W [E, I]), options as for
    ``ops.route_tokens``.  With ``balance`` there is a buffer of that name, [E] in float32 whatever the module's type, that is added to the
    keys of the choice; no gradient reaches it, :meth:`adjust` moves it against the load."""

    def __init__(self, E: int, I: int, top_k: int, balance: bool = False, **options):
        super().__init__()
        self.E, self.I, self.top_k, self.options = E, I, top_k, options
        self.W = nn.Parameter(torch.empty(E, I))
        self.register_buffer("balance", torch.zeros(E) if balance else None)
        nn.init.uniform_(self.W, -1 / math.sqrt(I), 1 / math.sqrt(I))

    def _apply(self, fn, *args, **kwargs):
        kept = self.balance
        super()._apply(fn, *args, **kwargs)
        if kept is not None and self.balance.dtype != torch.float32:      # steps of an adjustment are too small for 16 bits
            self.balance = kept.to(self.balance.device)
        return self

    def forward(self, x):
        return route_tokens(F.linear(x, self.W), self.top_k, self.balance, **self.options)

    @torch.no_grad()
    def adjust(self, plan: ops.ExpertPlan, rate: float) -> None:
        """Lowers the keys of experts with more rows than the mean by ``rate``, raises those of the others (no synchronisation)."""
        if self.balance is None:
            raise RuntimeError("the router was made without balance")
        counts = plan.counts().float()
        self.balance += rate * torch.sign(counts.mean() - counts)


class RoutedExperts(nn.Module):
    """``out[t] = sum_j weights[t, j] * act(x[t] @ up[e]) @ down[e]`` over the experts ``e`` that the router chose for token t;
    x [..., I] -> [..., I], up [E, I, J], down [E, J, I], act = SiLU.  No token is dropped, whatever the load of an expert.  Options go to
    :class:`TokenRouter`.  In 16 bits the rows between the products are rounded to the tensors' type, each once, as the module's
    activations are; sums over tokens, experts and features are float32.  With ``float32_rows`` products leave float32 rows, so that only what
    they are made into is rounded (``act(..)``, the output, gradients ahead of their products): about half of the rounding errors' variance,
    for twice the bytes of those rows."""

    def __init__(self, E: int, I: int, J: int, top_k: int, *, float32_rows: bool = False, **options):
        super().__init__()
        self.E, self.I, self.J, self.float32_rows = E, I, J, float32_rows
        self.router = TokenRouter(E, I, top_k, **options)
        self.up = nn.Parameter(torch.empty(E, I, J))
        self.down = nn.Parameter(torch.empty(E, J, I))
        nn.init.uniform_(self.up, -1 / math.sqrt(I), 1 / math.sqrt(I))
        nn.init.uniform_(self.down, -1 / math.sqrt(J), 1 / math.sqrt(J))
        self.plan = None                                   # of the last call: what router.adjust takes

    def forward(self, x):
        weights, experts = self.router(x)
        self.plan = plan = ops.plan_experts(experts, self.E)
        wide = torch.float32 if self.float32_rows else None
        h = F.silu(expert_matmul(x, self.up, plan, out_dtype=wide)).to(x.dtype)
        return combine(expert_matmul(h, self.down, plan, rows="sorted", out_dtype=wide), weights, plan, out_dtype=x.dtype).view(x.shape)

    @torch.no_grad()
    def few(self, x):
        """The layer for a decoding step's few tokens (``ops.routed_experts_few``, and its limits), without gradients.  Logits and what lies between
        the products stay float32 here, so that results are nearer to the definition than :meth:`forward`'s."""
        return ops.routed_experts_few(x, self.router.W, self.up, self.down, self.router.top_k, self.router.balance, **self.router.options)[0]

    @torch.no_grad()
    def quantized(self, bits: int = 8):
        """The layer for serving, on weights in 8 bits (:class:`RoutedExpertsInt8`) or 4 (:class:`RoutedExpertsFp4`)."""
        if bits not in (8, 4):
            raise ValueError("bits must be 8 or 4")
        return RoutedExpertsInt8(self) if bits == 8 else RoutedExpertsFp4(self)


def _in_pitch(q):
    """Rows of bytes a multiple of 16 apart, as ``ops.quantize_rows`` lays them out and the products read them without a copy."""
    pitch = (q.shape[-1] + 15) // 16 * 16
    if q.stride(-1) == 1 and q.stride(-2) == pitch:
        return q
    rows = q.new_zeros((*q.shape[:-1], pitch))[..., :q.shape[-1]]
    return rows.copy_(q)


class RoutedExpertsInt8(nn.Module):
    """A :class:`RoutedExperts` for serving: weights in 8 bits with a scale for each output channel, rows quantised on the way into each
    product with a scale for each row.  It has a router of its own, a copy without gradients: what becomes of the layer it was made from,
    or of its type or device, does not reach it, nor the other way round.  The scales stay in float32 whatever the module is cast to."""

    def __init__(self, layer: RoutedExperts):
        super().__init__()
        self.E, self.float32_rows = layer.E, layer.float32_rows
        self.router = copy.deepcopy(layer.router).requires_grad_(False)
        for name in ("up", "down"):
            q, scale = ops.quantize_rows(getattr(layer, name).detach().transpose(1, 2))
            self.register_buffer(name, q)
            self.register_buffer(name + "_scale", scale)

    def _apply(self, fn, *args, **kwargs):
        kept = {name: getattr(self, name + "_scale") for name in ("up", "down")}
        super()._apply(fn, *args, **kwargs)
        for name, scale in kept.items():
            setattr(self, name, _in_pitch(getattr(self, name)))           # (a copy to another device has its rows together)
            if getattr(self, name + "_scale").dtype != torch.float32:
                setattr(self, name + "_scale", scale.to(getattr(self, name).device))
        return self

    @torch.no_grad()
    def forward(self, x):
        weights, experts = self.router(x)
        plan = ops.plan_experts(experts, self.E)
        rows = torch.float32 if self.float32_rows else x.dtype
        h = F.silu(ops.expert_matmul_int8(*ops.quantize_rows(x), self.up, self.up_scale, plan, out_dtype=rows))
        y = ops.expert_matmul_int8(*ops.quantize_rows(h), self.down, self.down_scale, plan, rows="sorted", out_dtype=rows)
        return ops.combine(y, weights, plan, out_dtype=x.dtype).view(x.shape)


class RoutedExpertsFp4(nn.Module):
    """A :class:`RoutedExperts` for serving: weights in 4 bits (``ops.quantize_rows_fp4`` along their contractions), rows rounded to 4 bits on the way
    into each product.  A call of a few tokens (``ops.FEW_TOKENS``, ``ops.FEW_SLOTS``) that need not read weights over and over is one of
    ``ops.routed_experts_few``, whose logits stay float32; in others the router is the module's own.  Rows that are summed over a token's experts are float32 up to
    ``ops.FEW_TOKENS`` tokens, and beyond, as :class:`RoutedExperts` has them, of x's type unless the layer had ``float32_rows``.  It has a router of its own, as
    :class:`RoutedExpertsInt8` has."""

    def __init__(self, layer: RoutedExperts):
        super().__init__()
        self.E, self.I, self.float32_rows = layer.E, layer.I, layer.float32_rows
        self.router = copy.deepcopy(layer.router).requires_grad_(False)
        for name in ("up", "down"):
            q, scale = ops.quantize_rows_fp4(getattr(layer, name).detach().transpose(1, 2))
            self.register_buffer(name, q)
            self.register_buffer(name + "_scale", scale)

    def _apply(self, fn, *args, **kwargs):
        super()._apply(fn, *args, **kwargs)
        for name in ("up", "down", "up_scale", "down_scale"):
            setattr(self, name, _in_pitch(getattr(self, name)))           # (a copy to another device has its rows together)
        return self

    def _in_one_call(self, x) -> bool:
        """Whether ``ops.routed_experts_few`` takes x, and sooner than the separate operators.  It shares a read of an expert's weights among four tokens: with no more
        nothing is read twice.  With more its time goes with the slots and a matrix's size, that of the operators, 30 to 45 us of launches aside, with the experts that are used.
        us in a graph, one call and five: 32 tokens, 4 of 8 experts, 2048 x 512 33 and 32, 2048 x 2048 85 and 39, 4096 x 4096 273 and 75; 16 tokens, 8 of 64, 2048 x 512 52 and 55,
        2048 x 2048 140 and 90; 8 tokens, 2 of 8, 4096 x 4096 73 and 77, 8 of 8, 124 and 76; 4 tokens, 8 of 8, 77 and 81.  (Of 150 sizes the choice costs 0.4 % over the better one in the
        mean, the host's 14 and 46 us counted for half of them.)"""
        tokens = x.numel() // max(self.I, 1)
        slots = tokens * self.router.top_k
        if tokens > ops.FEW_TOKENS or slots > ops.FEW_SLOTS or x.dtype != self.router.W.dtype:       # (autocast hands over rows of another type, which the router's product takes)
            return False
        return tokens <= 4 or slots * self.I * self.up.shape[1] <= 200_000_000

    @torch.no_grad()
    def forward(self, x):
        if self._in_one_call(x):
            return ops.routed_experts_few(x, self.router.W, self.up, self.down, self.router.top_k, self.router.balance, up_scale=self.up_scale, down_scale=self.down_scale,
                                          **self.router.options)[0]
        weights, experts = self.router(x)
        plan = ops.plan_experts(experts, self.E)
        h = ops.expert_matmul_fp4_rows(*ops.quantize_rows_fp4(x), self.up, self.up_scale, plan, activation="silu")
        wide = self.float32_rows or x.numel() <= ops.FEW_TOKENS * self.I
        y = ops.expert_matmul_fp4(*h, self.down, self.down_scale, plan, rows="sorted", out_dtype=torch.float32 if wide else x.dtype)
        return ops.combine(y, weights, plan, out_dtype=x.dtype).view(x.shape)
