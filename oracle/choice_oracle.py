"""Operators for tokens that choose experts, from their definitions in float64 (torch, any device)."""
import torch


def scores(logits, score):
    x = logits.double()
    if score == "sigmoid":
        return torch.sigmoid(x)
    top = x.amax(-1, keepdim=True)
    return torch.where(top == -float("inf"), torch.zeros_like(x), torch.softmax(x, -1))


def group_values(key, groups, group_top):
    per = key.shape[-1] // groups
    best = key.view(*key.shape[:-1], groups, per).sort(dim=-1, descending=True).values
    return best[..., :group_top].sum(-1)


def weights_of(s, experts, renormalize, scale):
    w = s.gather(-1, experts.long())
    if renormalize:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
    return w * scale


def plan(experts, E):
    """offsets, slots, position of the flat ids (stable sort; ids outside [0, E) behind the others)."""
    ids = experts.flatten().long()
    ids = torch.where((ids < 0) | (ids >= E), torch.full_like(ids, E), ids)
    slots = ids.sort(stable=True).indices
    offsets = torch.zeros(E + 1, dtype=torch.long, device=ids.device)
    offsets[1:] = torch.bincount(ids, minlength=E + 1)[:E].cumsum(0)
    position = torch.empty_like(slots)
    position[slots] = torch.arange(slots.numel(), device=ids.device)
    return offsets, slots, torch.where(ids == E, ~position, position)


def matmul(X, W, experts, E, rows):
    """Sorted rows Y, and the same product of magnitudes (what rounding errors are measured against).  W [E, C, N]."""
    offsets, slots, _ = plan(experts, E)
    k = experts.shape[-1]
    n = slots.numel()
    Y = torch.zeros(n, W.shape[2], dtype=torch.float64, device=X.device)
    size = torch.zeros_like(Y)
    Xs = X.reshape(-1, X.shape[-1])
    Xs = Xs[slots // k] if rows == "tokens" else Xs
    for e in range(E):
        a, b = offsets[e].item(), offsets[e + 1].item()
        if b > a:
            Y[a:b] = Xs[a:b].double() @ W[e].double()
            size[a:b] = Xs[a:b].double().abs() @ W[e].double().abs()
    return Y, size


def dweight(X, dY, experts, E, rows):
    offsets, slots, _ = plan(experts, E)
    k = experts.shape[-1]
    Xs = X.reshape(-1, X.shape[-1])
    Xs = Xs[slots // k] if rows == "tokens" else Xs
    dW = torch.zeros(E, Xs.shape[1], dY.shape[1], dtype=torch.float64, device=X.device)
    size = torch.zeros_like(dW)
    for e in range(E):
        a, b = offsets[e].item(), offsets[e + 1].item()
        if b > a:
            dW[e] = Xs[a:b].double().t() @ dY[a:b].double()
            size[e] = Xs[a:b].double().abs().t() @ dY[a:b].double().abs()
    return dW, size


def combine(Y, weights, position, tokens, k):
    pos = position.view(tokens, k).long()
    rows = Y.double()[pos.clamp(min=0)] * (pos >= 0).unsqueeze(-1)
    rows = torch.where((pos >= 0).unsqueeze(-1), rows, torch.zeros_like(rows))
    w = torch.ones(tokens, k, dtype=torch.float64, device=Y.device) if weights is None else weights.view(tokens, k).double()
    return (w.unsqueeze(-1) * rows).sum(1), (w.abs().unsqueeze(-1) * rows.abs()).sum(1)


def quantize(X):
    x = X.double()
    top = x.abs().amax(-1) if x.shape[-1] else torch.zeros(x.shape[:-1], dtype=torch.float64, device=x.device)
    scale = top / 127
    q = torch.where(scale.unsqueeze(-1) == 0, torch.zeros_like(x), (127 * x / top.unsqueeze(-1))).round()
    return q, scale


def scores_of_gradient(x, score):
    """The scores as a differentiable function of float64 logits."""
    return torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, -1)
