"""Oracle of the causal token mixers beside FLARE: straight from the definitions, token by token, in the inputs' own type
(fp64 in the tests) and differentiable by torch's automatic differentiation.  Test infrastructure only."""

import torch


def runs(documents):
    """[B, N] number of the run of equal ids that a token belongs to, and whether it is none of the padding."""
    border = torch.zeros_like(documents, dtype=torch.long)
    border[:, 1:] = documents[:, 1:] != documents[:, :-1]
    return border.cumsum(1), documents >= 0


def _who(x, documents, lengths):
    B, N = x.shape[:2]
    if documents is not None:
        return runs(documents)
    run = torch.zeros(B, N, dtype=torch.long, device=x.device)
    if lengths is None:
        return run, torch.ones_like(run, dtype=torch.bool)
    return run, torch.arange(N, device=x.device)[None] < lengths[:, None]


def causal_conv(x, weight, bias=None, state=None, silu=False, documents=None, lengths=None):
    """y [B, N, C] and the last W - 1 inputs."""
    B, N, C = x.shape
    W = weight.shape[1]
    run, on = _who(x, documents, lengths)
    state = x.new_zeros(B, W - 1, C) if state is None else state
    ys = []
    for t in range(N):
        v = x[:, t] * weight[:, W - 1]
        for j in range(1, W):
            if t - j >= 0:
                tap = torch.where((run[:, t - j] == run[:, t])[:, None], x[:, t - j], torch.zeros_like(v))
            else:
                tap = state[:, W - 1 + t - j]
            v = v + tap * weight[:, W - 1 - j]
        if bias is not None:
            v = v + bias
        if silu:
            v = v * torch.sigmoid(v)
        ys.append(torch.where(on[:, t, None], v, torch.zeros_like(v)))
    ends = [N] * B if lengths is None else [min(N, max(0, int(n))) for n in lengths]
    full = torch.cat([state, x], 1)
    return torch.stack(ys, 1), torch.stack([full[b, e:e + W - 1] for b, e in enumerate(ends)])


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, softplus=False, documents=None, lengths=None):
    """y [B, N, C] and the last state [B, C, S].  B, C [B, N, G, S]."""
    nb, N, ch = x.shape
    G = B.shape[2]
    run, on = _who(x, documents, lengths)
    h = x.new_zeros(nb, ch, A.shape[1]) if state is None else state
    ys = []
    for t in range(N):
        delta = dt[:, t] if dt_bias is None else dt[:, t] + dt_bias
        if softplus:
            delta = torch.nn.functional.softplus(delta, threshold=60.0)
        b, c = (p[:, t].repeat_interleave(ch // G, 1) for p in (B, C))
        if t > 0:
            h = torch.where((run[:, t] == run[:, t - 1])[:, None, None], h, torch.zeros_like(h))
        new = torch.exp(delta[..., None] * A) * h + (delta * x[:, t])[..., None] * b
        h = torch.where(on[:, t, None, None], new, h)
        y = (h * c).sum(-1)
        if D is not None:
            y = y + D * x[:, t]
        if z is not None:
            y = y * z[:, t] * torch.sigmoid(z[:, t])
        ys.append(torch.where(on[:, t, None], y, torch.zeros_like(y)))
    return torch.stack(ys, 1), h
