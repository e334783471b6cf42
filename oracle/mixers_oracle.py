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


def in_sight(N, documents=None, prefix=None, window=None):
    """[B, N, N] truth values: does token i see token j?  B is 1 without documents and prefix."""
    B = 1 if documents is None and prefix is None else (documents if documents is not None else prefix).shape[0]
    device = next((t.device for t in (documents, prefix) if t is not None), "cpu")
    see = torch.zeros(B, N, N, dtype=torch.bool)
    run = torch.zeros(B, N, dtype=torch.long) if documents is None else runs(documents)[0].cpu()
    on = torch.ones(B, N, dtype=torch.bool) if documents is None else (documents >= 0).cpu()
    led = torch.zeros(B, N, dtype=torch.bool)
    for b in range(B):
        for j in range(N if prefix is not None else 0):
            led[b, j] = prefix[b, j] and (j == 0 or run[b, j] != run[b, j - 1] or led[b, j - 1])
    i, j = torch.arange(N)[:, None], torch.arange(N)[None]
    for b in range(B):
        see[b] = ((j <= i) | led[b][None]) & (run[b][:, None] == run[b][None]) & on[b][:, None] & on[b][None]
        if window is not None:
            see[b] &= j > i - window
    return see.to(device)


class Attention:
    """Softmax attention of q [B, N, H, D] over k, v [B, M, J, D] where ``see`` [B or 1, N, M] holds; positions of the queries: first
    [B] + 0..N-1.  With ``dy`` the gradients, in closed form.  ``eps``: half a step of the type that weights and outputs are rounded to; the
    ``*_off`` are then bounds on how far a kernel that rounds P, dS and its outputs once, and computes in fp32 otherwise, may be off.  fp16 has steps of
    2^-24 at its lower end, where half of one is what a value is off by: 2^-32 for weights that are laid down times 2^7, 2^-37 |dy| |v| (of the longest
    rows) for dS that is laid down times the power of two that takes its bound, 2 |dy| |v|, to 2^13 at least."""

    def __init__(self, q, k, v, see, scale, cap=None, slopes=None, first=None, dy=None, eps=0.0):
        B, N, H, D = q.shape
        M, J = k.shape[1], k.shape[2]
        qh = q.transpose(1, 2)
        kh, vh = (t.transpose(1, 2).repeat_interleave(H // J, 1) for t in (k, v))
        s = scale * qh @ kh.transpose(2, 3)
        t = torch.zeros_like(s)
        if cap is not None:
            t = torch.tanh(s / cap)
            s = cap * t
        if slopes is not None:
            at = torch.arange(N, device=q.device)[None] + (0 if first is None else first[:, None])
            s = s - slopes[None, :, None, None] * (at[..., None] - torch.arange(M, device=q.device)).abs()[:, None]
        see = see[:, None].expand(B, H, N, M)
        some = see.any(-1, keepdim=True)
        p = torch.softmax(torch.where(some, s.masked_fill(~see, -torch.inf), torch.zeros_like(s)), -1) * some
        y = p @ vh
        # fp32: scores and exponents, a few units of 2^-22 of the largest score in sight
        f = 2.0 ** -21 * (1 + (s.abs() * see).amax((-1, -2), keepdim=True))
        fp16 = eps == 2.0 ** -11
        rounded = lambda x, floor=0.0: (eps * x.abs()).clamp(min=floor if fp16 else 0.0) * see  # noqa: E731
        y_off = (rounded(p, 2.0 ** -32) + f * p) @ vh.abs() + eps * y.abs()
        back = lambda x: x.transpose(1, 2)  # noqa: E731
        fold = lambda x: back(x).reshape(B, M, J, H // J, D).sum(3)  # noqa: E731
        self.y, self.y_off = back(y), back(y_off)
        if dy is None:
            return
        g = dy.transpose(1, 2)
        dp = g @ vh.transpose(2, 3)
        slope = 1 - t * t
        raw = p * (dp - (g * y).sum(-1, keepdim=True)) * some
        ds = raw * slope
        floor = 2.0 ** -37 * float(dy.norm(dim=-1).amax() * v.norm(dim=-1).amax())
        ds_off = rounded(ds, floor) + (ds.abs() + raw.abs()) * f + p * ((g.abs() * y_off).sum(-1, keepdim=True) + f * (g.abs() @ vh.abs().transpose(2, 3)))
        self.dq, self.dk, self.dv = back(scale * ds @ kh), fold(scale * ds.transpose(2, 3) @ qh), fold(p.transpose(2, 3) @ g)
        self.dq_off = back(scale * ds_off @ kh.abs()) + eps * self.dq.abs()
        self.dk_off = fold(scale * ds_off.transpose(2, 3) @ qh.abs()) + eps * self.dk.abs()
        self.dv_off = fold((rounded(p, 2.0 ** -32) + f * p).transpose(2, 3) @ g.abs()) + eps * self.dv.abs()
