"""Workloads of the causal token mixers beside FLARE: the short causal convolution, the selective scan and attention.

A case is a dict of plain values.  ``op`` names the operator, ``mode`` the direction:

* ``train``   forward and backward over whole sequences; ``documents``: several documents packed into each row, with
              padding behind the last one
* ``prompt``  prompts of different lengths, right-padded, on top of a carried state (for attention: of a filled cache)
* ``step``    one token for every sequence of a batch, states updated in place

B rows of N tokens; C channels, W taps, S states per channel, G groups of B / C projections; H query heads and J key /
value heads of width D, caches of L slots.  ``own`` selects the framework's kernels instead of the plain form below.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _package():
    path = os.path.abspath("causal-flare_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import causal_flare

    return causal_flare


def listed():
    return [
        # one user's next token: the smallest call there is, once per token and layer
        dict(name="conv_step", op="conv", mode="step", dtype="bf16", B=1, C=2048, W=4, silu=True),
        # a batch of prompts in half precision behind earlier text, odd length, three taps
        dict(name="conv_prompt", op="conv", mode="prompt", dtype="fp16", B=3, N=777, C=1544, W=3, silu=True),
        # the convolution of a training step
        dict(name="conv_train", op="conv", mode="train", dtype="bf16", B=4, N=4096, C=4096, W=4, silu=True),
        # a server's decode batch: all states are read and written
        dict(name="scan_step", op="scan", mode="step", dtype="bf16", B=256, C=8192, S=16, G=1, gate=True),
        # one long prompt: few channels, many tokens
        dict(name="scan_prompt", op="scan", mode="prompt", dtype="bf16", B=1, N=8191, C=2048, S=16, G=1, gate=True),
        # the scan of a training step
        dict(name="scan_train", op="scan", mode="train", dtype="bf16", B=4, N=4096, C=2048, S=16, G=1, gate=True),
        # single precision, packed documents, two groups, odd sizes: a small run that results are checked with
        dict(name="scan_fp32", op="scan", mode="train", dtype="fp32", B=2, N=777, C=200, S=8, G=2, gate=False, documents=True),
        # one user's next token on a short text, distance bias
        dict(name="attention_step_one", op="attention", mode="step", dtype="bf16", B=1, H=8, J=8, D=64, L=512, bias=True),
        # a server's decode batch with shared key heads, caches filled to different lengths, capped scores
        dict(name="attention_step", op="attention", mode="step", dtype="bf16", B=32, H=32, J=8, D=128, L=4096, cap=30.0),
        # parts of long prompts behind caches filled to different lengths, capped scores, a sliding window
        dict(name="attention_prompt", op="attention", mode="prompt", dtype="bf16", B=2, N=4000, H=16, J=4, D=128, L=8192, cap=30.0, window=2048),
        # packed documents with bidirectional prefixes and a distance bias, half precision, odd length, shared key heads
        dict(name="attention_documents", op="attention", mode="train", dtype="fp16", B=3, N=2049, H=12, J=4, D=64, bias=True, documents=True, prefix=True),
        # the attention of a training step
        dict(name="attention_train", op="attention", mode="train", dtype="bf16", B=2, N=4096, H=16, J=16, D=128, cap=30.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "attention", "attention", "attention"])
    mode = rng.choice(["train", "train", "prompt", "step"])
    c = dict(op=op, mode=mode, dtype=rng.choice(["bf16", "bf16", "fp16"] if op == "attention" else ["bf16", "bf16", "fp16", "fp32"]))
    if mode == "step":
        c["B"] = _log_int(rng, 1, 32 if op == "attention" else 256)
    else:
        c["B"] = _log_int(rng, 1, 4)
        c["N"] = _log_int(rng, 1, 4096)
        if mode == "train" and rng.random() < 0.4:
            c["documents"] = True
    if op == "conv":
        c.update(C=8 * _log_int(rng, 4, 512), W=rng.choice([2, 3, 4]), silu=rng.random() < 0.7)
    elif op == "scan":
        c.update(C=8 * _log_int(rng, 4, 256), S=rng.choice([8, 16, 16, 32]), G=1, gate=rng.random() < 0.6)
        if c["C"] % 16 == 0 and rng.random() < 0.3:
            c["G"] = 2
        if mode != "step":
            while c["B"] * c["N"] * c["C"] * c["S"] > 4 * 4096 * 2048 * 16:
                c["N"] = (c["N"] + 1) // 2
    else:
        c["J"] = rng.choice([1, 2, 4, 8])
        c.update(H=c["J"] * rng.choice([1, 2, 4]), D=rng.choice([64, 64, 72, 96, 128, 128]))
        if rng.random() < 0.4:
            c["cap"] = rng.choice([15.0, 30.0, 50.0])
        if rng.random() < 0.4:
            c["bias"] = True
        if rng.random() < 0.3:
            c["window"] = _log_int(rng, 16, 2048)
        if mode == "train" and rng.random() < 0.3:
            c["prefix"] = True
        if mode != "train":
            c["L"] = _log_int(rng, 64, 4096) + c.get("N", 1)
        while work(c)["flops"] > work(listed()[-1])["flops"]:
            c["L"], c["N"] = c.get("L", 0) - c["N"] // 2, c["N"] - c["N"] // 2
        if mode == "train":
            c.pop("L", None)
    return c


class _State:
    pass


def _documents(B, N, g):
    """Ids of documents packed into rows: about one border in every 300 tokens, and up to an eighth of padding at the end."""
    border = torch.rand(B, N, generator=g, device="cuda") < 1 / 300
    ids = border.int().cumsum(1).int()
    used = N - torch.randint(0, N // 8 + 1, (B, 1), generator=g, device="cuda")
    return torch.where(torch.arange(N, device="cuda")[None] < used, ids, -1).to(torch.int32)


def prepare(case, seed):
    """What a program holds before the call: activations of N(0, 1), weights of a freshly initialised layer, the states
    or caches of the text so far, upstream gradients."""
    s = _State()
    s.case = case
    B, N, mode, dt = case["B"], case.get("N", 1), case["mode"], _DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    def integers(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    s.documents = _documents(B, N, g) if case.get("documents") else None
    s.lengths = None
    if mode == "prompt":
        s.lengths = integers(N - N // 4, N + 1, B)
        s.lengths[0] = N
    tokens = (B, N) if mode != "step" else (B,)
    if case["op"] == "conv":
        C, W = case["C"], case["W"]
        s.x = normal(*tokens, C)
        s.weight = normal(C, W, dtype=torch.float32) * W ** -0.5
        s.bias = 0.1 * normal(C, dtype=torch.float32)
        s.state = normal(B, W - 1, C) if mode != "train" else None
        s.leaves = (s.x, s.weight, s.bias)
        s.dy = normal(*tokens, C) if mode == "train" else None
    elif case["op"] == "scan":
        C, S, G = case["C"], case["S"], case["G"]
        s.x, s.dt = normal(*tokens, C), normal(*tokens, C)
        s.A = -torch.arange(1, S + 1, device="cuda", dtype=torch.float32) * torch.exp(0.1 * normal(C, S, dtype=torch.float32))
        s.B, s.C = normal(*tokens, G, S), normal(*tokens, G, S)
        s.D = 1 + 0.1 * normal(C, dtype=torch.float32)
        s.z = normal(*tokens, C) if case["gate"] else None
        # biases under which softplus(bias) lies between a thousandth and a tenth
        rate = torch.exp(torch.rand(C, generator=g, device="cuda") * math.log(100) + math.log(1e-3))
        s.bias = rate + torch.log(-torch.expm1(-rate))
        s.state = normal(B, C, S, dtype=torch.float32) if mode != "train" else None
        s.leaves = (s.x, s.dt, s.A, s.B, s.C, s.D, s.bias) + ((s.z,) if case["gate"] else ())
        s.dy = normal(*tokens, C) if mode == "train" else None
    else:
        H, J, D = case["H"], case["J"], case["D"]
        s.q, s.k, s.v = normal(*tokens, H, D), normal(*tokens, J, D), normal(*tokens, J, D)
        s.slopes = 2 ** (-8 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H) if case.get("bias") else None
        s.prefix = None
        if case.get("prefix"):  # the first quarter of the row is a question, and so is what follows a document's border
            s.prefix = (torch.arange(N, device="cuda")[None] < N // 4).repeat(B, 1)
            if s.documents is not None:
                run = torch.cat([torch.ones_like(s.documents[:, :1], dtype=torch.bool), s.documents[:, 1:] != s.documents[:, :-1]], 1)
                at = torch.arange(N, device="cuda")[None]
                s.prefix = at - torch.where(run, at, 0).cummax(1).values < 100
        if mode != "train":
            L = case["L"]
            s.k_cache, s.v_cache = normal(B, L, J, D), normal(B, L, J, D)
            s.cached = integers((L - N) // 2, L - N + 1, B)
            s.cached[0] = L - N
        s.leaves = (s.q, s.k, s.v)
        s.dy = normal(*tokens, H, D) if mode == "train" else None
    if mode == "train":
        for t in s.leaves:
            t.requires_grad_()
    return s


def _call(s):
    """The calls that a user makes of the framework."""
    cf, case = _package(), s.case
    op, mode = case["op"], case["mode"]
    if op == "conv":
        act = "silu" if case["silu"] else None
        if mode == "step":
            return cf.flare_causal_conv_decode(s.x, s.weight, s.bias, s.state, activation=act)
        if mode == "prompt":
            return cf.flare_causal_conv_prefill(s.x, s.weight, s.bias, s.state, activation=act, lengths=s.lengths)
        y = cf.flare_causal_conv(s.x, s.weight, s.bias, activation=act, documents=s.documents)
    elif op == "scan":
        args = (s.x, s.dt, s.A, s.B, s.C)
        more = dict(D=s.D, z=s.z, dt_bias=s.bias, dt_softplus=True)
        if mode == "step":
            return cf.flare_selective_scan_decode(*args, s.state, **more)
        if mode == "prompt":
            return cf.flare_selective_scan_prefill(*args, s.state, lengths=s.lengths, **more)
        y = cf.flare_selective_scan(*args, documents=s.documents, **more)
    else:
        more = dict(cap=case.get("cap"), slopes=s.slopes, window=case.get("window"))
        if mode == "step":
            y = cf.flare_causal_attention_decode(s.q, s.k, s.v, s.k_cache, s.v_cache, s.cached, **more)
            return y, s.k_cache, s.v_cache
        if mode == "prompt":
            y = cf.flare_causal_attention_prefill(s.q, s.k, s.v, s.k_cache, s.v_cache, cached=s.cached, lengths=s.lengths, **more)
            return y, s.k_cache, s.v_cache
        y = cf.flare_causal_attention(s.q, s.k, s.v, documents=s.documents, prefix=s.prefix, **more)
    return y, torch.autograd.grad(y, s.leaves, s.dy)


def run(s):
    if own:
        return _call(s)
    with torch.no_grad():
        return {"conv": _plain_conv, "scan": _plain_scan, "attention": _plain_attention}[s.case["op"]](s)


# ---- plain forms ---------------------------------------------------------------------------------------------------


def _valid(s, B, N):
    """[B, N] truth values: the tokens that are none of the padding."""
    if s.documents is not None:
        return s.documents >= 0
    if s.lengths is not None:
        return torch.arange(N, device="cuda")[None] < s.lengths[:, None]
    return torch.ones(B, N, dtype=torch.bool, device="cuda")


def _silu_and_slope(x):
    r = 1 / (1 + torch.exp(-x))
    return x * r, r * (1 + x * (1 - r))


def _taps(x, before, W):
    """[B, N, C] and the W - 1 rows in front of it as [B, N, C, W], a token's own value last."""
    return torch.cat([before, x], 1).unfold(1, W, 1)


def _plain_conv(s):
    case, dt = s.case, s.x.dtype
    W, B, C = case["W"], case["B"], case["C"]
    x = s.x.float() if s.x.dim() == 3 else s.x.float()[:, None]
    N = x.shape[1]
    before = s.state.float() if s.state is not None else x.new_zeros(B, W - 1, C)
    taps = _taps(x, before, W)
    valid = _valid(s, B, N)
    same = None
    if s.documents is not None:
        ids = _taps(s.documents[..., None], s.documents.new_full((B, W - 1, 1), -1), W)
        # a tap counts where no border lies between it and the token: a run of equal ids is one document
        same = (ids[..., 1:] == ids[..., :-1]).int().flip(-1).cumprod(-1).flip(-1).bool()
        same = torch.cat([same, torch.ones_like(same[..., :1])], -1)
        taps = torch.where(same, taps, 0)
    pre = (taps * s.weight).sum(-1) + s.bias
    y, slope = _silu_and_slope(pre) if case["silu"] else (pre, torch.ones_like(pre))
    y = torch.where(valid[..., None], y, 0).to(dt)
    if case["mode"] == "step":
        s.state.copy_(torch.cat([s.state, s.x[:, None]], 1)[:, 1:])
        return y[:, 0], s.state
    if case["mode"] == "prompt":
        at = s.lengths[:, None].long() + torch.arange(W - 1, device="cuda")
        return y, torch.cat([s.state, s.x], 1).gather(1, at[..., None].expand(B, W - 1, C))
    g = torch.where(valid[..., None], s.dy.float() * slope, 0)
    dw = (g[..., None] * taps).sum((0, 1))
    spread = g[..., None] * s.weight
    if same is not None:
        spread = torch.where(same, spread, 0)
    dx = torch.stack([torch.nn.functional.pad(spread[:, W - 1 - j :, :, j], (0, 0, 0, min(N, W - 1 - j))) for j in range(W)]).sum(0)
    return y, (dx.to(dt), dw, g.sum((0, 1)))


def _linear_recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, by doubling."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], torch.addcmul(b[:, step:], a[:, step:], b[:, :-step])], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _plain_scan(s):
    case, dt = s.case, s.x.dtype
    B, C, S, G = case["B"], case["C"], case["S"], case["G"]
    step = case["mode"] == "step"

    def wide(t):
        t = t.float()
        return t[:, None] if step else t

    x, raw = wide(s.x), wide(s.dt) + s.bias
    N = x.shape[1]
    Bn, Cn = (wide(t).repeat_interleave(C // G, 2) for t in (s.B, s.C))
    valid = _valid(s, B, N)[..., None]
    # softplus without loss for large and for very small values
    delta = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20))))
    x, delta = torch.where(valid, x, 0), torch.where(valid, delta, 0)
    a = torch.exp(delta[..., None] * s.A)
    if s.documents is not None:
        first = torch.cat([torch.ones_like(s.documents[:, :1], dtype=torch.bool), s.documents[:, 1:] != s.documents[:, :-1]], 1)
        a = torch.where(first[..., None, None], 0, a)
    b = (delta * x)[..., None] * Bn
    if s.state is not None:
        b[:, 0] += a[:, 0] * s.state
    h = _linear_recurrence(a, b)
    plain = (h * Cn).sum(-1) + s.D * x
    gate, slope = _silu_and_slope(wide(s.z)) if s.z is not None else (torch.ones_like(plain), None)
    y = torch.where(valid, plain * gate, 0).to(dt)
    if step:
        s.state.copy_(h[:, 0])
        return y[:, 0], s.state
    if case["mode"] == "prompt":
        return y, h[:, -1].clone()
    dy = torch.where(valid, s.dy.float(), 0)
    gy = dy * gate
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _linear_recurrence(later.flip(1), (gy[..., None] * Cn).flip(1)).flip(1)
    del later
    gB = (g * Bn).sum(-1)
    back = g * a
    back[:, 1:] *= h[:, :-1]
    back[:, 0] = 0
    ddelta = torch.where(valid, (gB * x + (back * s.A).sum(-1)) * torch.sigmoid(raw), 0)
    out = [torch.where(valid, gB * delta + s.D * gy, 0).to(dt), ddelta.to(dt), (back * delta[..., None]).sum((0, 1))]
    del back
    out.append((g * (delta * x)[..., None]).view(B, N, G, C // G, S).sum(3).to(dt))
    out.append((h * gy[..., None]).view(B, N, G, C // G, S).sum(3).to(dt))
    out += [(gy * x).sum((0, 1)), ddelta.sum((0, 1))]
    if s.z is not None:
        out.append((dy * plain * slope).to(dt))
    return y, tuple(out)


def _plain_attention(s):
    case, dt = s.case, s.q.dtype
    B, H, J, D = case["B"], case["H"], case["J"], case["D"]
    mode, window, cap = case["mode"], case.get("window"), case.get("cap")
    q, k, v = (t[:, None] if mode == "step" else t for t in (s.q, s.k, s.v))
    N = q.shape[1]
    at = torch.arange(N, device="cuda")
    valid = _valid(s, B, N)
    place = at[None].expand(B, N) if mode == "train" else s.cached[:, None] + at
    lo, hi = torch.zeros_like(place), place + 1
    if s.documents is not None:
        first = torch.cat([torch.ones_like(valid[:, :1]), s.documents[:, 1:] != s.documents[:, :-1]], 1)
        lo = torch.where(first, at, 0).cummax(1).values
    if s.prefix is not None:
        # the first token of the row that is no longer part of its document's prefix
        led = torch.where(s.prefix & valid, N, at)
        stop = torch.full_like(lo, N).scatter_reduce_(1, lo, led, "amin")
        ends = torch.full_like(lo, 0).scatter_reduce_(1, lo, at + 1 + torch.zeros_like(lo), "amax")
        hi = torch.maximum(hi, torch.minimum(stop, ends).gather(1, lo))
    if window is not None:
        lo = torch.maximum(lo, place - window + 1)
    if mode != "train":
        row = torch.arange(B, device="cuda")[:, None].expand(B, N)[valid]
        s.k_cache[row, place[valid].long()] = k[valid]
        s.v_cache[row, place[valid].long()] = v[valid]
        k, v = s.k_cache, s.v_cache
    M = k.shape[1]
    q, k, v = (t.float().transpose(1, 2) for t in (q, k, v))
    q = q.reshape(B, J, H // J * N, D)
    scale = D ** -0.5
    key = torch.arange(M, device="cuda")
    seen = (key >= lo[..., None]) & (key < hi[..., None]) & valid[..., None]
    p = (q @ k.transpose(2, 3)).view(B, H, N, M) * scale
    t = None
    if cap is not None:
        t = torch.tanh(p / cap)
        p = cap * t
    if s.slopes is not None:
        p = p - s.slopes[:, None, None] * (place[..., None] - key).abs()[:, None]
    p = p.masked_fill(~seen[:, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1, total)
    y = (p.view(B, J, H // J * N, M) @ v).view(B, H, N, D)
    out = y.transpose(1, 2).to(dt)
    if mode == "step":
        return out[:, 0], s.k_cache, s.v_cache
    if mode == "prompt":
        return out, s.k_cache, s.v_cache
    dy = s.dy.float().transpose(1, 2)
    dp = (dy.reshape(B, J, H // J * N, D) @ v.transpose(2, 3)).view(B, H, N, M)
    dp = p * (dp - (dy * y).sum(-1, keepdim=True))
    if t is not None:
        dp = dp * (1 - t * t)
    dp = (dp * scale).view(B, J, H // J * N, M)
    dv = p.view(B, J, H // J * N, M).transpose(2, 3) @ dy.reshape(B, J, H // J * N, D)
    grads = ((dp @ k).view(B, H, N, D), dp.transpose(2, 3) @ q, dv)
    return out, tuple(x.transpose(1, 2).to(dt) for x in grads)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "attention": _exact_attention}[case["op"]](s)


def _leaf(t):
    return t.detach().double().requires_grad_()


def _exact_conv(s):
    """Term by term, gradients by automatic differentiation."""
    case = s.case
    W = case["W"]
    x = s.x if case["mode"] != "step" else s.x[:, None]
    B, N = x.shape[:2]
    x, w, b = _leaf(x), _leaf(s.weight), _leaf(s.bias)
    state = s.state.double() if s.state is not None else x.new_zeros(B, W - 1, case["C"])
    full = torch.cat([state, x], 1)
    pre = b + full[:, W - 1 :] * w[:, W - 1]
    linked = torch.ones(B, N, dtype=torch.bool, device="cuda")
    for j in range(1, W):
        if s.documents is not None:
            d = s.documents
            now = torch.zeros_like(linked)
            if j < N:
                now[:, j:] = d[:, j:] == d[:, :-j]
                for i in range(1, j):
                    now[:, j:] &= d[:, j:] == d[:, j - i : N - i]
            linked = now
        pre = pre + torch.where(linked[..., None], full[:, W - 1 - j : W - 1 - j + N] * w[:, W - 1 - j], 0)
    y = pre * torch.sigmoid(pre) if case["silu"] else pre
    if s.documents is not None:
        y = torch.where((s.documents >= 0)[..., None], y, 0)
    if s.lengths is not None:
        y = torch.where((torch.arange(N, device="cuda") < s.lengths[:, None])[..., None], y, 0)
    if case["mode"] == "train":
        return y.detach(), torch.autograd.grad(y, (x, w, b), s.dy.double())
    full = full.detach()
    ends = [N] * B if s.lengths is None else s.lengths.tolist()
    left = torch.stack([full[i, e : e + W - 1] for i, e in enumerate(ends)])
    return (y[:, 0] if case["mode"] == "step" else y).detach(), left


def _exact_scan(s):
    """Token by token, forward and in reverse."""
    case = s.case
    C, S, G = case["C"], case["S"], case["G"]
    many = case["mode"] != "step"

    def wide(t):
        return t.detach().double() if many else t.detach().double()[:, None]

    x, z = wide(s.x), wide(s.z) if s.z is not None else None
    B, N = x.shape[:2]
    A, D = s.A.detach().double(), s.D.detach().double()
    u = wide(s.dt) + s.bias.detach().double()
    delta = torch.nn.functional.softplus(u, threshold=50)
    Bp, Cp = wide(s.B), wide(s.C)

    def per_channel(t, n):
        return t[:, n].repeat_interleave(C // G, 1)

    on = torch.ones(B, N, 1, device="cuda", dtype=torch.float64)
    new = torch.zeros(B, N, 1, 1, device="cuda", dtype=torch.bool)
    if s.documents is not None:
        on = (s.documents >= 0).double()[..., None]
        new[:, 0] = True
        new[:, 1:, 0, 0] = s.documents[:, 1:] != s.documents[:, :-1]
    if s.lengths is not None:
        on = (torch.arange(N, device="cuda")[None] < s.lengths[:, None]).double()[..., None]
    h = s.state.double() if s.state is not None else x.new_zeros(B, C, S)
    train = case["mode"] == "train"
    before, plain = [], []
    for n in range(N):
        h = h.masked_fill(new[:, n], 0.0)
        if train:
            before.append(h)
        move = on[:, n, :, None]
        d = delta[:, n, :, None]
        h = torch.exp(d * A * move) * h + move * d * per_channel(Bp, n) * x[:, n, :, None]
        plain.append((h * per_channel(Cp, n)).sum(-1))
    plain = torch.stack(plain, 1) + D * x
    r = torch.sigmoid(z) if z is not None else None
    y = on * (plain * z * r if z is not None else plain)
    if not train:
        return (y if many else y[:, 0]), h
    dy = s.dy.double() * on
    gy = dy * z * r if z is not None else dy
    g, dA = torch.zeros_like(h), torch.zeros_like(A)
    dx, du, dB, dC = [], [], [], []
    for n in reversed(range(N)):
        b, c, d, past = per_channel(Bp, n), per_channel(Cp, n), delta[:, n, :, None], before[n]
        move = on[:, n, :, None]
        a = torch.exp(d * A * move)
        now = a * past + move * d * b * x[:, n, :, None]
        g = g + gy[:, n, :, None] * c
        dC.append((gy[:, n, :, None] * now).view(B, G, C // G, S).sum(2))
        dB.append((move * g * d * x[:, n, :, None]).view(B, G, C // G, S).sum(2))
        slope = g * a * past * move
        dA += (slope * d).sum(0)
        inner = (g * b).sum(-1) * on[:, n]
        dx.append(inner * delta[:, n] + D * gy[:, n])
        du.append((inner * x[:, n] + (slope * A).sum(-1)) * torch.sigmoid(u[:, n]))
        g = (g * a).masked_fill(new[:, n], 0.0)
    dx, du, dB, dC = (torch.stack(t[::-1], 1) for t in (dx, du, dB, dC))
    grads = [dx, du, dA, dB, dC, (gy * x).sum((0, 1)), du.sum((0, 1))]
    if z is not None:
        grads.append(dy * plain * r * (1 + z * (1 - r)))
    return y, tuple(grads)


def _exact_attention(s):
    """Row by row and head by head, masks from their definitions, gradients by automatic differentiation."""
    case = s.case
    B, H, J, D = case["B"], case["H"], case["J"], case["D"]
    mode, cap, window = case["mode"], case.get("cap"), case.get("window")
    q, k, v = (t[:, None] if mode == "step" else t for t in (s.q, s.k, s.v))
    N = q.shape[1]
    keys, values = (k, v) if mode == "train" else (s.k_cache.clone(), s.v_cache.clone())
    counts = [N] * B if s.lengths is None else s.lengths.tolist()
    starts = [0] * B if mode == "train" else s.cached.tolist()
    if mode != "train":
        for i in range(B):
            keys[i, starts[i] : starts[i] + counts[i]] = k[i, : counts[i]]
            values[i, starts[i] : starts[i] + counts[i]] = v[i, : counts[i]]
    M = keys.shape[1]
    y = torch.zeros(B, N, H, D, device="cuda", dtype=torch.float64)
    grads = [torch.zeros(t.shape, device="cuda", dtype=torch.float64) for t in (q, k, v)] if mode == "train" else None
    for i in range(B):
        n = counts[i]
        m = M if mode == "train" else starts[i] + n
        rows = torch.arange(n, device="cuda")[:, None] + starts[i]
        cols = torch.arange(m, device="cuda")[None]
        see = cols <= rows
        if mode == "train":
            run = torch.zeros(N, dtype=torch.long, device="cuda")
            live = torch.ones(N, dtype=torch.bool, device="cuda")
            if s.documents is not None:
                run[1:] = (s.documents[i, 1:] != s.documents[i, :-1]).cumsum(0)
                live = s.documents[i] >= 0
            if s.prefix is not None:
                other = (~s.prefix[i]).long()
                total = other.cumsum(0)
                begun = torch.searchsorted(run, run)  # where the token's run begins
                see = see | (total - total[begun] + other[begun] == 0)[None]
            see = see & (run[:, None] == run[None]) & live[:, None] & live[None]
        if window is not None:
            see = see & (cols > rows - window)
        some = see.any(1)
        far = (rows - cols).abs().double()
        for head in range(H):
            a, b, c = _leaf(q[i, :n, head]), _leaf(keys[i, :m, head * J // H]), _leaf(values[i, :m, head * J // H])
            score = a @ b.T / math.sqrt(D)
            if cap is not None:
                score = cap * torch.tanh(score / cap)
            if s.slopes is not None:
                score = score - s.slopes[head].double() * far
            # rows without keys: any finite scores, and nothing of what they give
            score = torch.where(see, score, -math.inf)
            score = torch.where(some[:, None], score, 0)
            o = torch.where(some[:, None], torch.softmax(score, 1) @ c, 0)
            y[i, :n, head] = o.detach()
            if mode == "train":
                for to, got, at in zip(grads, torch.autograd.grad(o, (a, b, c), s.dy[i, :, head].double()), (head, head * J // H, head * J // H)):
                    to[i, :, at] += got
    if mode == "train":
        return y, tuple(grads)
    return (y[:, 0] if mode == "step" else y), keys.double(), values.double()


def work(case):
    """Every input read once, every output written once.  Convolution: two operations per tap forward, four in the
    backward.  Scan: per token, channel and state an exponential (as one operation) and six, three times that in the
    backward.  Attention: 4 D operations for each query head and key in sight (all tokens of a causal half, or of the
    window; documents of about 300 tokens), and two and a half times that in the backward."""
    B, N, e, mode = case["B"], case.get("N", 1), _BYTES[case["dtype"]], case["mode"]
    train = mode == "train"
    ids = 4 * B * N if case.get("documents") else 0
    if case["op"] == "conv":
        C, W = case["C"], case["W"]
        rows = B * N * C * e
        size = 2 * rows + 4 * C * (W + 1) + ids + (0 if train else 2 * B * (W - 1) * C * e)
        flops = 2 * W * B * N * C
        if train:
            size += 2 * rows + 4 * C * (W + 1)
            flops *= 3
        return {"bytes": size, "flops": flops}
    if case["op"] == "scan":
        C, S, G = case["C"], case["S"], case["G"]
        rows, wide = B * N * C * e, 2 * B * N * G * S * e
        gate = rows if case["gate"] else 0
        weights = 4 * C * (S + 2)
        size = 3 * rows + gate + wide + weights + ids + (0 if train else 8 * B * C * S)
        flops = 7 * B * N * C * S
        if train:
            size += 3 * rows + gate + wide + weights  # upstream gradient in; gradients of x, dt, z, B, C and weights out
            flops *= 4
        return {"bytes": size, "flops": flops}
    H, J, D = case["H"], case["J"], case["D"]
    qs, ks = B * N * H * D * e, 2 * B * N * J * D * e
    if mode == "train":
        span = min(N, 300) if case.get("documents") else N
        pairs = N * (span + 1) / 2
        past = 0
    else:
        past = 3 * (case["L"] - N) / 4
        pairs = N * (past + (N + 1) / 2)
    if case.get("window"):
        pairs = min(pairs, N * case["window"])
        past = min(past, case["window"])
    size = 2 * qs + ks + ids + (B * N if case.get("prefix") else 0)
    flops = 4 * D * H * B * pairs
    if train:
        size += 2 * qs + ks
        flops *= 3.5
    else:
        size += 2 * B * past * J * D * e + ks  # the cache so far, and the new rows into it
    return {"bytes": int(size), "flops": int(flops)}
