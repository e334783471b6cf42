"""gpu: causal attention against the oracle in 64 bits: head layouts, lengths around the tiles, caps, distance biases, windows, documents,
prefixes, padding, caches, single tokens.

Tolerances: the oracle's bounds (oracle/mixers_oracle.py): one rounding of half a step for every weight P, dS and output, fp32
otherwise, taken through the formulas with absolute values."""
import pytest
import torch

import causal_flare as cf
from causal_flare import _mixers, _ops, attention
from causal_flare._common import _resolve_attn_scale
from oracle import mixers_oracle as orc

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def close(got, want, off, what):
    got = got.detach().double()
    assert got.shape == want.shape, what
    tol = off * 1.01 + 2.0 ** -25  # (half the smallest step of fp16)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol).max()):.2f} of what is allowed"


def ids(kind, B, N, g):
    if kind is None:
        return None
    if kind == "every":
        return torch.arange(N, device="cuda", dtype=torch.int32)[None].repeat(B, 1)
    if kind == "padding":
        return torch.full((B, N), -1, device="cuda", dtype=torch.int32)
    d = (torch.rand(B, N, generator=g, device="cuda") < (0.3 if kind == "short" else 0.015)).int().cumsum(1)
    if kind == "again":
        d = d % 2
    if kind == "holes":
        d = torch.where(d % 4 == 0, -1, d)
    return d.int()


CASES = [  # B, N, H, J, D, cap, bias, window, documents, prefix
    (1, 1, 1, 1, 64, None, False, None, None, False), (2, 2, 2, 1, 8, None, False, None, None, False), (1, 63, 2, 2, 128, 5.0, False, None, None, False),
    (1, 64, 3, 1, 40, None, True, None, None, False), (2, 65, 2, 2, 64, None, False, None, None, False), (1, 127, 4, 2, 72, 2.0, True, None, None, False),
    (1, 128, 2, 2, 128, None, False, None, None, False), (2, 129, 2, 1, 96, None, False, 17, None, False), (1, 255, 1, 1, 64, 30.0, False, 128, None, True),
    (1, 256, 2, 2, 128, None, True, None, "again", False), (1, 257, 6, 2, 128, 10.0, False, None, "holes", True), (2, 300, 2, 2, 64, None, True, 100, "holes", True),
    (1, 513, 2, 1, 128, None, False, None, None, True), (3, 640, 4, 2, 64, None, False, None, "holes", False), (1, 700, 8, 8, 128, 50.0, True, 256, None, False),
    (2, 200, 2, 1, 64, None, False, None, "every", False), (2, 130, 2, 2, 128, None, True, None, "padding", True), (1, 1100, 2, 2, 128, None, False, None, "short", True),
    (2, 390, 5, 1, 120, 20.0, False, 1, "again", False),
]


def inputs(case, dtype, seed=0):
    B, N, H, J, D, cap, bias, window, kind, with_prefix = case
    g = gen(N * 31 + D + seed)
    q, k, v, dy = randn(g, B, N, H, D, dtype=dtype), randn(g, B, N, J, D, dtype=dtype), randn(g, B, N, J, D, dtype=dtype), randn(g, B, N, H, D, dtype=dtype)
    how = dict(cap=cap, slopes=torch.rand(H, generator=g, device="cuda") * 0.2 if bias else None, window=window, documents=ids(kind, B, N, g),
               prefix=torch.rand(B, N, generator=g, device="cuda") < 0.9 if with_prefix else None)
    return q, k, v, dy, how


def oracle(q, k, v, dy, how, dtype):
    see = orc.in_sight(q.shape[1], how["documents"], how["prefix"], how["window"]).to(q.device)
    s = how["slopes"]
    return orc.Attention(q.double(), k.double(), v.double(), see, _resolve_attn_scale(None, q.shape[-1]), how["cap"], None if s is None else s.double(), dy=dy.double(),
                         eps=torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention_and_its_gradients(case, dtype):
    q, k, v, dy, how = inputs(case, dtype)
    for t in (q, k, v):
        t.requires_grad_()
    y = cf.flare_causal_attention(q, k, v, **how)
    grads = torch.autograd.grad(y, (q, k, v), dy)
    assert y.dtype == dtype and all(t.dtype == dtype for t in grads)
    o = oracle(q.detach(), k.detach(), v.detach(), dy, how, dtype)
    close(y, o.y, o.y_off, "y")
    for name, got in zip(("dq", "dk", "dv"), grads):
        close(got, getattr(o, name), getattr(o, name + "_off"), name)
    with torch.no_grad():
        assert torch.equal(cf.flare_causal_attention(q, k, v, **how), y)
    assert _ops.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_sharp_scores(dtype):
    # scores of a few hundred: the running maximum grows by more than its slack again and again
    q, k, v, dy, how = inputs((1, 500, 2, 2, 64, None, False, None, None, False), dtype)
    q = q * 16
    k = k * torch.linspace(0.1, 3, 500, device="cuda")[None, :, None, None].to(dtype)
    for t in (q, k, v):
        t.requires_grad_()
    y = cf.flare_causal_attention(q, k, v)
    o = oracle(q.detach(), k.detach(), v.detach(), dy, how, dtype)
    close(y, o.y, o.y_off, "y")
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(y, (q, k, v), dy)):
        close(got, getattr(o, name), getattr(o, name + "_off"), name)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_padding_may_hold_anything(value):
    for case in ((2, 300, 4, 2, 64, None, False, None, "holes", False), (1, 390, 2, 2, 128, 10.0, True, 50, "holes", True)):
        q, k, v, dy, how = inputs(case, torch.bfloat16)
        pad = (how["documents"] < 0)[..., None, None]

        def run(fill):
            a, b, c, d = (t.masked_fill(pad, value) if fill else t.clone() for t in (q, k, v, dy))
            for t in (a, b, c):
                t.requires_grad_()
            y = cf.flare_causal_attention(a, b, c, **how)
            return (y, *torch.autograd.grad(y, (a, b, c), d))

        assert pad.any()
        for a, c in zip(run(True), run(False)):
            assert torch.equal(a, c)


def test_strided_inputs():
    q, k, v, dy, how = inputs((2, 200, 4, 2, 64, None, True, None, "again", False), torch.bfloat16)

    def run(q, k, v, dy):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        y = cf.flare_causal_attention(q, k, v, **how)
        return (y, *torch.autograd.grad(y, (q, k, v), dy))

    def heads_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def part_of_a_row(t):
        w = torch.zeros(*t.shape[:3], t.shape[3] + 8, device="cuda", dtype=t.dtype)
        w[..., :t.shape[3]] = t
        return w[..., :t.shape[3]]

    def unaligned(t):
        w = torch.zeros(t.numel() + 1, device="cuda", dtype=t.dtype)
        w[1:] = t.flatten()
        return w[1:].view(t.shape)

    def turned(t):
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)

    first = run(q, k, v, dy)
    for f in (heads_first, part_of_a_row, unaligned, turned):
        for a, c in zip(run(*(f(t) for t in (q, k, v, dy))), first):
            assert torch.equal(a, c), f.__name__
    one = dy[:1, :1].expand_as(dy)
    for a, c in zip(run(q, k, v, one), run(q, k, v, one.contiguous())):
        assert torch.equal(a, c)
    # one key row for all tokens
    for a, c in zip(run(q, k[:, :1].expand_as(k), v, dy), run(q, k[:, :1].expand_as(k).contiguous(), v, dy)):
        assert torch.equal(a, c)


def test_same_bits_on_another_stream_and_from_a_graph():
    q, k, v, dy, how = inputs((2, 333, 4, 2, 128, 20.0, True, None, "holes", True), torch.bfloat16)
    for t in (q, k, v):
        t.requires_grad_()

    def step():
        y = cf.flare_causal_attention(q, k, v, **how)
        return [y.detach(), *torch.autograd.grad(y, (q, k, v), dy)]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    for t in third:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(3, 2, 2, 1, 128, None, None), (2, 32, 4, 2, 64, 15.0, None), (1, 200, 3, 1, 40, None, 3), (1, 150, 6, 2, 96, 20.0, 32)], ids=str)
def test_few_keys_whose_values_are_much_alike(case, dtype):
    # dP - <dy, y> is a twentieth of either: the rounding of y, or of the weights in it, would show twenty times.  Rows of up to 32 keys go without either:
    # half a step of the result is left, dS within half^2 (two parts), and roundings of 2^-22 of sums twenty times as large.
    B, N, H, J, D, cap, window = case
    g = gen(N)
    q, k, dy = randn(g, B, N, H, D, dtype=dtype), randn(g, B, N, J, D, dtype=dtype), randn(g, B, N, H, D, dtype=dtype)
    v = (1 + 0.05 * randn(g, B, N, J, D)).to(dtype)
    slopes = torch.rand(H, generator=g, device="cuda") * 0.1
    for t in (q, k, v):
        t.requires_grad_()
    got = torch.autograd.grad(cf.flare_causal_attention(q, k, v, cap=cap, window=window, slopes=slopes), (q, k), dy)
    half = torch.finfo(dtype).eps / 2
    o = orc.Attention(q.detach().double(), k.detach().double(), v.detach().double(), orc.in_sight(N, window=window).cuda(), D ** -0.5, cap, slopes.double(),
                      dy=dy.double(), eps=half)
    for a, b in zip(got, (o.dq, o.dk)):
        assert float((a.double() - b).norm() / b.norm()) <= 1.01 * half + half ** 2 + 20 * 30 * 2.0 ** -22


def test_a_backward_without_the_forwards_plan_forms_it_again():
    case = (2, 300, 4, 2, 64, None, True, 100, "holes", True)
    q, k, v, dy, how = inputs(case, torch.bfloat16)
    for t in (q, k, v):
        t.requires_grad_()
    y = cf.flare_causal_attention(q, k, v, **how)
    want = torch.autograd.grad(y, (q, k, v), dy)
    a = attention._fill(q, k, v, (64 ** -0.5, 0.0, 100), how["slopes"], how["documents"], how["prefix"])
    out, lse = torch.empty_like(y), torch.empty(2, 4, 384, device="cuda")
    grads = [torch.empty_like(t) for t in (q, k, v)]
    a.y, a.lse = out.data_ptr(), lse.data_ptr()
    _mixers.run("flare_attention_forward", a, q.device, "flare_attention_forward_workspace_bytes")
    a.dy = dy.data_ptr()
    _mixers.put_strides(a, "dy", dy, "bnh")
    a.dq, a.dk, a.dv = (t.data_ptr() for t in grads)
    _mixers.run("flare_attention_backward", a, q.device, "flare_attention_backward_workspace_bytes")
    for x, z in zip((out, *grads), (y, *want)):
        assert torch.equal(x, z)


def test_no_tokens():
    q, k = torch.empty(2, 0, 4, 64, device="cuda", dtype=torch.float16, requires_grad=True), torch.empty(2, 0, 2, 64, device="cuda", dtype=torch.float16)
    y = cf.flare_causal_attention(q, k, k)
    assert y.shape == q.shape and torch.autograd.grad(y.sum(), q)[0].shape == q.shape


# ---- caches --------------------------------------------------------------------------------------------------------------


def behind_a_cache(B, N, L, cached, lengths, window):
    """[B, N, L] in sight."""
    i = torch.arange(N, device="cuda")[None, :, None]
    j = torch.arange(L, device="cuda")[None, None]
    at = cached[:, None, None] + i
    see = (j <= at) & (i < lengths[:, None, None]) & (at < L) & (cached[:, None, None] >= 0)
    return see if window is None else see & (j > at - window)


PROMPTS = [  # N, H, J, D, L, cap, bias, window
    (1, 2, 1, 64, 70, None, False, None), (5, 4, 4, 40, 300, 3.0, False, None), (130, 4, 2, 128, 400, None, True, None), (257, 2, 2, 72, 600, 20.0, True, 100),
    (300, 3, 1, 64, 301, None, False, 40),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", PROMPTS, ids=str)
def test_prompts_behind_a_cache(case, dtype):
    N, H, J, D, L, cap, bias, window = case
    B = 5
    g = gen(N + L)
    q, k, v = randn(g, B, N, H, D, dtype=dtype), randn(g, B, N, J, D, dtype=dtype), randn(g, B, N, J, D, dtype=dtype)
    # in the middle, at the very end, empty, over the end, outside
    cached = torch.tensor([(L - N) // 2, L - N, 0, L - max(1, N // 2), -1], device="cuda", dtype=torch.int32)
    lengths = torch.tensor([N, max(1, N - 3), 0, N, N], device="cuda", dtype=torch.int32)
    slopes = torch.rand(H, generator=g, device="cuda") * 0.1 if bias else None
    kc, vc = randn(g, B, L, J, D, dtype=dtype), randn(g, B, L, J, D, dtype=dtype)
    for b in range(B):  # unused slots hold anything
        kc[b, max(0, int(cached[b])):] = float("nan")
        vc[b, max(0, int(cached[b])):] = float("inf")
    kw, vw = kc.clone(), vc.clone()
    for b in range(B):
        for t in range(int(lengths[b])):
            if cached[b] >= 0 and cached[b] + t < L:
                kw[b, cached[b] + t], vw[b, cached[b] + t] = k[b, t], v[b, t]
    y = cf.flare_causal_attention_prefill(q, k, v, kc, vc, cached=cached, lengths=lengths, cap=cap, slopes=slopes, window=window)
    assert torch.equal(kc.view(torch.int16), kw.view(torch.int16)) and torch.equal(vc.view(torch.int16), vw.view(torch.int16))
    see = behind_a_cache(B, N, L, cached, lengths, window)
    o = orc.Attention(q.double(), kw.double().nan_to_num(0, 0, 0), vw.double().nan_to_num(0, 0, 0), see, _resolve_attn_scale(None, D), cap,
                      None if slopes is None else slopes.double(), cached, eps=torch.finfo(dtype).eps / 2)
    close(y, o.y, o.y_off, "y")
    assert not y[2].any() and not y[4].any()


def test_prompt_in_parts_with_a_prefix():
    g = gen(2)
    B, N, H, D = 2, 150, 2, 64
    q, k, v = (randn(g, B, N, H, D, dtype=torch.float16) for _ in range(3))
    prefix = torch.arange(N, device="cuda")[None].repeat(B, 1) < 40
    kc, vc = (torch.zeros(B, 200, H, D, device="cuda", dtype=torch.float16) for _ in range(2))
    whole = cf.flare_causal_attention(q, k, v, prefix=prefix)
    first = cf.flare_causal_attention_prefill(q[:, :70], k[:, :70], v[:, :70], kc, vc, prefix=prefix[:, :70])
    rest = cf.flare_causal_attention_prefill(q[:, 70:], k[:, 70:], v[:, 70:], kc, vc, cached=torch.full((B,), 70, device="cuda"))
    see = orc.in_sight(N, None, prefix)
    o = orc.Attention(q.double(), k.double(), v.double(), see, _resolve_attn_scale(None, D), eps=2.0 ** -11)
    close(whole, o.y, o.y_off, "whole")
    close(torch.cat([first, rest], 1), o.y, o.y_off, "parts")
    assert cf.flare_causal_attention_prefill(q[:, :0], k[:, :0], v[:, :0], kc, vc).shape == (B, 0, H, D)


STEPS = [  # H, J, D, L, cap, bias, window
    (1, 1, 64, 1, None, False, None), (8, 8, 64, 100, None, True, None), (8, 2, 128, 1000, 30.0, False, None), (24, 1, 72, 333, None, True, 50),
    (16, 1, 40, 64, 5.0, False, 1), (4, 4, 96, 2000, None, False, 700), (40, 1, 128, 515, 8.0, True, None), (2, 1, 8, 17, None, False, None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", STEPS, ids=str)
def test_single_tokens(case, dtype):
    H, J, D, L, cap, bias, window = case
    B = 6
    g = gen(L + D)
    q, k, v = randn(g, B, H, D, dtype=dtype), randn(g, B, J, D, dtype=dtype), randn(g, B, J, D, dtype=dtype)
    cached = torch.tensor([0, L - 1, L // 2, -1, L, min(15, L - 1)], device="cuda")
    slopes = torch.rand(H, generator=g, device="cuda") * 0.1 if bias else None
    kc, vc = randn(g, B, L, J, D, dtype=dtype), randn(g, B, L, J, D, dtype=dtype)
    for b in range(B):
        kc[b, max(0, int(cached[b])):] = float("nan")
        vc[b, max(0, int(cached[b])):] = float("inf")
    kw, vw = kc.clone(), vc.clone()
    for b in range(B):
        if 0 <= cached[b] < L:
            kw[b, cached[b]], vw[b, cached[b]] = k[b], v[b]
    y = cf.flare_causal_attention_decode(q, k[:, None], v[:, None], kc, vc, cached, cap=cap, slopes=slopes, window=window)
    assert torch.equal(kc.view(torch.int16), kw.view(torch.int16)) and torch.equal(vc.view(torch.int16), vw.view(torch.int16))
    see = behind_a_cache(B, 1, L, cached, torch.ones(B, device="cuda"), window)
    o = orc.Attention(q[:, None].double(), kw.double().nan_to_num(0, 0, 0), vw.double().nan_to_num(0, 0, 0), see, _resolve_attn_scale(None, D), cap,
                      None if slopes is None else slopes.double(), cached, eps=torch.finfo(dtype).eps / 2)
    close(y, o.y[:, 0], o.y_off[:, 0], "y")
    assert not y[3].any() and not y[4].any()


@pytest.mark.parametrize("heads", [(4, 8, 2), (4, 18, 1), (60, 8, 2)], ids=str)
@pytest.mark.parametrize("parts", range(1, 11))
def test_caches_in_every_number_of_parts(parts, heads):
    # parts of 64 keys and more: up to eight are joined by the blocks among themselves, more of them, or those of many rows, by a second kernel
    B, H, J = heads
    D, L = 72, 64 * parts - 3
    g = gen(parts)
    q, k, v = randn(g, B, H, D, dtype=torch.float16), randn(g, B, J, D, dtype=torch.float16), randn(g, B, J, D, dtype=torch.float16)
    kc, vc = randn(g, B, L, J, D, dtype=torch.float16), randn(g, B, L, J, D, dtype=torch.float16)
    cached = torch.tensor([L - 1, -1, 0, L // 3], device="cuda").repeat(B // 4)  # (of the last ones most parts have no keys)
    kw, vw = kc.clone(), vc.clone()
    for b in range(B):
        if b % 4 != 1:
            kw[b, cached[b]], vw[b, cached[b]] = k[b], v[b]
    y = cf.flare_causal_attention_decode(q, k, v, kc, vc, cached)
    o = orc.Attention(q[:, None].double(), kw.double(), vw.double(), behind_a_cache(B, 1, L, cached, torch.ones(B, device="cuda"), None),
                      _resolve_attn_scale(None, D), None, None, cached, eps=2.0 ** -11)
    close(y, o.y[:, 0], o.y_off[:, 0], "y")
    assert not y[1::4].any()


def test_tokens_follow_a_prompt():
    # a whole sequence at once, as a prompt and tokens one by one
    g = gen(4)
    B, N, H, J, D = 2, 90, 4, 2, 64
    q, k, v = randn(g, B, N, H, D, dtype=torch.bfloat16), randn(g, B, N, J, D, dtype=torch.bfloat16), randn(g, B, N, J, D, dtype=torch.bfloat16)
    kc, vc = (torch.empty(B, 100, J, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    how = dict(cap=10.0, slopes=torch.tensor([0.1, 0.2, 0.3, 0.4], device="cuda"), window=33)
    o = orc.Attention(q.double(), k.double(), v.double(), orc.in_sight(N, window=33).cuda(), D ** -0.5, 10.0, how["slopes"].double(), eps=2.0 ** -8)
    close(cf.flare_causal_attention(q, k, v, **how), o.y, o.y_off, "whole")
    parts = [cf.flare_causal_attention_prefill(q[:, :60], k[:, :60], v[:, :60], kc, vc, **how)]
    cached = torch.full((B,), 60, device="cuda", dtype=torch.int32)
    for t in range(60, N):
        parts.append(cf.flare_causal_attention_decode(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], kc, vc, cached, **how))
        cached += 1
    close(torch.cat(parts, 1), o.y, o.y_off, "parts")


def test_caches_of_other_layouts():
    g = gen(6)
    B, H, D, L = 2, 4, 64, 50
    q, k, v = (randn(g, B, H, D, dtype=torch.float16) for _ in range(3))
    base = [randn(g, B, L, H, D, dtype=torch.float16) for _ in range(2)]
    cached = torch.tensor([20, 49], device="cuda")
    want = [t.clone() for t in base]
    y = cf.flare_causal_attention_decode(q, k, v, *want, cached)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in base]
    assert torch.equal(cf.flare_causal_attention_decode(q, k, v, *heads_first, cached), y)
    both = torch.stack(base, 2)  # keys and values of a token side by side
    assert torch.equal(cf.flare_causal_attention_decode(q, k, v, both[:, :, 0], both[:, :, 1], cached), y)
    for a, b, c in zip(want, heads_first, (both[:, :, 0], both[:, :, 1])):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_decode_from_a_graph():
    g = gen(9)
    B, H, J, D, L = 3, 8, 2, 128, 700
    q, k, v = randn(g, B, H, D, dtype=torch.bfloat16), randn(g, B, J, D, dtype=torch.bfloat16), randn(g, B, J, D, dtype=torch.bfloat16)
    kc, vc = randn(g, B, L, J, D, dtype=torch.bfloat16), randn(g, B, L, J, D, dtype=torch.bfloat16)
    cached = torch.tensor([5, 300, 690], device="cuda", dtype=torch.int32)
    k2, v2, c2 = kc.clone(), vc.clone(), cached.clone()
    want = []
    for _ in range(3):
        want.append(cf.flare_causal_attention_decode(q, k, v, k2, v2, c2))
        c2 += 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cf.flare_causal_attention_decode(q, k, v, kc, vc, cached)
        cached += 1
    for w in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w)
    assert torch.equal(kc, k2) and torch.equal(vc, v2)
