"""gpu: attention at the ends of what its types hold: gradients in fp16 that are small or large, weights below fp16's normal numbers, scales
and caps whose quotient is far from one, scores of minus infinity."""
import pytest
import torch

import causal_flare as cf
from causal_flare import _mixers, attention
from oracle import mixers_oracle as orc

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -11  # half a step of fp16
STEP = 2.0 ** -25  # half the smallest step of fp16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def gradients(q, k, v, dy, **how):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    y = cf.flare_causal_attention(q, k, v, **how)
    return torch.autograd.grad(y, (q, k, v), dy)


def exact(q, k, v, dy, scale, **how):
    see = orc.in_sight(q.shape[1], how.get("documents"), None, how.get("window")).to(q.device)
    s = how.get("slopes")
    o = orc.Attention(q.double(), k.double(), v.double(), see, scale, how.get("cap"), None if s is None else s.double(), dy=dy.double())
    return o.dq, o.dk, o.dv


def near(got, want, off, what):
    """Norms: `off` of the result's, and the rounding of values below fp16's normal numbers."""
    assert torch.isfinite(got).all(), what
    err, ref = float((got.double() - want).norm()), float(want.norm())
    assert err <= off * ref + STEP * want.numel() ** 0.5, f"{what}: {err / ref:.2e}, {off:.2e} allowed"


# Rows of at most 32 keys sum P dP itself, so dQ and dK are as near as their own rounding (1.01: of what is not quite the result), dS in two parts (half^2)
# and fp32 allow.  fp32: exponents of up to 17 (scores up to 12) are off by 2^-22 a few times over, dP - delta is a third of either: 100 2^-22.
OFF = 1.01 * HALF + HALF ** 2 + 100 * 2.0 ** -22


SIZES = [  # of dy and of v; scale
    (1e-6, 1, 16), (1e-5, 1, 16), (1e-4, 1, 16), (1, 1, 16), (1e-3, 1e-3, 16), (1e3, 1, 0.01), (3e3, 8, 0.01), (2, 1e4, 0.01),
]


@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("wide", ["q", "k"])
@pytest.mark.parametrize("size, values, scale", SIZES)
def test_gradients_in_fp16_of_every_size(size, values, scale, wide, cap):
    # dS of 1e-6 has five bits in fp16, and one of 1e5 none; dQ = scale dS K (`wide`: or dK) is a normal number in either case.  Scores have a deviation of 2.
    B, N, H, J, D = 2, 300, 4, 2, 64
    g = gen(int(1000 * size) + 3)
    one = max(1.0, (0.25 / scale) ** 0.5)
    q_size, k_size = (one, 0.25 / scale / one) if wide == "q" else (0.25 / scale / one, one)
    q, k = (randn(g, B, N, H, D) * q_size).half(), (randn(g, B, N, J, D) * k_size).half()
    v, dy = (randn(g, B, N, J, D) * values).half(), (randn(g, B, N, H, D) * size).half()
    how = dict(window=32, cap=cap)
    got, want = gradients(q, k, v, dy, scale=scale, **how), exact(q, k, v, dy, scale, **how)
    near(got[0], want[0], OFF, "dq")
    near(got[1], want[1], OFF, "dk")
    near(got[2], want[2], OFF + 1.01 * HALF, "dv")  # (every weight rounded once as well)


def test_rows_of_very_different_gradients_in_fp16():
    # a document whose gradients are ten thousand times another's, in one row, and a row between theirs
    B, N, H, D, scale = 2, 400, 2, 64, 16
    g = gen(1)
    q, k, v = (randn(g, B, N, H, D) * (0.25 / scale)).half(), randn(g, B, N, H, D, dtype=torch.float16), randn(g, B, N, H, D, dtype=torch.float16)
    docs = (torch.arange(N, device="cuda")[None].repeat(B, 1) >= 170).int()
    size = torch.where(docs == 0, 1.0, 1e-4)
    size[1] = 1e-2
    dy = (randn(g, B, N, H, D) * size[..., None, None]).half()
    how = dict(window=32, documents=docs)
    got, want = gradients(q, k, v, dy, scale=scale, **how), exact(q, k, v, dy, scale, **how)
    for name, a, b in zip(("dq", "dk"), got, want):
        for row, part in ((0, slice(0, 170)), (0, slice(170, N)), (1, slice(0, N))):
            # (dK's sums go by the row's largest |dY| |V|: with a second part that ends 2^38 below it, terms of 1e-4 of that keep 24 bits)
            near(a[row, part], b[row, part], OFF, name)


def test_a_row_whose_gradient_is_not_finite_leaves_the_others_alone():
    B, N, H, D = 2, 200, 2, 64
    g = gen(2)
    q, k, v, dy = (randn(g, B, N, H, D, dtype=torch.float16) for _ in range(4))
    docs = (torch.arange(N, device="cuda")[None].repeat(B, 1) >= 100).int()
    clean = gradients(q, k, v, dy, documents=docs)
    for value in (float("inf"), float("nan")):
        bad = dy.clone()
        bad[0, 150, 1, 3] = value
        got = gradients(q, k, v, bad, documents=docs)
        # another document: all but dV, whose products have 0 times what is not finite, as they have in any form with matrix products
        assert torch.equal(got[0][0, :100], clean[0][0, :100]) and torch.equal(got[1][0, :100], clean[1][0, :100])
        for a, c in zip(got, clean):
            assert torch.equal(a[1], c[1]) and torch.equal(a[0, :, 0], c[0, :, 0])  # another row of the batch, another head


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 6e4])
def test_padding_does_not_count_in_fp16(value):
    # neither for the norms by which dS is scaled, nor for anything else
    B, N, H, J, D = 2, 300, 4, 2, 64
    g = gen(7)
    q, k, v, dy = (randn(g, B, N, h, D, dtype=torch.float16) for h in (H, J, J, H))
    docs = (torch.rand(B, N, generator=g, device="cuda") < 0.015).int().cumsum(1).int()
    docs = torch.where(docs % 3 == 0, -1, docs)
    pad = (docs < 0)[..., None, None]
    assert pad.any()
    clean = gradients(q, k, v, dy, documents=docs)
    for a, c in zip(gradients(*(t.masked_fill(pad, value) for t in (q, k, v, dy)), documents=docs), clean):
        assert torch.equal(a, c)


def test_a_backward_without_the_forwards_plan_in_fp16():
    B, N, H, J, D = 2, 300, 4, 2, 64
    g = gen(8)
    q, k, v, dy = (randn(g, B, N, h, D, dtype=torch.float16) for h in (H, J, J, H))
    want = gradients(q, k, v, dy, window=100)
    a = attention._fill(q, k, v, (D ** -0.5, 0.0, 100), None)
    out, lse = torch.empty_like(q), torch.empty(B, H, 384, device="cuda")
    grads = [torch.empty_like(t) for t in (q, k, v)]
    a.y, a.lse = out.data_ptr(), lse.data_ptr()
    _mixers.run("flare_attention_forward", a, q.device, "flare_attention_forward_workspace_bytes")
    a.dy = dy.data_ptr()
    _mixers.put_strides(a, "dy", dy, "bnh")
    a.dq, a.dk, a.dv = (t.data_ptr() for t in grads)
    _mixers.run("flare_attention_backward", a, q.device, "flare_attention_backward_workspace_bytes")
    for x, z in zip(grads, want):
        assert torch.equal(x, z)


def test_gradients_of_nothing_are_nothing():
    g = gen(4)
    q, k, v = (randn(g, 1, 70, 2, 64, dtype=torch.float16) for _ in range(3))
    for t in gradients(q, k, v, torch.zeros_like(q)):
        assert not t.any()
    dq, dk, dv = gradients(q, k, torch.zeros_like(v), torch.ones_like(q))
    assert not dq.any() and not dk.any() and dv.any()


def test_gradients_in_fp16_from_a_graph():
    # replayed with gradients of another size: what they are scaled by is found anew
    B, N, H, D = 2, 150, 2, 64
    g = gen(5)
    q, k, v, dy = (randn(g, B, N, H, D, dtype=torch.float16) for _ in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        return torch.autograd.grad(cf.flare_causal_attention(*leaves), leaves, dy)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for size in (1, 1e3, 1e-4):
        dy.copy_(randn(gen(6), B, N, H, D) * size)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("form", ["whole", "prompt", "step"])
def test_small_weights_beside_a_large_one_in_fp16(form):
    # the first key has a weight of one and a value of zero, the others 1.4 2^-20: fp16's steps there are a twenty-second of that.  Tolerance: half a step for a
    # weight and for what comes out, scores of 20 that are off by 2^-19 in all, and products that add 16 tokens at a time, each sum cut off in its last bit (2^-23).
    N, D = 3000, 64
    q, k = torch.zeros(1, N, 1, D, device="cuda").half(), torch.zeros(1, N, 1, D, device="cuda").half()
    v = torch.ones(1, N, 1, D, device="cuda").half()
    q[..., 0] = 1
    k[:, 0, :, 0] = 13.53
    v[:, 0] = 0
    w = torch.exp(-k[0, 0, 0, 0].double())
    i = torch.arange(N, device="cuda", dtype=torch.float64)
    want = i * w / (1 + i * w)
    off = 2 * HALF + 2.0 ** -19 + N / 16 * 2.0 ** -23
    if form == "whole":
        y = cf.flare_causal_attention(q, k, v, scale=1.0)[0, :, 0]
        dv = gradients(q, k, v, torch.full_like(v, 500), scale=1.0)[2][0, 1:, 0].double()
        each = (500 * w / (1 + i * w)).flip(0).cumsum(0).flip(0)[1:, None]
        normal = each[:, 0] > 2.0 ** -14
        assert normal.sum() > 2900 and float(((dv - each).abs() / each)[normal].max()) <= off
    else:
        kc, vc = k.clone(), v.clone()
        if form == "prompt":
            y = cf.flare_causal_attention_prefill(q, k, v, kc, vc, scale=1.0)[0, :, 0]
        else:
            # so many rows that a cache is read by one block: a quarter of the keys meet the large one
            want, rows = want[-1:], 75
            kc, vc = (t.expand(rows, N, 8, D).contiguous() for t in (kc, vc))
            one = [t[:, -1].expand(rows, 8, D).contiguous() for t in (q, k, v)]
            y = cf.flare_causal_attention_decode(*one, kc, vc, torch.full((rows,), N - 1, device="cuda", dtype=torch.int32), scale=1.0)[0, :1]
    assert float(((y.double() - want[:, None]).abs() - STEP).max() / want.max()) <= off
    many = want > 0.1 * want.max()  # (of the others y is a few of fp16's smallest steps)
    assert float(((y.double() - want[:, None]).abs() / want[:, None])[many].max()) <= off


@pytest.mark.parametrize("scale, cap", [(5e-4, 1024.0), (1e-5, 1000.0), (2e-9, 300.0), (1e4, 0.01), (0.125, 50.0)])
def test_scales_and_caps_whose_quotient_is_far_from_one(scale, cap):
    # Two keys, a score of 0.349 (before tanh) and one of 0, and a bias that makes them equal: y is the mean, and moves by half of what the
    # score is off.  That is cap 2^-21 at most, and half a step for the weights and for y.
    D = 64
    side = (0.349 * cap / scale / D) ** 0.5
    q = torch.full((1, 2, 1, D), side, device="cuda").half()
    k = q.clone()
    k[:, 1] = 0
    score = cap * torch.tanh(scale * (q[0, 1, 0].double() @ k[0, 0, 0].double()) / cap)
    v = torch.ones(1, 2, 1, D, device="cuda").half()
    v[:, 1] = -1
    dy = torch.ones_like(q)
    how = dict(cap=cap, slopes=score[None].float())
    score_off = cap * 2.0 ** -21 + 2 * float(score) * 2.0 ** -24
    y = cf.flare_causal_attention(q, k, v, scale=scale, **how)
    o = orc.Attention(q.double(), k.double(), v.double(), orc.in_sight(2).cuda(), scale, cap, how["slopes"].double())
    assert float((y.double() - o.y).abs().max()) <= score_off / 2 + 2 * HALF
    for name, a, b in zip(("dq", "dk", "dv"), gradients(q, k, v, dy, scale=scale, **how), exact(q, k, v, dy, scale, **how)):
        near(a, b, OFF + score_off + HALF, name)
    zero = torch.zeros_like(q)
    assert torch.equal(cf.flare_causal_attention(zero, zero, v, scale=scale, cap=cap)[0, 1], torch.zeros(1, D, device="cuda").half())


@pytest.mark.parametrize("L", [60, 700, 3000])
def test_a_token_none_of_whose_scores_is_above_minus_infinity(L):
    # no weights: zeros, in however many parts the cache is read
    q, k = torch.full((2, 4, 64), 1e30, device="cuda").bfloat16(), torch.full((2, 2, 64), -1e30, device="cuda").bfloat16()
    kc, vc = k[:, None].expand(2, L, 2, 64).contiguous(), torch.ones(2, L, 2, 64, device="cuda").bfloat16()
    y = cf.flare_causal_attention_decode(q, k, torch.ones_like(k), kc, vc, torch.tensor([L - 1, 3], device="cuda", dtype=torch.int32))
    assert not y.any()


@pytest.mark.parametrize("N", [5, 200])
def test_rows_none_of_whose_scores_is_above_minus_infinity(N):
    q, k = torch.full((1, N, 2, 64), 1e30, device="cuda").bfloat16(), torch.full((1, N, 2, 64), -1e30, device="cuda").bfloat16()
    v = torch.ones_like(k)
    assert not cf.flare_causal_attention(q, k, v).any()
    for t in gradients(q, k, v, torch.ones_like(q)):
        assert not t.any()
