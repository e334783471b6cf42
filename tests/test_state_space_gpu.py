"""gpu: the short causal convolution and the selective scan against the oracle in 64 bits (gradients by its automatic
differentiation): types, sizes around the tiles, documents, padding, carried states, segments of long rows, strided inputs.

Tolerances.  One rounding to a type costs half a step, eps / 2 of the value; everything in front of it is fp32.  A step of the
recurrence multiplies by a factor that is off by 2^-22 at most (argument, ex2, product) and adds a term off by as much, so behind N
tokens a sum is off by N 2^-22 of the sum of its terms' magnitudes; sums and products behind it add a dozen roundings of
2^-24.  `scale` below is that sum of magnitudes: the oracle itself, run on absolute values."""
import pytest
import torch

import causal_flare as cf
from oracle import mixers_oracle as orc

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, scale, steps, what):
    """Every element: half a step of the result, and `steps` roundings of 2^-22 of what was summed."""
    assert got.shape == want.shape, what
    tol = half_step(got.dtype) * want.abs() * 1.01 + (steps + 16) * 2.0 ** -22 * scale + torch.finfo(got.dtype).tiny * half_step(got.dtype)
    got = got.detach().double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max()):.3e}"


def near(got, want, dtype, steps, what):
    """Norms: half a step for every element, and `steps` roundings of 2^-22.  Gradients are sums over tokens, channels and states whose terms cancel:
    the norm of the terms is taken as at most 30 times the sum's."""
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    err, ref = float((got - want).norm()), float(want.norm())
    assert err <= (half_step(dtype) * 1.01 + 30 * (steps + 16) * 2.0 ** -22) * ref + torch.finfo(dtype).tiny * half_step(dtype) * want.numel() ** 0.5, f"{what}: {err / max(ref, 1e-30):.3e}"


def ids(kind, B, N, g):
    if kind is None:
        return None
    t = torch.arange(N, device="cuda")
    if kind == "every":  # every token a document
        return t[None].repeat(B, 1).int()
    if kind == "padding":
        return torch.full((B, N), -1, device="cuda", dtype=torch.int32)
    d = (torch.rand(B, N, generator=g, device="cuda") < 0.15).int().cumsum(1)
    if kind == "again":  # ids that come back are other documents
        d = d % 2
    if kind == "holes":  # padding in front, between documents and at the end
        d = torch.where(d % 4 == 0, -1, d)
    return d.int()


# ---- convolution -------------------------------------------------------------------------------------------------------

CONV = [  # B, N, C, W, bias, silu, documents
    (1, 1, 1, 2, True, False, None), (1, 1, 8, 4, True, True, None), (2, 2, 24, 3, False, True, None), (3, 3, 16, 4, True, True, "some"),
    (2, 33, 264, 4, True, True, None), (1, 100, 13, 3, True, False, "again"), (2, 257, 40, 2, False, False, "holes"),
    (1, 70, 520, 4, True, True, "every"), (2, 9, 8, 4, True, True, "padding"), (4, 600, 256, 4, True, True, "holes"),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CONV, ids=str)
def test_conv_and_its_gradients(case, dtype):
    B, N, C, W, with_bias, silu, kind = case
    g = gen(N * 7 + C)
    x, w = randn(g, B, N, C, dtype=dtype), randn(g, C, W)
    bias = randn(g, C) if with_bias else None
    docs = ids(kind, B, N, g)
    dy = randn(g, B, N, C, dtype=dtype)
    leaves = [t for t in (x, w, bias) if t is not None]
    for t in leaves:
        t.requires_grad_()
    y = cf.flare_causal_conv(x, w, bias, activation="silu" if silu else None, documents=docs)
    assert y.dtype == dtype
    got = torch.autograd.grad(y, leaves, dy)
    exact = [t.detach().double().requires_grad_() for t in leaves]
    want = orc.causal_conv(exact[0], exact[1], exact[2] if with_bias else None, silu=silu, documents=docs)[0]
    grads = torch.autograd.grad(want, exact, dy.double())
    size = orc.causal_conv(exact[0].abs(), exact[1].abs(), exact[2].abs() if with_bias else None, documents=docs)[0]
    close(y, want.detach(), size.detach(), W, "y")
    for name, a, b, t in zip(("dx", "dw", "dbias"), got, grads, (dtype, torch.float32, torch.float32)):
        assert a.dtype == t
        near(a, b, t, W, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
def test_conv_weight_types(dtype, wdtype):
    g = gen(3)
    x, w, b = randn(g, 2, 50, 32, dtype=dtype), randn(g, 32, 4, dtype=wdtype).requires_grad_(), randn(g, 32, dtype=wdtype).requires_grad_()
    y = cf.flare_causal_conv(x, w, b, activation="silu")
    dw, db = torch.autograd.grad(y, (w, b), torch.ones_like(y))
    ex = [t.detach().double().requires_grad_() for t in (w, b)]
    want = torch.autograd.grad(orc.causal_conv(x.double(), *ex, silu=True)[0].sum(), ex)
    near(dw, want[0], wdtype, 4, "dw")
    near(db, want[1], wdtype, 4, "db")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("C", [16, 5])
def test_conv_prompt_and_tokens_continue_one_another(dtype, W, C):
    g = gen(W)
    B, N = 3, 41
    x, w, b = randn(g, B, N, C, dtype=dtype), randn(g, C, W), randn(g, C)
    state = randn(g, B, W - 1, C, dtype=dtype)
    lengths = torch.tensor([N, 0, 2], device="cuda")
    y, out = cf.flare_causal_conv_prefill(x, w, b, state, activation="silu", lengths=lengths)
    want, left = orc.causal_conv(x.double(), w.double(), b.double(), state.double(), True, lengths=lengths)
    size = orc.causal_conv(x.double().abs(), w.double().abs(), b.double().abs(), state.double().abs(), lengths=lengths)[0]
    close(y, want, size, W, "y")
    assert torch.equal(out.double(), left)  # copies
    # the same tokens one by one, and in two parts
    whole, end = cf.flare_causal_conv_prefill(x, w, b, state, activation="silu")
    st = state.clone()
    for t in range(N):
        yt, same = cf.flare_causal_conv_decode(x[:, t] if t % 2 else x[:, t:t + 1], w, b, st, activation="silu")
        assert same.data_ptr() == st.data_ptr() and torch.equal(yt.reshape(B, C), whole[:, t])
    assert torch.equal(st, end)
    ya, mid = cf.flare_causal_conv_prefill(x[:, :1], w, b, state, activation="silu")
    yb, end2 = cf.flare_causal_conv_prefill(x[:, 1:], w, b, mid, activation="silu")
    assert torch.equal(torch.cat([ya, yb], 1), whole) and torch.equal(end2, end)
    empty, same = cf.flare_causal_conv_prefill(x[:, :0], w, b, state)
    assert empty.shape == (B, 0, C) and torch.equal(same, state)


# ---- scan --------------------------------------------------------------------------------------------------------------


def scan_inputs(g, B, N, C, S, G, dtype, D=True, z=True, bias=True, lead=None):
    lead = (B, N) if lead is None else lead
    t = dict(x=randn(g, *lead, C, dtype=dtype), dt=(0.5 * randn(g, *lead, C) - (0 if bias else 3)).to(dtype),
             A=-torch.exp(randn(g, C, S) * 0.5 + 0.5), B=randn(g, *lead, G, S, dtype=dtype), C=randn(g, *lead, G, S, dtype=dtype))
    if D:
        t["D"] = randn(g, C)
    if z:
        t["z"] = randn(g, *lead, C, dtype=dtype)
    if bias:
        t["dt_bias"] = randn(g, C) * 0.5 - 3
    return t


def magnitudes(t, **more):
    """The oracle on absolute values, with the same factors: delta is positive in these tests."""
    a = {k: (v.double() if k in ("A", "dt", "dt_bias") else v.double().abs()) for k, v in t.items() if k != "z"}
    y, h = orc.selective_scan(**a, **more)
    return y * t["z"].double().abs() if "z" in t else y, h


SCAN = [  # B, N, C, S, G, D, z, bias and softplus, documents
    (1, 1, 1, 8, 1, False, False, True, None), (1, 1, 64, 16, 1, True, True, True, None), (2, 3, 72, 16, 1, True, True, True, None),
    (2, 31, 8, 32, 1, True, False, True, None), (1, 33, 200, 8, 2, True, True, True, "some"), (2, 100, 100, 16, 4, False, True, True, "again"),
    (2, 65, 128, 16, 2, True, True, True, "holes"), (1, 40, 64, 16, 1, True, True, True, "every"), (2, 20, 16, 32, 1, True, True, True, "padding"),
    (1, 600, 64, 16, 1, True, True, True, None), (1, 700, 40, 8, 1, True, False, True, "holes"), (2, 420, 70, 32, 2, True, True, True, "some"),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", SCAN, ids=str)
def test_scan_and_its_gradients(case, dtype):
    B, N, C, S, G, D, z, bias, kind = case
    g = gen(N + 3 * C)
    t = scan_inputs(g, B, N, C, S, G, dtype, D, z, bias)
    docs = ids(kind, B, N, g)
    dy = randn(g, B, N, C, dtype=dtype)
    for v in t.values():
        v.requires_grad_()
    y = cf.flare_selective_scan(**t, dt_softplus=True, documents=docs)
    assert y.dtype == dtype
    got = torch.autograd.grad(y, list(t.values()), dy)
    exact = {k: v.detach().double().requires_grad_() for k, v in t.items()}
    want = orc.selective_scan(**exact, softplus=True, documents=docs)[0]
    grads = torch.autograd.grad(want, list(exact.values()), dy.double())
    close(y, want.detach(), magnitudes({k: v.detach() for k, v in t.items()}, softplus=True, documents=docs)[0], N, "y")
    for (name, v), a, b in zip(t.items(), got, grads):
        assert a.dtype == v.dtype, name
        near(a, b, v.dtype, N, name)


def test_scan_without_softplus_and_positive_exponents():
    g = gen(5)
    t = scan_inputs(g, 2, 40, 24, 16, 1, torch.float32, True, False, False)
    t["dt"] = t["dt"].abs() * 0.05
    t["A"] = randn(g, 24, 16) * 0.5
    want = orc.selective_scan(**{k: v.double() for k, v in t.items()})[0]
    close(cf.flare_selective_scan(**t), want, magnitudes(t)[0], 40, "y")


def test_scan_of_negative_time_steps():
    # without softplus a time step is what it is, also where its sum over a part of a long row is negative
    g = gen(6)
    t = scan_inputs(g, 1, 900, 16, 16, 1, torch.float32, True, False, False)
    t["dt"] = randn(g, 1, 900, 16) * 0.02 - 0.01
    t["A"] = randn(g, 16, 16) * 0.2
    for v in t.values():
        v.requires_grad_()
    y = cf.flare_selective_scan(**t)
    got = torch.autograd.grad(y.sum(), list(t.values()))
    ex = {k: v.detach().double().requires_grad_() for k, v in t.items()}
    want = orc.selective_scan(**ex)[0]
    near(y, want.detach(), torch.float32, 900, "y")
    for name, a, b in zip(t, got, torch.autograd.grad(want.sum(), list(ex.values()))):
        near(a, b, torch.float32, 900, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 41, 24, 16, 1), (2, 500, 16, 8, 2), (2, 300, 37, 32, 1)], ids=str)
def test_scan_prompt_and_tokens_continue_one_another(dtype, shape):
    B, N, C, S, G = shape
    g = gen(N)
    t = scan_inputs(g, B, N, C, S, G, dtype)
    state = randn(g, B, C, S)
    lengths = torch.tensor([N, 0, 7][:B], device="cuda", dtype=torch.int32)
    y, out = cf.flare_selective_scan_prefill(**t, state=state, dt_softplus=True, lengths=lengths)
    ex = {k: v.double() for k, v in t.items()}
    want, left = orc.selective_scan(**ex, state=state.double(), softplus=True, lengths=lengths)
    ys, hs = magnitudes(t, state=state.double().abs(), softplus=True, lengths=lengths)
    close(y, want, ys, N, "y")
    close(out, left, hs, N, "state")
    assert torch.equal(out[1], state[1])
    # token by token: the oracle is the measure of both
    st = state.clone()
    want, left = orc.selective_scan(**ex, state=state.double(), softplus=True)
    ys, hs = magnitudes(t, state=state.double().abs(), softplus=True)
    for n in range(min(N, 60)):
        cut = {k: (v[:, n] if k in ("x", "dt", "z", "B", "C") else v) for k, v in t.items()}
        yn, same = cf.flare_selective_scan_decode(**cut, state=st, dt_softplus=True)
        assert same.data_ptr() == st.data_ptr()
        close(yn, want[:, n], ys[:, n], n + 1, f"token {n}")
    empty, same = cf.flare_selective_scan_prefill(**{k: (v[:, :0] if k in ("x", "dt", "z", "B", "C") else v) for k, v in t.items()}, state=state)
    assert empty.shape == (B, 0, C) and torch.equal(same, state)


def test_scan_of_large_time_steps_and_saturated_factors():
    # softplus of large values is the value, the factors underflow to 0 and stay finite
    g = gen(8)
    t = scan_inputs(g, 1, 50, 16, 16, 1, torch.float32)
    t["dt"] = t["dt"] + 30 * (torch.rand(1, 50, 16, generator=g, device="cuda") < 0.3)
    for v in t.values():
        v.requires_grad_()
    y = cf.flare_selective_scan(**t, dt_softplus=True)
    got = torch.autograd.grad(y.sum(), list(t.values()))
    ex = {k: v.detach().double().requires_grad_() for k, v in t.items()}
    want = torch.autograd.grad(orc.selective_scan(**ex, softplus=True)[0].sum(), list(ex.values()))
    for name, a, b in zip(t, got, want):
        near(a, b, torch.float32, 50, name)


# ---- both ----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_padding_may_hold_anything(value):
    g = gen(11)
    B, N, C = 2, 70, 40
    docs = ids("holes", B, N, g)
    pad = docs < 0
    x, w, b = randn(g, B, N, C), randn(g, C, 4), randn(g, C)
    t = scan_inputs(g, B, N, C, 16, 1, torch.float32)
    dy = randn(g, B, N, C)

    def both(fill):
        def put(v):
            return v.masked_fill(pad.view(B, N, *[1] * (v.dim() - 2)), value) if fill else v.clone()
        u = {k: (put(v) if k in ("x", "dt", "z", "B", "C") else v.clone()).requires_grad_() for k, v in t.items()}
        xx = put(x).requires_grad_()
        ww = w.clone().requires_grad_()
        y1 = cf.flare_causal_conv(xx, ww, b, activation="silu", documents=docs)
        y2 = cf.flare_selective_scan(**u, dt_softplus=True, documents=docs)
        return (y1, y2, *torch.autograd.grad(y1, (xx, ww), put(dy)), *torch.autograd.grad(y2, list(u.values()), put(dy)))

    for a, c in zip(both(True), both(False)):
        assert torch.equal(a, c)
    # behind a prompt's length
    lengths = torch.tensor([30, 64], device="cuda")
    late = torch.arange(N, device="cuda")[None] >= lengths[:, None]
    dirty = {k: (v.masked_fill(late.view(B, N, *[1] * (v.dim() - 2)), value) if k in ("x", "dt", "z", "B", "C") else v) for k, v in t.items()}
    for softplus in (True, False):  # (without it these states overflow, the same way on both sides)
        for a, c in zip(cf.flare_selective_scan_prefill(**dirty, lengths=lengths, dt_softplus=softplus),
                        cf.flare_selective_scan_prefill(**t, lengths=lengths, dt_softplus=softplus)):
            assert bool(((a == c) | (a.isnan() & c.isnan())).all()) and (not softplus or torch.equal(a, c))
    xd = x.masked_fill(late[..., None], value)
    for a, c in zip(cf.flare_causal_conv_prefill(xd, w, b, lengths=lengths), cf.flare_causal_conv_prefill(x, w, b, lengths=lengths)):
        assert torch.equal(a, c)


def layouts(v):
    """The same values behind other strides and alignments."""
    wide = torch.zeros(*v.shape[:-1], 3 * v.shape[-1] + 5, device=v.device, dtype=v.dtype)
    wide[..., 3:3 + v.shape[-1]] = v
    yield wide[..., 3:3 + v.shape[-1]]
    yield v.transpose(0, 1).contiguous().transpose(0, 1)
    yield v.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_inputs(dtype):
    g = gen(12)
    B, N, C = 2, 45, 48
    x, w, b, dy = randn(g, B, N, C, dtype=dtype), randn(g, C, 4), randn(g, C), randn(g, B, N, C, dtype=dtype)
    t = scan_inputs(g, B, N, C, 16, 2, dtype)

    def conv(x, dy):
        x = x.detach().requires_grad_()
        y = cf.flare_causal_conv(x, w, b, activation="silu")
        return y, *torch.autograd.grad(y, x, dy)

    def scan(t, dy):
        t = {k: v.detach().requires_grad_() for k, v in t.items()}
        y = cf.flare_selective_scan(**t, dt_softplus=True)
        return y, *torch.autograd.grad(y, list(t.values()), dy)

    first, second = conv(x, dy), scan(t, dy)
    for i in range(3):
        for a, c in zip(conv(list(layouts(x))[i], list(layouts(dy))[i]), first):
            assert torch.equal(a, c)
        moved = {k: (list(layouts(v))[i] if k not in ("D", "dt_bias") else v) for k, v in t.items()}
        for a, c in zip(scan(moved, list(layouts(dy))[i]), second):
            assert torch.equal(a, c)
    # one gradient row for all tokens (the gradient of a sum)
    same = dy[:1, :1].expand(B, N, C)
    for a, c in zip(conv(x, same), conv(x, same.contiguous())):
        assert torch.equal(a, c)
    for a, c in zip(scan(t, same), scan(t, same.contiguous())):
        assert torch.equal(a, c)


def test_weights_at_odd_addresses():
    g = gen(14)
    t = scan_inputs(g, 2, 40, 24, 16, 1, torch.float32)
    w, b = randn(g, 24, 4), randn(g, 24)

    def shifted(v):
        s = torch.zeros(v.numel() + 1, device="cuda", dtype=v.dtype)
        s[1:] = v.flatten()
        return s[1:].view(v.shape)

    moved = {k: (shifted(v) if k in ("A", "D", "dt_bias") else v) for k, v in t.items()}
    assert torch.equal(cf.flare_selective_scan(**moved, dt_softplus=True), cf.flare_selective_scan(**t, dt_softplus=True))
    one = lambda t: {k: (v[:, 0] if k in ("x", "dt", "z", "B", "C") else v) for k, v in t.items()}  # noqa: E731
    for a, c in zip(cf.flare_selective_scan_decode(**one(moved), dt_softplus=True), cf.flare_selective_scan_decode(**one(t), dt_softplus=True)):
        assert torch.equal(a, c)
    assert torch.equal(cf.flare_causal_conv(t["x"], shifted(w), shifted(b)), cf.flare_causal_conv(t["x"], w, b))


def test_same_bits_on_another_stream_and_from_a_graph():
    g = gen(13)
    t = scan_inputs(g, 1, 600, 64, 16, 1, torch.bfloat16)
    for v in t.values():
        v.requires_grad_()
    w, b = randn(g, 64, 4).requires_grad_(), randn(g, 64).requires_grad_()
    dy = randn(g, 1, 600, 64, dtype=torch.bfloat16)

    def step():
        u = cf.flare_causal_conv(t["x"], w, b, activation="silu")
        y = cf.flare_selective_scan(**{**t, "x": u}, dt_softplus=True)
        return [y.detach(), *torch.autograd.grad(y, [w, b, *t.values()], dy)]  # (no eager graph of the leaves outlives the step)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    for v in third:
        v.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, c, d in zip(first, second, third):
        assert torch.equal(a, c) and torch.equal(a, d)


def test_no_tokens_and_no_gradient():
    x = torch.empty(2, 0, 16, device="cuda", requires_grad=True)
    w = torch.randn(16, 3, device="cuda", requires_grad=True)
    y = cf.flare_causal_conv(x, w)
    assert y.shape == (2, 0, 16)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert dx.shape == x.shape and not dw.any()
    t = scan_inputs(gen(1), 2, 0, 16, 8, 1, torch.float32)
    for v in t.values():
        v.requires_grad_()
    y = cf.flare_selective_scan(**t)
    assert all(not d.any() for d in torch.autograd.grad(y.sum(), list(t.values())))
    with torch.no_grad():
        assert not cf.flare_causal_conv(torch.randn(1, 4, 16, device="cuda"), w).requires_grad
