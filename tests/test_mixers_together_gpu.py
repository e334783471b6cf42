"""gpu: the token mixers together, as layers of a decoder.  Training on packed documents: convolution, scan and attention behind one another,
gradients of everything.  Serving: a convolution, a scan, a FLARE and an attention layer take a batch of prompts of different
lengths, then tokens one by one, and say what they say of the whole sequences.

Tolerance: every layer's inputs, outputs and gradients are rounded to bf16 (half a step: 2^-8 of a norm at most), the layers here pass
an error on at most doubled (projections with orthonormal rows; softmax averages; factors of at most 1 in the scan, a filter
of taps whose magnitudes add up to about 2): 2 * 2^-8 for each of the roundings on the way."""
import pytest
import torch

import causal_flare as cf
from oracle import mixers_oracle as orc

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def orthonormal(g, n, m):
    return torch.linalg.qr(torch.randn(n, n, generator=g, device="cuda"))[0][:, :m].contiguous()


def rel(a, b):
    return float((a.detach().double() - b.double()).norm() / b.double().norm())


class Layers:
    """C channels: a convolution, a scan with 16 states, attention with H heads over J."""

    def __init__(self, g, C=128, H=4, J=2):
        self.C, self.H, self.J, self.D = C, H, J, C // H
        self.filter, self.fbias = randn(g, C, 4) * 0.5, randn(g, C) * 0.1
        self.A, self.skip, self.dt_bias = -torch.exp(randn(g, C, 16) * 0.5), torch.ones(C, device="cuda"), randn(g, C) * 0.5 - 2
        self.to_dt, self.to_bc, self.to_z = orthonormal(g, C, C), orthonormal(g, C, 32), orthonormal(g, C, C)
        self.to_qkv = torch.cat([orthonormal(g, C, C), orthonormal(g, C, 2 * J * self.D)], 1)
        self.weights = [self.filter, self.fbias, self.A, self.skip, self.dt_bias, self.to_dt, self.to_bc, self.to_z, self.to_qkv]

    def scan_inputs(self, u, f):
        """What the scan takes: x, dt, A, B, C and the rest."""
        bc = f(u @ self.to_bc.to(u.dtype))
        return dict(x=u, dt=f(u @ self.to_dt.to(u.dtype)), A=self.A, B=bc[..., :16], C=bc[..., 16:], D=self.skip, z=f(u @ self.to_z.to(u.dtype)), dt_bias=self.dt_bias)

    def heads(self, s):
        qkv = (s @ self.to_qkv.to(s.dtype)).unflatten(-1, (self.H + 2 * self.J, self.D))
        return qkv[..., :self.H, :], qkv[..., self.H:self.H + self.J, :], qkv[..., self.H + self.J:, :]


def test_training_on_packed_documents():
    g = torch.Generator(device="cuda").manual_seed(0)
    B, N = 2, 300
    net = Layers(g)
    x = randn(g, B, N, net.C, dtype=BF)
    documents = (torch.rand(B, N, generator=g, device="cuda") < 0.03).int().cumsum(1)
    documents[:, 270:] = -1
    dy = randn(g, B, N, net.H, net.D, dtype=BF)
    leaves = [x, *net.weights]
    for t in leaves:
        t.requires_grad_()
    u = cf.flare_causal_conv(x, net.filter, net.fbias, activation="silu", documents=documents)
    s = cf.flare_selective_scan(**net.scan_inputs(u, lambda t: t), dt_softplus=True, documents=documents)
    y = cf.flare_causal_attention(*net.heads(s), cap=20.0, documents=documents)
    grads = torch.autograd.grad(y, leaves, dy)

    exact = Layers.__new__(Layers)
    exact.__dict__.update(net.__dict__)
    ex = [t.detach().double().requires_grad_() for t in leaves]
    exact.filter, exact.fbias, exact.A, exact.skip, exact.dt_bias, exact.to_dt, exact.to_bc, exact.to_z, exact.to_qkv = ex[1:]
    u = orc.causal_conv(ex[0], exact.filter, exact.fbias, silu=True, documents=documents)[0]
    t = exact.scan_inputs(u, lambda t: t)
    t["B"], t["C"] = t["B"].unsqueeze(2), t["C"].unsqueeze(2)
    s = orc.selective_scan(**t, softplus=True, documents=documents)[0]
    want = orc.Attention(*exact.heads(s), orc.in_sight(N, documents).cuda(), net.D ** -0.5, 20.0).y
    assert rel(y, want.detach()) <= 6 * 2 * 2.0 ** -8
    assert not y[:, 270:].any()
    for a, b in zip(grads, torch.autograd.grad(want, ex, dy.double())):
        assert a.shape == b.shape and rel(a, b) <= 12 * 2 * 2.0 ** -8


def test_serving_prompts_and_tokens():
    g = torch.Generator(device="cuda").manual_seed(1)
    B, N, M, L = 3, 90, 64, 128
    net = Layers(g)
    latents = randn(g, net.J, M, 2 * net.D, dtype=BF)  # FLARE heads of 64
    wide = orthonormal(g, net.C, net.C)
    x = randn(g, B, N, net.C, dtype=BF)
    lengths = torch.tensor([70, 1, 33], device="cuda", dtype=torch.int32)

    def flare_inputs(s):
        h = (s @ wide.to(BF)).unflatten(-1, (net.J, 2 * net.D))
        return h, h

    # all of every sequence at once
    u = cf.flare_causal_conv(x, net.filter, net.fbias, activation="silu")
    s = cf.flare_selective_scan(**net.scan_inputs(u, lambda t: t), dt_softplus=True)
    f, _ = cf.flare_autoregressive_prefill_triton(latents, *flare_inputs(s), scale=0.125)
    whole = cf.flare_causal_attention(*net.heads(f.flatten(-2)), window=40)

    # prompts of different lengths, padded on the right, then single tokens
    kc, vc = (torch.empty(B, L, net.J, net.D, device="cuda", dtype=BF) for _ in range(2))
    n = int(lengths.max())
    u, conv_state = cf.flare_causal_conv_prefill(x[:, :n], net.filter, net.fbias, activation="silu", lengths=lengths)
    s, scan_state = cf.flare_selective_scan_prefill(**net.scan_inputs(u, lambda t: t), dt_softplus=True, lengths=lengths)
    mask = torch.arange(n, device="cuda")[None] < lengths[:, None]
    f, flare_state = cf.flare_autoregressive_prefill_triton(latents, *flare_inputs(s), scale=0.125, attention_mask=mask)
    y = cf.flare_causal_attention_prefill(*net.heads(f.flatten(-2)), kc, vc, lengths=lengths, window=40)
    tol = 8 * 2 * 2.0 ** -8
    for b in range(B):
        assert rel(y[b, :lengths[b]], whole[b, :lengths[b]]) <= tol and not y[b, lengths[b]:].any()
    at = lengths.clone()
    for _ in range(N - n):
        token = x[torch.arange(B, device="cuda"), at.long()]
        u, conv_state = cf.flare_causal_conv_decode(token, net.filter, net.fbias, conv_state, activation="silu")
        s, scan_state = cf.flare_selective_scan_decode(**net.scan_inputs(u, lambda t: t), state=scan_state, dt_softplus=True)
        f, flare_state = cf.flare_autoregressive_decode_triton(latents, *flare_inputs(s), flare_state, scale=0.125)
        y = cf.flare_causal_attention_decode(*net.heads(f.flatten(-2)), kc, vc, at, window=40)
        assert rel(y[:, 0], whole[torch.arange(B, device="cuda"), at.long()]) <= tol
        at += 1
