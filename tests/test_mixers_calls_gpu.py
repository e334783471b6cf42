"""gpu: calls of the mixers that their documentation allows: states at odd addresses, slopes that are parameters, batches
of many rows."""
import pytest
import torch

import causal_flare as cf
from causal_flare import _mixers
from test_mixers_host_gpu import Nothing, gen, randn

pytestmark = pytest.mark.gpu


def at_odd_address(t):
    flat = torch.zeros(t.numel() + 1, device="cuda", dtype=t.dtype)
    flat[1:] = t.flatten()
    return flat[1:].view(t.shape)


@pytest.mark.parametrize("native", [True, False])
def test_states_at_odd_addresses_are_updated_in_place(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_mixers, "_host", Nothing())
    g = gen(31)
    x, dt, bc, A = randn(g, 3, 40), randn(g, 3, 40), randn(g, 3, 16), -torch.rand(40, 16, generator=g, device="cuda")
    for state, call in ((randn(g, 3, 40, 16), lambda s: cf.flare_selective_scan_decode(x, dt, A, bc, bc, s, dt_softplus=True)),
                        (randn(g, 3, 2, 40), lambda s: cf.flare_causal_conv_decode(x, A[:, :3].contiguous(), None, s))):
        moved = at_odd_address(state)
        first = moved.data_ptr()
        version = moved._version
        for _ in range(2):  # (a state that stays behind shows at the second token at the latest)
            want, state = call(state)
            y, same = call(moved)
            assert same is moved and moved.data_ptr() == first and torch.equal(y, want) and torch.equal(moved, state)
        assert moved._version > version


def test_a_captured_step_updates_a_state_at_an_odd_address():
    g = gen(32)
    x, dt, bc, A = randn(g, 2, 24), randn(g, 2, 24), randn(g, 2, 8), -torch.rand(24, 8, generator=g, device="cuda")
    state = randn(g, 2, 24, 8)
    moved = at_odd_address(state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = cf.flare_selective_scan_decode(x, dt, A, bc, bc, moved, dt_softplus=True)
    for _ in range(3):
        want, _ = cf.flare_selective_scan_decode(x, dt, A, bc, bc, state, dt_softplus=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(moved, state)


@pytest.mark.parametrize("native", [True, False])
def test_slopes_that_are_parameters(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_mixers, "_host", Nothing())
    g = gen(33)
    q, k = randn(g, 2, 9, 4, 64, dtype=torch.float16), randn(g, 2, 9, 2, 64, dtype=torch.float16)
    fixed = torch.rand(4, generator=g, device="cuda")
    slopes = fixed.clone().requires_grad_()

    def served(s):
        kc, vc = (torch.zeros(2, 20, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2))
        y = cf.flare_causal_attention_prefill(q, k, k, kc, vc, slopes=s)
        return y, cf.flare_causal_attention_decode(q[:, 0], k[:, 0], k[:, 0], kc, vc, torch.tensor([9, 3], device="cuda"), slopes=s)

    for a, b in zip(served(slopes), served(fixed)):
        assert torch.equal(a, b) and not a.requires_grad
    with torch.no_grad():
        assert torch.equal(cf.flare_causal_attention(q, k, k, slopes=slopes), cf.flare_causal_attention(q, k, k, slopes=fixed))
    with pytest.raises(ValueError, match="no gradient of the slopes"):
        cf.flare_causal_attention(q, k, k, slopes=slopes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_more_rows_than_a_grids_second_dimension_holds(dtype):
    # what the forward takes the backward takes too; every row is its own, so the last ones are those of a small batch
    B, N, H, J, D = 65_539, 3, 2, 1, 8
    g = gen(34)
    q, k, v, dy = (randn(g, B, N, h, D, dtype=dtype) for h in (H, J, J, H))

    def run(rows):
        leaves = [t[rows].detach().requires_grad_() for t in (q, k, v)]
        y = cf.flare_causal_attention(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy[rows])]

    for rows in (slice(0, 5), slice(65_530, B)):
        for a, b in zip(run(slice(0, B)), run(rows)):
            assert torch.equal(a[rows], b)
