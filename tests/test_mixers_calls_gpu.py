"""gpu: calls of the mixers that their documentation allows: states at odd addresses."""
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
