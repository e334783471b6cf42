"""CPU: calls of the mixers that their documentation allows, up to where they would need a GPU."""
import ctypes as C

import pytest
import torch

import causal_flare as cf
from causal_flare import _mixers
from test_state_space_cpu import conv_args, scan_args


@pytest.mark.parametrize("N", [0, -3, 64, 2 ** 31 - 1])
@pytest.mark.parametrize("call, args", [("flare_conv_decode", conv_args), ("flare_scan_decode", scan_args)])
def test_single_tokens_do_not_look_at_the_number_of_tokens(call, args, N):
    # (no state: a null pointer is what they complain about)
    assert getattr(_mixers.load(), call)(C.byref(args(N=N)), None) == 3
    assert getattr(_mixers.load(), call)(C.byref(args(N=N, B=0)), None) == 1
    assert getattr(_mixers.load(), call)(None, None) == 3


def test_slopes_that_are_parameters_serve_where_no_gradient_is_formed():
    q, k, slopes = torch.randn(2, 5, 4, 64).half(), torch.randn(2, 5, 2, 64).half(), torch.rand(4, requires_grad=True)
    cache = torch.zeros(2, 9, 2, 64).half()
    for call in (lambda: cf.flare_causal_attention_prefill(q, k, k, cache, cache, slopes=slopes),
                 lambda: cf.flare_causal_attention_decode(q[:, 0], k[:, 0], k[:, 0], cache, cache, torch.zeros(2, dtype=torch.int32), slopes=slopes)):
        with pytest.raises(RuntimeError, match="requires CUDA tensors"):  # (and nothing else is wrong with them)
            call()
    with torch.no_grad(), pytest.raises(RuntimeError, match="requires CUDA tensors"):
        cf.flare_causal_attention(q, k, k, slopes=slopes)
    with pytest.raises(ValueError, match="no gradient of the slopes"):
        cf.flare_causal_attention(q, k, k, slopes=slopes)
