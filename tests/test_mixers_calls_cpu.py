"""CPU: calls of the mixers that their documentation allows, up to where they would need a GPU."""
import ctypes as C

import pytest

from causal_flare import _mixers
from test_state_space_cpu import conv_args, scan_args


@pytest.mark.parametrize("N", [0, -3, 64, 2 ** 31 - 1])
@pytest.mark.parametrize("call, args", [("flare_conv_decode", conv_args), ("flare_scan_decode", scan_args)])
def test_single_tokens_do_not_look_at_the_number_of_tokens(call, args, N):
    # (no state: a null pointer is what they complain about)
    assert getattr(_mixers.load(), call)(C.byref(args(N=N)), None) == 3
    assert getattr(_mixers.load(), call)(C.byref(args(N=N, B=0)), None) == 1
    assert getattr(_mixers.load(), call)(None, None) == 3
