"""CPU: the oracle of the state-space mixers against numerical differences, argument checks and struct layouts."""
import ctypes as C

import pytest
import torch

import causal_flare as cf
from causal_flare import _mixers
from oracle import mixers_oracle as orc


def f64(*shape):
    return torch.randn(*shape, dtype=torch.float64, requires_grad=True)


def test_oracle_gradients_against_differences():
    torch.manual_seed(0)
    docs = torch.tensor([[0, 0, 0, 1, 1, -1], [2, 2, -1, -1, 3, 3]])
    assert torch.autograd.gradcheck(lambda x, w, b: orc.causal_conv(x, w, b, silu=True, documents=docs)[0], (f64(2, 6, 2), f64(2, 3), f64(2)))
    args = (f64(2, 6, 2), f64(2, 6, 2), f64(2, 2), f64(2, 6, 1, 2), f64(2, 6, 1, 2), f64(2), f64(2, 6, 2), f64(2))
    assert torch.autograd.gradcheck(lambda *a: orc.selective_scan(*a, softplus=True, documents=docs)[0], args)


def test_oracle_states_continue_a_sequence():
    torch.manual_seed(1)
    x, w = torch.randn(2, 9, 3, dtype=torch.float64), torch.randn(3, 4, dtype=torch.float64)
    whole, end = orc.causal_conv(x, w, silu=True)
    a, st = orc.causal_conv(x[:, :4], w, silu=True)
    b, st = orc.causal_conv(x[:, 4:], w, state=st, silu=True)
    assert torch.equal(torch.cat([a, b], 1), whole) and torch.equal(st, end)


def test_struct_layouts():
    lib = _mixers.load()
    for which, struct in enumerate(_mixers._STRUCTS):
        assert lib.flare_mixers_abi_sizeof(which) == C.sizeof(struct)
    assert lib.flare_mixers_abi_sizeof(99) == 0


def conv(**kw):
    a = dict(x=torch.randn(2, 5, 8), weight=torch.randn(8, 4), bias=torch.randn(8))
    a.update(kw)
    return cf.flare_causal_conv(**a)


def scan(**kw):
    a = dict(x=torch.randn(2, 5, 8), dt=torch.randn(2, 5, 8), A=-torch.rand(8, 16), B=torch.randn(2, 5, 16), C=torch.randn(2, 5, 16))
    a.update(kw)
    return cf.flare_selective_scan(**a)


@pytest.mark.parametrize("kw, match", [
    (dict(x=torch.randn(5, 8)), r"expects x \[B, N, C\]"),
    (dict(weight=torch.randn(7, 4)), "weight"),
    (dict(weight=torch.randn(8, 1)), "2 to 4 taps"),
    (dict(weight=torch.randn(8, 5)), "2 to 4 taps"),
    (dict(bias=torch.randn(4)), "bias"),
    (dict(bias=torch.randn(8).bfloat16()), "weight's type"),
    (dict(activation="relu"), "activation"),
    (dict(x=torch.randn(2, 5, 8).double()), "float32, bfloat16 and float16"),
])
def test_conv_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        conv(**kw)


def test_tensors_must_be_on_the_gpu():
    for call in (conv, scan):
        with pytest.raises(RuntimeError, match="requires CUDA tensors"):
            call()


@pytest.mark.parametrize("kw, match", [
    (dict(x=torch.randn(5, 8)), r"expects x \[B, N, C\]"),
    (dict(A=-torch.rand(8, 12)), "states per channel"),
    (dict(A=-torch.rand(4, 16)), r"A \[C, S\]"),
    (dict(A=-torch.rand(8, 16).bfloat16()), "float32"),
    (dict(dt=torch.randn(2, 4, 8)), "dt"),
    (dict(dt=torch.randn(2, 5, 8).half()), "inputs' type"),
    (dict(B=torch.randn(2, 5, 8)), "B and C"),
    (dict(B=torch.randn(2, 5, 3, 16), C=torch.randn(2, 5, 3, 16)), "groups of equal size"),
    (dict(B=torch.randn(2, 5, 2, 16)), "B and C"),
    (dict(z=torch.randn(2, 5, 4)), "z"),
    (dict(D=torch.randn(4)), "D"),
])
def test_scan_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        scan(**kw)


def test_states_and_ids_are_checked():
    x, w = torch.randn(2, 8), torch.randn(8, 4)
    with pytest.raises(ValueError, match=r"x \[B, C\] or \[B, 1, C\]"):
        cf.flare_causal_conv_decode(torch.randn(2, 3, 8), w)
    with pytest.raises(RuntimeError, match="requires CUDA tensors"):
        cf.flare_causal_conv_decode(x, w)
    with pytest.raises(ValueError, match="documents"):
        _mixers.whole_numbers("f", "documents", torch.zeros(2, 4, dtype=torch.int32), (2, 5))
    with pytest.raises(ValueError, match="integer type"):
        _mixers.whole_numbers("f", "documents", torch.zeros(2, 5), (2, 5))
    assert _mixers.whole_numbers("f", "lengths", torch.tensor([1, 2]), (2,)).dtype == torch.int32


def conv_args(**kw):
    a = _mixers.ConvArgs()
    a.x = a.weight = a.y = a.dy = a.dx = a.dweight = 0x1000  # never dereferenced: calls that are refused
    a.B, a.N, a.C, a.W = 2, 64, 32, 4
    a.dtype = a.weight_dtype = 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("call, kw, status", [
    ("flare_conv_forward", dict(N=0), 1), ("flare_conv_forward", dict(W=5), 2), ("flare_conv_forward", dict(x=None), 3),
    ("flare_conv_forward", dict(dtype=7), 5), ("flare_conv_forward", dict(activation=3), 6), ("flare_conv_forward", dict(y=None), 3),
    ("flare_conv_forward", dict(documents=0x1000, state_in=0x1000), 6), ("flare_conv_forward", dict(state_in=0x1000, state_out=0x1000), 3),
    ("flare_conv_backward", {}, 4), ("flare_conv_backward", dict(lengths=0x1000), 6), ("flare_conv_decode", {}, 3),
])
def test_conv_entry_points_refuse(call, kw, status):
    assert getattr(_mixers.load(), call)(C.byref(conv_args(**kw)), None) == status


def scan_args(**kw):
    a = _mixers.ScanArgs()
    for k in ("x", "dt", "b", "c", "A", "y"):
        setattr(a, k, 0x1000)
    a.B, a.N, a.C, a.S, a.G = 2, 64, 32, 16, 1
    a.dtype = 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("call, kw, status", [
    ("flare_scan_forward", dict(C=0), 1), ("flare_scan_forward", dict(G=3), 1), ("flare_scan_forward", dict(S=12), 2),
    ("flare_scan_forward", dict(A=None), 3), ("flare_scan_forward", dict(dtype=3), 5), ("flare_scan_forward", dict(state_in=0x1004), 3),
    ("flare_scan_forward", dict(documents=0x1000, state_out=0x1000), 6), ("flare_scan_forward", dict(N=4096), 4),
    ("flare_scan_backward", {}, 3), ("flare_scan_decode", {}, 3),
])
def test_scan_entry_points_refuse(call, kw, status):
    assert getattr(_mixers.load(), call)(C.byref(scan_args(**kw)), None) == status


def test_workspaces_of_long_rows_of_few_channels():
    lib = _mixers.load()
    assert lib.flare_scan_forward_workspace_bytes(C.byref(scan_args())) == 0
    assert lib.flare_scan_forward_workspace_bytes(C.byref(scan_args(N=4096))) > 0
    assert lib.flare_scan_keep_bytes(C.byref(scan_args())) == 2 * 2 * 32 * 16 * 4
