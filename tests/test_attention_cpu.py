"""CPU: the attention oracle against automatic differentiation, argument checks, refusals of the C entry points."""
import ctypes as C

import pytest
import torch

import causal_flare as cf
from causal_flare import _mixers
from oracle import mixers_oracle as orc


@pytest.mark.parametrize("cap, bias", [(None, False), (2.0, True)])
def test_oracle_gradients(cap, bias):
    torch.manual_seed(0)
    B, N, H, J, D = 2, 9, 4, 2, 8
    q, k, v, dy = (torch.randn(B, N, h, D, dtype=torch.float64) for h in (H, J, J, H))
    docs = torch.tensor([[0, 0, 0, 1, 1, 1, 1, -1, -1], [3, 3, -1, 3, 3, 3, 5, 5, 5]])
    prefix = torch.rand(B, N) < 0.7
    see = orc.in_sight(N, docs, prefix, 4)
    slopes = torch.rand(H, dtype=torch.float64) if bias else None
    o = orc.Attention(q, k, v, see, 0.3, cap, slopes, dy=dy)
    for t in (q, k, v):
        t.requires_grad_()
    y = orc.Attention(q, k, v, see, 0.3, cap, slopes).y
    for want, got in zip(torch.autograd.grad(y, (q, k, v), dy), (o.dq, o.dk, o.dv)):
        assert torch.allclose(want, got, atol=1e-12)
    assert not o.y[0, 7:].any() and not o.y[1, 2].any()


def test_who_sees_whom():
    docs = torch.tensor([[7, 7, 7, 7, -1, 7, 7, 2]])
    prefix = torch.tensor([[1, 1, 0, 1, 1, 1, 1, 1]], dtype=torch.bool)
    see = orc.in_sight(8, docs, prefix)[0].int().tolist()
    assert see == [
        [1, 1, 0, 0, 0, 0, 0, 0],
        [1, 1, 0, 0, 0, 0, 0, 0],
        [1, 1, 1, 0, 0, 0, 0, 0],
        [1, 1, 1, 1, 0, 0, 0, 0],
        [0, 0, 0, 0, 0, 0, 0, 0],
        [0, 0, 0, 0, 0, 1, 1, 0],
        [0, 0, 0, 0, 0, 1, 1, 0],
        [0, 0, 0, 0, 0, 0, 0, 1],
    ]


def call(fn=None, **kw):
    a = dict(q=torch.randn(2, 5, 4, 64).bfloat16(), k=torch.randn(2, 5, 2, 64).bfloat16(), v=torch.randn(2, 5, 2, 64).bfloat16())
    a.update(kw)
    return (fn or cf.flare_causal_attention)(**a)


@pytest.mark.parametrize("kw, match", [
    (dict(q=torch.randn(2, 4, 64).bfloat16()), r"\[B, N, heads, D\]"),
    (dict(k=torch.randn(2, 6, 2, 64).bfloat16()), "agree"),
    (dict(v=torch.randn(2, 5, 4, 64).bfloat16()), "agree"),
    (dict(q=torch.randn(2, 5, 3, 64).bfloat16()), "multiple of the key heads"),
    (dict(q=torch.randn(2, 5, 4, 64), k=torch.randn(2, 5, 2, 64), v=torch.randn(2, 5, 2, 64)), "bfloat16 and float16"),
    (dict(k=torch.randn(2, 5, 2, 64).half()), "inputs' type"),
    (dict(scale=0.0), "positive scale"), (dict(scale=float("nan")), "positive scale"),
    (dict(cap=2000.0), "caps up to 1024"), (dict(cap=-1.0), "positive cap"), (dict(cap=float("inf")), "positive cap"),
    (dict(window=0), "window"), (dict(window=2.5), "window"),
    (dict(slopes=torch.rand(3)), "slopes"), (dict(slopes=torch.rand(4).half()), "slopes"),
    (dict(slopes=torch.rand(4, requires_grad=True)), "no gradient of the slopes"),
])
def test_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


@pytest.mark.parametrize("D", [4, 60, 136, 256])
def test_head_widths(D):
    q, k = torch.randn(1, 3, 2, D).half(), torch.randn(1, 3, 2, D).half()
    with pytest.raises(ValueError, match="multiple of 8 up to 128"):
        cf.flare_causal_attention(q, k, k)


def test_tensors_must_be_on_the_gpu():
    with pytest.raises(RuntimeError, match="requires CUDA tensors"):
        call()


def test_masks_and_layouts():
    with pytest.raises(ValueError, match="torch.bool"):
        from causal_flare.attention import _truth
        _truth("f", torch.zeros(2, 5), (2, 5))
    t = torch.randn(2, 5, 4, 64).half()
    assert _mixers.tiled_layout(t) and _mixers.tiled_layout(t.transpose(1, 2))
    assert not _mixers.tiled_layout(t[:, :1].expand(2, 5, 4, 64)) and not _mixers.tiled_layout(t.transpose(2, 3))
    assert not _mixers.tiled_layout(t.flatten()[4:4 + 2 * 4 * 4 * 64].view(2, 4, 4, 64))


def args(**kw):
    a = _mixers.AttentionArgs()
    for name in ("q", "k", "v", "y", "lse", "dy", "dq", "dk", "dv"):
        setattr(a, name, 0x1000)
    a.B, a.Nq, a.Nk, a.H, a.J, a.D = 2, 64, 64, 4, 2, 64
    for name in ("q", "k", "v", "dy"):
        setattr(a, name + "_stride_b", 64 * 256), setattr(a, name + "_stride_n", 256), setattr(a, name + "_stride_h", 64)
    a.scale, a.dtype = 0.125, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("call_, kw, status", [
    ("forward", dict(H=3), 1), ("forward", dict(D=68), 2), ("forward", dict(D=192), 2), ("forward", dict(dtype=0), 5), ("forward", dict(scale=-1.0), 6),
    ("forward", dict(cap=float("nan")), 6), ("forward", dict(cap=1025.0), 6), ("forward", dict(cap=1e-40), 6), ("forward", dict(scale=float("inf")), 6), ("forward", dict(window=-1), 6), ("forward", dict(Nk=65), 6), ("forward", dict(cached=0x1000, documents=0x1000), 6),
    ("forward", dict(q=0x1008), 3), ("forward", dict(k_stride_n=260), 3), ("forward", {}, 4), ("backward", dict(cached=0x1000, Nk=100), 6),
    ("forward", dict(plan=0x1010), 3), ("backward", dict(dy=None), 3), ("backward", dict(plan=0x1000), 4), ("backward", dict(lse=None), 3), ("backward", {}, 4),
])
def test_entry_points_refuse(call_, kw, status):
    assert getattr(_mixers.load(), "flare_attention_" + call_)(C.byref(args(**kw)), None) == status


def cache_args(**kw):
    a = _mixers.CacheArgs()
    for name in ("q", "new_k", "new_v", "k_cache", "v_cache", "y", "cached"):
        setattr(a, name, 0x1000)
    a.B, a.N, a.H, a.J, a.D, a.L = 2, 3, 4, 2, 64, 4096
    a.scale, a.dtype = 0.125, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("call_, kw, status", [
    ("decode", dict(H=3), 1), ("decode", dict(L=0), 1), ("decode", dict(D=12), 2), ("decode", dict(dtype=0), 5), ("decode", dict(k_cache=0x1004), 3),
    ("decode", dict(cached=None), 3), ("decode", dict(scale=0.0), 6), ("decode", {}, 4), ("append", dict(N=0), 1), ("append", dict(new_k_stride_h=4), 3),
])
def test_cache_entry_points_refuse(call_, kw, status):
    assert getattr(_mixers.load(), "flare_attention_" + call_)(C.byref(cache_args(**kw)), None) == status


def test_ids_and_positions_of_64_bits():
    big = 1 << 32
    ids = torch.tensor([[big, big, 2 * big, 2 * big, -big, 0, 1 << 31, -1]])
    assert _mixers.whole_numbers("f", "documents", ids, (1, 8)).tolist() == [[0, 0, 1, 1, -1, 3, 4, -1]]
    assert _mixers.whole_numbers("f", "documents", ids[:, :0], (1, 0)).shape == (1, 0)
    assert _mixers.whole_numbers("f", "cached", torch.tensor([big, 5, -big]), (3,)).tolist() == [2 ** 31 - 1, 5, -1]
