"""Causal softmax attention over all tokens in sight, with capped scores, a bias on the distance, documents, prefixes and windows.

Whole sequences with gradients (``flare_causal_attention``), prompts into a key / value cache (``flare_causal_attention_prefill``) and
single tokens on it (``flare_causal_attention_decode``).  Tensors are [B, N, heads, D] as everywhere in this package; H query heads
share J key / value heads (head h reads h // (H // J)).  No counterpart in the operator API this package mirrors.

The score of the query at position i for the key at position j is ``cap * tanh(scale * <q, k> / cap) - slopes[h] * |i - j|`` (without
``cap``: ``scale * <q, k>``; a cap is at most 1024), and i sees the keys j <= i, subject to

* ``documents`` [B, N]: an id per token.  A document is a run of equal ids, and tokens see their own document only.  A negative id marks
  padding: it sees nothing and nobody sees it, output and gradients are 0.
* ``window``: only the keys j > i - window.
* ``prefix`` [B, N] truth values: the tokens with which a document begins and for which it holds are seen by all of the document.

A token that sees nothing, or none of whose scores is above -infinity, has output and gradients 0.  ``scale`` is D ** -0.5 unless it is given, but 1 for
heads that are 8 wide: the convention of all operators of this package (pass ``scale=8 ** -0.5`` for the usual one).
"""

from __future__ import annotations

import ctypes as C

import torch
from torch import autograd
from torch.autograd.function import once_differentiable

from . import _lib, _mixers
from ._common import _resolve_attn_scale
from ._mixers import has_shape, on_gpu, put_strides, same_device, same_dtype, tiled, whole_numbers


def _attention_args(name, q, k, v, scale, cap, slopes, window, tokens, differentiable=False):
    """Checks of what the three forms share; returns (scale, cap, window) as the kernels take them."""
    dims, layout = (4, "[B, N, heads, D]") if tokens else (3, "[B, heads, D] or [B, 1, heads, D]")
    if q.dim() != dims or k.dim() != dims or v.dim() != dims:
        raise ValueError(f"{name} expects q, k, v {layout}. Got {list(q.shape)}, {list(k.shape)}, {list(v.shape)}.")
    if k.shape != v.shape or q.shape[:-2] != k.shape[:-2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"{name} expects q, k, v to agree in all but the number of heads, k and v in that too. "
                         f"Got {list(q.shape)}, {list(k.shape)}, {list(v.shape)}.")
    H, J, D = q.shape[-2], k.shape[-2], q.shape[-1]
    if J < 1 or H < 1 or H % J:
        raise ValueError(f"{name} expects the query heads to be a multiple of the key heads. Got {H} and {J}.")
    if D < 8 or D % 8 or D > 128:
        raise ValueError(f"{name} supports heads of a multiple of 8 up to 128. Got D={D}.")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{name} supports bfloat16 and float16 inputs. Got {q.dtype}.")
    same_dtype(name, q, k=k, v=v)
    scale = _resolve_attn_scale(scale, D)
    if not (0.0 < scale < float("inf")):
        raise ValueError(f"{name} expects a positive scale. Got {scale}.")
    if cap is not None and not (0.0 < float(cap) < float("inf")):
        raise ValueError(f"{name} expects a positive cap. Got {cap}.")
    if cap is not None and float(cap) > 1024:
        raise ValueError(f"{name} supports caps up to 1024 (scores are off by up to cap * 2 ** -21). Got {cap}.")
    if window is not None and (int(window) != window or not 1 <= window):
        raise ValueError(f"{name} expects a window of at least one token. Got {window}.")
    has_shape(name, "slopes", slopes, (H,))
    if slopes is not None and slopes.dtype != torch.float32:
        raise ValueError(f"{name} expects slopes in torch.float32. Got {slopes.dtype}.")
    if differentiable and slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} forms no gradient of the slopes: pass them detached.")
    on_gpu(name, q)
    same_device(name, q, k=k, v=v, slopes=slopes)
    return scale, 0.0 if cap is None else float(cap), 0 if window is None else min(int(window), 2 ** 31 - 1)


def _truth(name, prefix, shape):
    if prefix is None:
        return None
    if prefix.dtype != torch.bool:
        raise ValueError(f"{name} expects prefix of type torch.bool. Got {prefix.dtype}.")
    has_shape(name, "prefix", prefix, shape)
    return prefix.contiguous()


def _fill(q, k, v, how, slopes, documents=None, prefix=None):
    a = _mixers.AttentionArgs()
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.documents, a.prefix, a.slopes = _lib.ptr(documents), _lib.ptr(prefix), _lib.ptr(slopes)
    a.B, a.Nq, a.H, a.D = q.shape
    a.Nk, a.J = k.shape[1], k.shape[2]
    for name, t in (("q", q), ("k", k), ("v", v)):
        put_strides(a, name, t, "bnh")
    a.scale, a.cap, a.window = how
    a.dtype = _lib.dtype_code(q.dtype)
    return a


class CausalAttention(autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, how, slopes, documents, prefix):
        ctx.set_materialize_grads(False)
        ctx.how = how
        B, N, H, D = q.shape
        y = torch.empty((B, N, H, D), device=q.device, dtype=q.dtype)
        lse = plan = None
        if y.numel():
            qt, kt, vt = tiled(q), tiled(k), tiled(v)
            a = _fill(qt, kt, vt, how, slopes, documents, prefix)
            a.y = y.data_ptr()
            if any(ctx.needs_input_grad):
                lse = torch.empty((B, H, (N + 127) // 128 * 128), device=q.device, dtype=torch.float32)
                plan = torch.empty(_mixers.load().flare_attention_plan_bytes(C.byref(a)), device=q.device, dtype=torch.uint8)
                a.lse, a.plan = lse.data_ptr(), plan.data_ptr()
            _mixers.run("flare_attention_forward", a, q.device, "flare_attention_forward_workspace_bytes")
        ctx.save_for_backward(q, k, v, y, lse, slopes, documents, prefix, plan)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if dy is None:
            return (None,) * 7
        q, k, v, y, lse, slopes, documents, prefix, plan = ctx.saved_tensors
        new = torch.empty if y.numel() else torch.zeros
        dq, dk, dv = (new(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
        if y.numel():
            qt, kt, vt, dyt = tiled(q), tiled(k), tiled(v), tiled(dy)
            a = _fill(qt, kt, vt, ctx.how, slopes, documents, prefix)
            a.y, a.lse, a.plan, a.dy = y.data_ptr(), lse.data_ptr(), plan.data_ptr(), dyt.data_ptr()
            put_strides(a, "dy", dyt, "bnh")
            a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
            _mixers.run("flare_attention_backward", a, q.device, "flare_attention_backward_workspace_bytes")
        return dq, dk, dv, None, None, None, None


def flare_causal_attention(q, k, v, *, scale=None, cap=None, slopes=None, window=None, documents=None, prefix=None):
    """Causal attention (differentiable in q, k, v).  q [B, N, H, D]; k, v [B, N, J, D], bf16 or fp16, D a multiple of 8 up to 128.

    ``scale`` (D ** -0.5, for D = 8 it is 1), ``cap``, ``slopes`` [H] fp32 (which get no gradient: while gradients are recorded they have to be
    detached), ``window``, ``documents`` and ``prefix`` as the module says.  Returns y [B, N, H, D].  Softmax statistics and sums are in fp32; its weights meet V in the inputs' type.  The gradients are the same bits
    in every call."""
    if q.is_cuda:
        y = _mixers.host().attention(q, k, v, scale, cap, slopes, window, documents, prefix)
        if y is not None:
            return y
    name = "flare_causal_attention"
    how = _attention_args(name, q, k, v, scale, cap, slopes, window, True, differentiable=True)
    documents = whole_numbers(name, "documents", documents, q.shape[:2])
    prefix = _truth(name, prefix, q.shape[:2])
    same_device(name, q, documents=documents, prefix=prefix)
    return CausalAttention.apply(q, k, v, how, None if slopes is None else slopes.contiguous(), documents, prefix)


def _check_caches(name, q, k, k_cache, v_cache):
    B, J, D = k.shape[0], k.shape[-2], k.shape[-1]
    for what, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.dim() != 4 or t.shape[0] != B or t.shape[2:] != (J, D) or t.shape[1] < 1:
            raise ValueError(f"{name} expects {what} [B, L, heads, D] with B={B}, {J} heads, D={D}. Got {list(t.shape)}.")
        if not _mixers.tiled_layout(t):
            raise ValueError(f"{name} writes {what} in place: its rows have to be contiguous, 16-byte aligned and apart.")
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"{name} expects caches of one shape. Got {list(k_cache.shape)} and {list(v_cache.shape)}.")
    same_dtype(name, q, k_cache=k_cache, v_cache=v_cache)
    same_device(name, q, k_cache=k_cache, v_cache=v_cache)


def _fill_cache(k, v, k_cache, v_cache, cached):
    a = _mixers.CacheArgs()
    a.new_k, a.new_v, a.k_cache, a.v_cache = k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    a.cached = _lib.ptr(cached)
    a.B, a.L, a.J, a.D = k_cache.shape
    axes = "bnh" if k.dim() == 4 else "bh"
    put_strides(a, "new_k", k, axes)
    put_strides(a, "new_v", v, axes)
    put_strides(a, "k", k_cache, "bnh")
    put_strides(a, "v", v_cache, "bnh")
    a.dtype = _lib.dtype_code(k.dtype)
    return a


def flare_causal_attention_prefill(q, k, v, k_cache, v_cache, *, cached=None, lengths=None, scale=None, cap=None, slopes=None, window=None,
                                   prefix=None):
    """N new tokens per row behind the ``cached`` [B] tokens that the caches [B, L, J, D] hold already (None: none).

    The new keys and values are written into the caches, at positions cached[b] and on, and the queries see them and everything in
    front.  ``lengths`` [B]: tokens of row b (None: N); what lies behind is padding: nothing is written for it and y is 0.  A token
    whose position lies outside the cache is treated the same way (a row whose ``cached`` does: all of it).  ``prefix`` marks tokens of
    the prompt's beginning that all new tokens see.  ``scale`` (D ** -0.5, for D = 8 it is 1) and the rest as the module says.  Returns y [B, N, H, D]; not
    differentiable."""
    if q.is_cuda:
        y = _mixers.host().attention_prefill(q, k, v, k_cache, v_cache, cached, lengths, scale, cap, slopes, window, prefix)
        if y is not None:
            return y
    name = "flare_causal_attention_prefill"
    how = _attention_args(name, q, k, v, scale, cap, slopes, window, True)
    _check_caches(name, q, k, k_cache, v_cache)
    B, N = q.shape[:2]
    cached = whole_numbers(name, "cached", cached, (B,))
    lengths = whole_numbers(name, "lengths", lengths, (B,))
    prefix = _truth(name, prefix, (B, N))
    same_device(name, q, cached=cached, lengths=lengths, prefix=prefix)
    y = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    if not y.numel():
        return y
    if cached is None:
        cached = torch.zeros(B, device=q.device, dtype=torch.int32)
    qt, kt, vt = tiled(q), tiled(k), tiled(v)
    c = _fill_cache(kt, vt, k_cache, v_cache, cached)
    c.N, c.lengths = N, _lib.ptr(lengths)
    _mixers.run("flare_attention_append", c, q.device)
    _mixers.written(k_cache, v_cache)
    slopes = None if slopes is None else slopes.contiguous()
    a = _fill(qt, k_cache, v_cache, how, slopes, prefix=prefix)
    a.cached, a.lengths, a.y = cached.data_ptr(), _lib.ptr(lengths), y.data_ptr()
    _mixers.run("flare_attention_forward", a, q.device, "flare_attention_forward_workspace_bytes")
    return y


def flare_causal_attention_decode(q, k, v, k_cache, v_cache, cached, *, scale=None, cap=None, slopes=None, window=None):
    """One token per row: q [B, H, D] or [B, 1, H, D]; k, v [B, J, D] or [B, 1, J, D].

    Its key and value are written to position cached[b] of the caches [B, L, J, D] and it sees them and the cached[b] in front; the
    caller counts ``cached`` up.  A row whose position lies outside the cache is idle: y is 0 and nothing is written (-1 for an empty
    slot of a batch).  ``scale`` (D ** -0.5, for D = 8 it is 1) and the rest as the module says.  Returns y in q's shape; not differentiable."""
    if q.is_cuda:
        y = _mixers.host().attention_decode(q, k, v, k_cache, v_cache, cached, scale, cap, slopes, window)
        if y is not None:
            return y
    name = "flare_causal_attention_decode"
    shape = q.shape
    q, k, v = (t[:, 0] if t.dim() == 4 and t.shape[1] == 1 else t for t in (q, k, v))
    how = _attention_args(name, q, k, v, scale, cap, slopes, window, False)
    _check_caches(name, q, k, k_cache, v_cache)
    if cached is None:
        raise ValueError(f"{name} expects cached [B].")
    cached = whole_numbers(name, "cached", cached, q.shape[:1])
    same_device(name, q, cached=cached)
    y = torch.empty(shape, device=q.device, dtype=q.dtype)
    if not y.numel():
        return y
    q, k, v = tiled(q), tiled(k), tiled(v)
    slopes = None if slopes is None else slopes.contiguous()
    a = _fill_cache(k, v, k_cache, v_cache, cached)
    a.q, a.y, a.slopes, a.H = q.data_ptr(), y.data_ptr(), _lib.ptr(slopes), q.shape[1]
    put_strides(a, "q", q, "bh")
    a.scale, a.cap, a.window = how
    _mixers.run("flare_attention_decode", a, q.device, "flare_attention_decode_workspace_bytes")
    _mixers.written(k_cache, v_cache)
    return y
