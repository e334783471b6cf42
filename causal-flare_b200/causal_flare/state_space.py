"""State-space token mixers: the short causal convolution and the selective scan behind it.

Whole sequences with gradients (``flare_causal_conv``, ``flare_selective_scan``), prompts on top of a carried state
(``*_prefill``) and single tokens that update it in place (``*_decode``): the same three forms as the FLARE operators.  No
counterpart in the operator API this package mirrors.

Packed training batches: ``documents`` [B, N] holds an id per token.  A document is a run of equal ids; neither the taps of
the convolution nor the state of the scan cross its borders.  A negative id marks padding: output and gradients 0.
Padded prompts: ``lengths`` [B] says how many of a row's N tokens there are; the rest is padding, and the returned state is the
one behind the last token."""

from __future__ import annotations

import ctypes as C

import torch
from torch import autograd
from torch.autograd.function import once_differentiable

from . import _lib, _mixers
from ._mixers import has_shape, on_gpu, rows, same_device, same_dtype, whole_numbers

STATE_SIZES = (8, 16, 32)


# ---- short causal convolution ------------------------------------------------------------------------------------------


def _conv_args(name, x, weight, bias, activation, tokens):
    """Checks of what the three forms share.  ``tokens``: x is [B, N, C], else [B, C]."""
    if x.dim() != (3 if tokens else 2):
        raise ValueError(f"{name} expects x {'[B, N, C]' if tokens else '[B, C] or [B, 1, C]'}. Got {list(x.shape)}.")
    channels = x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] != channels:
        raise ValueError(f"{name} expects weight [C, W] with C={channels}. Got {list(weight.shape)}.")
    if not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"{name} supports filters of 2 to 4 taps. Got {weight.shape[1]}.")
    has_shape(name, "bias", bias, (channels,))
    code = _mixers.activation_code(name, activation)
    _lib.dtype_code(x.dtype)
    _lib.dtype_code(weight.dtype)
    if bias is not None and bias.dtype != weight.dtype:
        raise ValueError(f"{name} expects bias in the weight's type {weight.dtype}. Got {bias.dtype}.")
    on_gpu(name, x)
    same_device(name, x, weight=weight, bias=bias)
    return code


def _fill_conv(x, weight, bias, code, documents=None, lengths=None):
    a = _mixers.ConvArgs()
    a.x, a.weight, a.bias = x.data_ptr(), weight.data_ptr(), _lib.ptr(bias)
    a.documents, a.lengths = _lib.ptr(documents), _lib.ptr(lengths)
    a.B, a.C, a.W = x.shape[0], x.shape[-1], weight.shape[1]
    a.N = x.shape[1] if x.dim() == 3 else 1
    a.x_stride_b, a.x_stride_n = x.stride(0), x.stride(1) if x.dim() == 3 else 0
    a.dtype, a.weight_dtype, a.activation = _lib.dtype_code(x.dtype), _lib.dtype_code(weight.dtype), code
    return a


class CausalConv(autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, code, documents):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, documents)
        ctx.code = code
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        if x.numel():
            x, weight = rows(x), weight.contiguous()
            bias = None if bias is None else bias.contiguous()
            a = _fill_conv(x, weight, bias, code, documents)
            a.y = y.data_ptr()
            _mixers.run("flare_conv_forward", a, x.device)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if dy is None:
            return (None,) * 5
        x, weight, bias, documents = ctx.saved_tensors
        new = torch.empty if x.numel() else torch.zeros
        dx = new(x.shape, device=x.device, dtype=x.dtype)
        dw = new(weight.shape, device=x.device, dtype=weight.dtype)
        db = None if bias is None else new(bias.shape, device=x.device, dtype=bias.dtype)
        if x.numel():
            x, dy, weight = rows(x), rows(dy), weight.contiguous()
            bias = None if bias is None else bias.contiguous()
            a = _fill_conv(x, weight, bias, ctx.code, documents)
            a.dy, a.dy_stride_b, a.dy_stride_n = dy.data_ptr(), dy.stride(0), dy.stride(1)
            a.dx, a.dweight, a.dbias = dx.data_ptr(), dw.data_ptr(), _lib.ptr(db)
            _mixers.run("flare_conv_backward", a, x.device, "flare_conv_backward_workspace_bytes")
        return dx, dw, db, None, None


def flare_causal_conv(x, weight, bias=None, *, activation=None, documents=None):
    """Causal convolution along the tokens, one filter per channel (differentiable).

    x [B, N, C]; weight [C, W] of 2 to 4 taps, the last one for the token itself; bias [C] in the weight's type.
    ``activation``: None or "silu".  Returns y [B, N, C] in x's type; sums are in fp32, weight gradients in the weight's type."""
    if x.is_cuda:
        y = _mixers.host().conv(x, weight, bias, activation, documents)
        if y is not None:
            return y
    name = "flare_causal_conv"
    code = _conv_args(name, x, weight, bias, activation, True)
    documents = whole_numbers(name, "documents", documents, x.shape[:2])
    same_device(name, x, documents=documents)
    return CausalConv.apply(x, weight, bias, code, documents)


def flare_causal_conv_prefill(x, weight, bias=None, state=None, *, activation=None, lengths=None):
    """Tokens on top of a carried state [B, W - 1, C] (the inputs in front of them, oldest first; None: zeros).

    Returns ``(y [B, N, C], state)`` with a fresh state in x's type; not differentiable."""
    if x.is_cuda:
        out = _mixers.host().conv_prefill(x, weight, bias, state, activation, lengths)
        if out is not None:
            return out
    name = "flare_causal_conv_prefill"
    code = _conv_args(name, x, weight, bias, activation, True)
    B, N, channels = x.shape
    W = weight.shape[1]
    has_shape(name, "state", state, (B, W - 1, channels))
    same_dtype(name, x, state=state)
    lengths = whole_numbers(name, "lengths", lengths, (B,))
    same_device(name, x, state=state, lengths=lengths)
    y = torch.empty((B, N, channels), device=x.device, dtype=x.dtype)
    if not y.numel():
        return y, torch.zeros((B, W - 1, channels), device=x.device, dtype=x.dtype) if state is None else state.detach().clone()
    out = torch.empty((B, W - 1, channels), device=x.device, dtype=x.dtype)
    x, weight = rows(x), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    a = _fill_conv(x, weight, bias, code, lengths=lengths)
    state = None if state is None else state.contiguous()
    a.state_in, a.state_out, a.y = _lib.ptr(state), out.data_ptr(), y.data_ptr()
    _mixers.run("flare_conv_forward", a, x.device)
    return y, out


def flare_causal_conv_decode(x, weight, bias=None, state=None, *, activation=None):
    """One token: x [B, C] or [B, 1, C].  Returns ``(y in x's shape, state)``.

    The state is updated IN PLACE when it is contiguous (the returned one is then the same tensor); not differentiable."""
    if x.is_cuda:
        out = _mixers.host().conv_decode(x, weight, bias, state, activation)
        if out is not None:
            return out
    name = "flare_causal_conv_decode"
    shape = x.shape
    if x.dim() == 3 and x.shape[1] == 1:
        x = x[:, 0]
    code = _conv_args(name, x, weight, bias, activation, False)
    B, channels = x.shape
    W = weight.shape[1]
    has_shape(name, "state", state, (B, W - 1, channels))
    same_dtype(name, x, state=state)
    same_device(name, x, state=state)
    given, state = state, torch.zeros((B, W - 1, channels), device=x.device, dtype=x.dtype) if state is None else state.detach().contiguous()
    y = torch.empty(shape, device=x.device, dtype=x.dtype)
    if y.numel():
        x, weight = rows(x), weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        a = _fill_conv(x, weight, bias, code)
        a.state_out, a.y = state.data_ptr(), y.data_ptr()
        _mixers.run("flare_conv_decode", a, x.device)
        _mixers.written(state)
    return y, state if given is None or not given.is_contiguous() else given


# ---- selective scan ----------------------------------------------------------------------------------------------------


def _scan_args(name, x, dt, A, B, C_, D, z, dt_bias, tokens):
    """Checks of what the three forms share; returns the projections as [B, N, G, S] (tokens) or [B, G, S]."""
    lead = x.shape[:-1]
    if x.dim() != (3 if tokens else 2):
        raise ValueError(f"{name} expects x {'[B, N, C]' if tokens else '[B, C] or [B, 1, C]'}. Got {list(x.shape)}.")
    channels = x.shape[-1]
    if A.dim() != 2 or A.shape[0] != channels:
        raise ValueError(f"{name} expects A [C, S] with C={channels}. Got {list(A.shape)}.")
    S = A.shape[1]
    if S not in STATE_SIZES:
        raise ValueError(f"{name} supports {STATE_SIZES} states per channel. Got {S}.")
    has_shape(name, "dt", dt, x.shape)
    has_shape(name, "z", z, x.shape)
    has_shape(name, "D", D, (channels,))
    has_shape(name, "dt_bias", dt_bias, (channels,))
    if B.dim() == len(lead) + 1:
        B = B.unsqueeze(-2)
    if C_.dim() == len(lead) + 1:
        C_ = C_.unsqueeze(-2)
    if B.dim() != len(lead) + 2 or B.shape[:-2] != lead or B.shape[-1] != S or B.shape != C_.shape:
        raise ValueError(f"{name} expects B and C {list(lead)} + [S] or [G, S] with S={S}. Got {list(B.shape)} and {list(C_.shape)}.")
    G = B.shape[-2]
    if G < 1 or channels % G:
        raise ValueError(f"{name} expects the {channels} channels in groups of equal size. Got G={G}.")
    same_dtype(name, x, dt=dt, B=B, C=C_, z=z)
    for what, t in (("A", A), ("D", D), ("dt_bias", dt_bias)):
        if t is not None and t.dtype != torch.float32:
            raise ValueError(f"{name} expects {what} in torch.float32. Got {t.dtype}.")
    on_gpu(name, x)
    same_device(name, x, dt=dt, A=A, B=B, C=C_, D=D, z=z, dt_bias=dt_bias)
    return B, C_


def _fill_scan(x, dt, A, B, C_, D, z, dt_bias, softplus, documents=None, lengths=None):
    """Argument struct and the (possibly copied) tensors it points to."""
    a = _mixers.ScanArgs()
    held = []

    def put(name, t, axes):
        t = rows(t)
        held.append(t)
        setattr(a, name, t.data_ptr())
        for i, axis in enumerate(axes):
            if axis:
                setattr(a, f"{name}_stride_{axis}", t.stride(i))

    tokens = x.dim() == 3
    bn, bng = ("bn", "bng") if tokens else ("b", "bg")
    put("x", x, bn)
    put("dt", dt, bn)
    if z is not None:
        put("z", z, bn)
    put("b", B, bng)
    put("c", C_, bng)
    for name, t in (("A", A), ("D", D), ("dt_bias", dt_bias)):
        if t is not None:
            t = t.contiguous()
            if name == "A" and t.data_ptr() % 16:
                t = t.clone()
            held.append(t)
            setattr(a, name, t.data_ptr())
    a.documents, a.lengths = _lib.ptr(documents), _lib.ptr(lengths)
    a.B, a.N, a.C, a.S, a.G = x.shape[0], x.shape[1] if tokens else 1, x.shape[-1], A.shape[1], B.shape[-2]
    a.dtype, a.dt_softplus = _lib.dtype_code(x.dtype), int(bool(softplus))
    return a, held


class SelectiveScan(autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C_, D, z, dt_bias, softplus, documents):
        ctx.set_materialize_grads(False)
        ctx.softplus = softplus
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        keep = None
        if x.numel():
            a, held = _fill_scan(x, dt, A, B, C_, D, z, dt_bias, softplus, documents)
            a.y = y.data_ptr()
            if any(ctx.needs_input_grad):
                keep = torch.empty(_mixers.load().flare_scan_keep_bytes(C.byref(a)) // 4, device=x.device, dtype=torch.float32)
                a.keep = keep.data_ptr()
            _mixers.run("flare_scan_forward", a, x.device, "flare_scan_forward_workspace_bytes")
        ctx.save_for_backward(x, dt, A, B, C_, D, z, dt_bias, documents, keep)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if dy is None:
            return (None,) * 10
        x, dt, A, B, C_, D, z, dt_bias, documents, keep = ctx.saved_tensors
        new = torch.empty if x.numel() else torch.zeros
        grads = [None if t is None else new(t.shape, device=t.device, dtype=t.dtype) for t in (x, dt, A, B, C_, D, z, dt_bias)]
        if x.numel():
            a, held = _fill_scan(x, dt, A, B, C_, D, z, dt_bias, ctx.softplus, documents)
            dy = rows(dy)
            a.dy, a.dy_stride_b, a.dy_stride_n = dy.data_ptr(), dy.stride(0), dy.stride(1)
            a.keep = keep.data_ptr()
            a.dx, a.ddt, a.dA, a.db, a.dc, a.dD, a.dz, a.ddt_bias = (_lib.ptr(t) for t in grads)
            _mixers.run("flare_scan_backward", a, x.device, "flare_scan_backward_workspace_bytes")
        return (*grads, None, None)


def flare_selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, *, dt_softplus=False, documents=None):
    """Selective state space scan (differentiable):

        delta = dt + dt_bias, through softplus with ``dt_softplus``
        h[t] = exp(delta A) h[t-1] + delta B[t] x[t],    y[t] = (<C[t], h[t]> + D x[t]) silu(z[t])

    x, dt, z [B, N, C]; A [C, S] with S of 8, 16 or 32; B, C [B, N, S], or [B, N, G, S] for G groups of channels; D, dt_bias
    [C].  A, D and dt_bias are fp32, the others share one type, which y [B, N, C] has too.  States and sums are in fp32."""
    if x.is_cuda:
        y = _mixers.host().scan(x, dt, A, B, C, D, z, dt_bias, bool(dt_softplus), documents)
        if y is not None:
            return y
    name = "flare_selective_scan"
    B, C = _scan_args(name, x, dt, A, B, C, D, z, dt_bias, True)
    documents = whole_numbers(name, "documents", documents, x.shape[:2])
    same_device(name, x, documents=documents)
    return SelectiveScan.apply(x, dt, A, B, C, D, z, dt_bias, bool(dt_softplus), documents)


def _scan_state(name, x, state, S):
    shape = (x.shape[0], x.shape[-1], S)
    has_shape(name, "state", state, shape)
    if state is not None and state.dtype != torch.float32:
        raise ValueError(f"{name} expects state in torch.float32. Got {state.dtype}.")
    same_device(name, x, state=state)
    if state is None:
        return torch.zeros(shape, device=x.device, dtype=torch.float32)
    state = state.detach()
    return state if state.is_contiguous() and state.data_ptr() % 16 == 0 else state.clone(memory_format=torch.contiguous_format)


def flare_selective_scan_prefill(x, dt, A, B, C, state=None, *, D=None, z=None, dt_bias=None, dt_softplus=False, lengths=None):
    """Tokens on top of a carried state [B, C, S] fp32 (None: zeros).

    Returns ``(y [B, N, C], state)`` with a fresh state; not differentiable."""
    if x.is_cuda:
        out = _mixers.host().scan_prefill(x, dt, A, B, C, state, D, z, dt_bias, bool(dt_softplus), lengths)
        if out is not None:
            return out
    name = "flare_selective_scan_prefill"
    B, C = _scan_args(name, x, dt, A, B, C, D, z, dt_bias, True)
    lengths = whole_numbers(name, "lengths", lengths, x.shape[:1])
    same_device(name, x, lengths=lengths)
    state = _scan_state(name, x, state, A.shape[1])
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    if not x.numel():
        return y, state.clone()
    out = torch.empty_like(state)
    a, held = _fill_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, lengths=lengths)
    a.state_in, a.state_out, a.y = state.data_ptr(), out.data_ptr(), y.data_ptr()
    _mixers.run("flare_scan_forward", a, x.device, "flare_scan_forward_workspace_bytes")
    return y, out


def flare_selective_scan_decode(x, dt, A, B, C, state=None, *, D=None, z=None, dt_bias=None, dt_softplus=False):
    """One token: x, dt, z [B, C] or [B, 1, C]; B, C [B, S], [B, G, S] or [B, 1, G, S] with the same extra dimension as x.

    Returns ``(y in x's shape, state)``.  The state is updated IN PLACE when it is contiguous (the returned one is then the
    same tensor; one whose address is no multiple of 16 bytes costs two copies); not differentiable."""
    if x.is_cuda:
        out = _mixers.host().scan_decode(x, dt, A, B, C, state, D, z, dt_bias, bool(dt_softplus))
        if out is not None:
            return out
    name = "flare_selective_scan_decode"
    shape = x.shape
    if x.dim() == 3 and x.shape[1] == 1:
        x, dt, B, C = (t[:, 0] if t.dim() >= 3 and t.shape[1] == 1 else t for t in (x, dt, B, C))
        z = z[:, 0] if z is not None and z.dim() == 3 and z.shape[1] == 1 else z
    B, C = _scan_args(name, x, dt, A, B, C, D, z, dt_bias, False)
    given, state = state, _scan_state(name, x, state, A.shape[1])
    y = torch.empty(shape, device=x.device, dtype=x.dtype)
    if x.numel():
        a, held = _fill_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus)
        a.state_out, a.y = state.data_ptr(), y.data_ptr()
        _mixers.run("flare_scan_decode", a, x.device)
        _mixers.written(state)
    if given is None or not given.is_contiguous():
        return y, state
    if given.data_ptr() != state.data_ptr():  # (at an address that the kernel does not take)
        with torch.inference_mode():
            given.copy_(state)
        _mixers.written(given)
    return y, given
