"""ctypes binding and argument checks of the causal token mixers beside FLARE (include/flare_b200_mixers.h)."""

from __future__ import annotations

import ctypes as C

import torch
from torch import autograd

from . import _lib

IDENTITY, SILU = 0, 1
_ACTIVATIONS = {None: IDENTITY, "silu": SILU}


class ConvArgs(C.Structure):
    _fields_ = [
        *((name, C.c_void_p) for name in ("x", "weight", "bias", "documents", "lengths", "state_in", "state_out", "y", "dy", "dx",
                                          "dweight", "dbias", "workspace")),
        ("workspace_bytes", C.c_size_t),
        *((name, C.c_int32) for name in ("B", "N", "C", "W")),
        *((name, C.c_int64) for name in ("x_stride_b", "x_stride_n", "dy_stride_b", "dy_stride_n")),
        *((name, C.c_int32) for name in ("dtype", "weight_dtype", "activation")),
    ]


class ScanArgs(C.Structure):
    _fields_ = [
        *((name, C.c_void_p) for name in ("x", "dt", "z", "b", "c", "A", "D", "dt_bias", "documents", "lengths", "state_in", "state_out", "y",
                                          "keep", "dy", "dx", "ddt", "dz", "db", "dc", "dA", "dD", "ddt_bias", "workspace")),
        ("workspace_bytes", C.c_size_t),
        *((name, C.c_int32) for name in ("B", "N", "C", "S", "G")),
        *((f"{name}_stride_{axis}", C.c_int64) for name, axes in (("x", "bn"), ("dt", "bn"), ("z", "bn"), ("b", "bng"), ("c", "bng"), ("dy", "bn"))
          for axis in axes),
        ("dtype", C.c_int32), ("dt_softplus", C.c_int32),
    ]


class AttentionArgs(C.Structure):
    _fields_ = [
        *((name, C.c_void_p) for name in ("q", "k", "v", "y", "lse", "plan", "documents", "prefix", "cached", "lengths", "slopes", "dy", "dq", "dk", "dv",
                                          "workspace")),
        ("workspace_bytes", C.c_size_t),
        *((name, C.c_int32) for name in ("B", "Nq", "Nk", "H", "J", "D")),
        *((f"{name}_stride_{axis}", C.c_int64) for name in ("q", "k", "v", "dy") for axis in "bnh"),
        ("scale", C.c_float), ("cap", C.c_float), ("window", C.c_int32), ("dtype", C.c_int32),
    ]


class CacheArgs(C.Structure):
    _fields_ = [
        *((name, C.c_void_p) for name in ("q", "new_k", "new_v", "k_cache", "v_cache", "y", "cached", "lengths", "slopes", "workspace")),
        ("workspace_bytes", C.c_size_t),
        *((name, C.c_int32) for name in ("B", "N", "H", "J", "D", "L")),
        ("q_stride_b", C.c_int64), ("q_stride_h", C.c_int64),
        *((f"{name}_stride_{axis}", C.c_int64) for name in ("new_k", "new_v", "k", "v") for axis in "bnh"),
        ("scale", C.c_float), ("cap", C.c_float), ("window", C.c_int32), ("dtype", C.c_int32),
    ]


_STRUCTS = (ConvArgs, ScanArgs, AttentionArgs, CacheArgs)
_CALLS = {"flare_conv_forward": ConvArgs, "flare_conv_backward": ConvArgs, "flare_conv_decode": ConvArgs,
          "flare_scan_forward": ScanArgs, "flare_scan_backward": ScanArgs, "flare_scan_decode": ScanArgs,
          "flare_attention_forward": AttentionArgs, "flare_attention_backward": AttentionArgs,
          "flare_attention_append": CacheArgs, "flare_attention_decode": CacheArgs}
_SIZES = {"flare_conv_backward_workspace_bytes": ConvArgs, "flare_scan_keep_bytes": ScanArgs,
          "flare_scan_forward_workspace_bytes": ScanArgs, "flare_scan_backward_workspace_bytes": ScanArgs,
          "flare_attention_plan_bytes": AttentionArgs, "flare_attention_forward_workspace_bytes": AttentionArgs, "flare_attention_backward_workspace_bytes": AttentionArgs,
          "flare_attention_decode_workspace_bytes": CacheArgs}

_bound = None


def load() -> C.CDLL:
    """The shared library with these entry points bound; raises if its structs differ from ours."""
    global _bound
    if _bound is None:
        lib = _lib.load()
        for name, struct in _CALLS.items():
            getattr(lib, name).restype, getattr(lib, name).argtypes = C.c_int, [C.POINTER(struct), C.c_void_p]
        for name, struct in _SIZES.items():
            getattr(lib, name).restype, getattr(lib, name).argtypes = C.c_size_t, [C.POINTER(struct)]
        lib.flare_mixers_abi_sizeof.restype, lib.flare_mixers_abi_sizeof.argtypes = C.c_size_t, [C.c_int]
        for which, struct in enumerate(_STRUCTS):
            if lib.flare_mixers_abi_sizeof(which) != C.sizeof(struct):
                raise RuntimeError(f"ABI mismatch for {struct.__name__}: library {lib.flare_mixers_abi_sizeof(which)} bytes, "
                                   f"binding {C.sizeof(struct)} bytes")
        _bound = lib
    return _bound


_host = None


def host():
    """The native host layer (mixers_ext.cpp), bound to the loaded library: serves the plain calls of the operators."""
    global _host
    if _host is None:
        lib = load()
        try:
            from . import _mixers_host as native
        except ImportError as e:
            raise RuntimeError(f"the native host layer is missing ({e}). Build it with `python causal-flare_b200/build.py`.") from e
        names = (*_CALLS, *_SIZES, "flare_mixers_abi_sizeof", "flare_status_string", "flare_last_cuda_error")
        native.bind({name: C.cast(getattr(lib, name), C.c_void_p).value for name in names})
        _host = native
    return _host


def run(name: str, args, device, workspace: str | None = None) -> None:
    """Launch an entry point on the device's current stream, with a workspace of what `workspace` (a size query) asks for."""
    lib = load()
    ws = None
    with torch.cuda.device(device):
        if workspace is not None:
            need = getattr(lib, workspace)(C.byref(args))
            if need:
                ws = torch.empty(need, dtype=torch.uint8, device=device)
                args.workspace, args.workspace_bytes = ws.data_ptr(), need
        _lib.check(getattr(lib, name)(C.byref(args), _lib.stream_handle(device)), name)
    # `ws` is stream-ordered torch memory: safe to release after the launches are enqueued.


# ---- argument checks -------------------------------------------------------------------------------------------------


def on_gpu(name: str, x: torch.Tensor) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{name} requires CUDA tensors.")


def same_device(name: str, x: torch.Tensor, **others) -> None:
    for what, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} expects {what} on {x.device}. Got {t.device}.")


def same_dtype(name: str, x: torch.Tensor, **others) -> None:
    _lib.dtype_code(x.dtype)
    for what, t in others.items():
        if t is not None and t.dtype != x.dtype:
            raise ValueError(f"{name} expects {what} in the inputs' type {x.dtype}. Got {t.dtype}.")


def has_shape(name: str, what: str, t, shape) -> None:
    if t is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} expects {what} {list(shape)}. Got {list(t.shape)}.")


def activation_code(name: str, activation) -> int:
    try:
        return _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"{name} supports activation=None and 'silu'. Got {activation!r}.") from None


def whole_numbers(name: str, what: str, t, shape):
    """Ids or lengths as the kernels read them: int32, contiguous (None stays None)."""
    if t is None:
        return None
    if t.dtype not in (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8):
        raise ValueError(f"{name} expects {what} of an integer type. Got {t.dtype}.")
    has_shape(name, what, t, shape)
    if t.dtype == torch.int64:
        t = _narrow_ids(t) if what == "documents" else t.clamp(-1, 2 ** 31 - 1)
    return t.to(torch.int32).contiguous()


def _narrow_ids(t):
    """Ids of 64 bits need not fit 32: documents are numbered anew, in the order of their runs."""
    new = torch.zeros(t.shape, dtype=torch.int32, device=t.device)
    torch.cumsum(t[:, 1:] != t[:, :-1], 1, dtype=torch.int32, out=new[:, 1:])
    return new.masked_fill_(t < 0, -1)


def written(*tensors) -> None:
    """What a kernel wrote in place has a new version: autograd notices graphs that hold the old one."""
    for t in tensors:
        if not t.is_inference():
            autograd.graph.increment_version(t)


def rows(t):
    """`t`, with its innermost dimension contiguous."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def tiled_layout(t) -> bool:
    """Can tiled copies fetch the rows of ``t`` where they are?  (16-byte aligned rows, none of them shared)"""
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
        size == 1 or (stride > 0 and stride % 8 == 0) for size, stride in zip(t.shape[:-1], t.stride()[:-1]))


def tiled(t):
    return t if tiled_layout(t) else t.clone(memory_format=torch.contiguous_format)


def put_strides(a, name: str, t, axes: str) -> None:
    for axis, size, stride in zip(axes, t.shape, t.stride()):
        setattr(a, f"{name}_stride_{axis}", stride if size > 1 else 0)
