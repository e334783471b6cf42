"""Causal FLARE attention for NVIDIA B200: drop-in for the `causal_flare` operator API.

Same function names, argument shapes, return values and autograd behaviour as the Triton package
it replaces; the work is done by hand-written sm_100a CUDA kernels in libflare_b200.so, reached
through a C ABI.  There is no Triton, no alternative backend and no CPU fallback.
"""

from . import autoregressive, semi_autoregressive
from .autoregressive.training import flare_autoregressive_triton
from .autoregressive.inference import (
    flare_autoregressive_decode_triton,
    flare_autoregressive_prefill_triton,
)
from .autoregressive.recurrent import flare_recurrent_triton
from .semi_autoregressive.training import flare_semi_autoregressive_trition
from .semi_autoregressive.inference import (
    flare_semi_autoregressive_decode_trition,
    flare_semi_autoregressive_prefill_trition,
)
from .attention import flare_causal_attention, flare_causal_attention_decode, flare_causal_attention_prefill
from .state_space import (
    flare_causal_conv,
    flare_causal_conv_decode,
    flare_causal_conv_prefill,
    flare_selective_scan,
    flare_selective_scan_decode,
    flare_selective_scan_prefill,
)

__version__ = "0.0.1"

__all__ = [
    "autoregressive",
    "semi_autoregressive",
    "flare_autoregressive_triton",
    "flare_autoregressive_decode_triton",
    "flare_autoregressive_prefill_triton",
    "flare_causal_attention",
    "flare_causal_attention_decode",
    "flare_causal_attention_prefill",
    "flare_causal_conv",
    "flare_causal_conv_decode",
    "flare_causal_conv_prefill",
    "flare_recurrent_triton",
    "flare_selective_scan",
    "flare_selective_scan_decode",
    "flare_selective_scan_prefill",
    "flare_semi_autoregressive_decode_trition",
    "flare_semi_autoregressive_prefill_trition",
    "flare_semi_autoregressive_trition",
    "__version__",
]
