"""B200 execution backend for KTIR (Kernel Tile IR) kernels.

Drop-in for the ktir-cpu interpreter's execution path: same
``KTIRInterpreter`` API, execution lowered onto hand-written sm_100a kernels
through the C ABI in include/ktir_b200.h (libktir_b200.so).  The serving
operators (kv_append, prompt_attention, paged_decode) are called on torch
tensors directly.
"""

from .interpreter import KTIRInterpreter
from .latency import HardwareConfig, LatencyCategory, LatencyReport
from .parser import KTIRParser, KTIRParserBase

__all__ = ["KTIRInterpreter", "KTIRParser", "KTIRParserBase", "HardwareConfig",
           "LatencyCategory", "LatencyReport"]

# imported by name: a star import would bring torch with it
_SERVING = ("check_status", "kv_append", "paged_decode", "prompt_attention", "rotary_table")


def __getattr__(name):
    # the serving operators import torch; the interpreter's host side does not
    if name in _SERVING:
        from . import serving
        return globals().setdefault(name, getattr(serving, name))
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def __dir__():
    return sorted({*globals(), *_SERVING})
