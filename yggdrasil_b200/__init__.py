"""yggdrasil_b200: Yggdrasil's int8 streaming inference step on NVIDIA B200 (sm_100a).

The compute path is libygg_b200.so (hand-written CUDA behind a C-ABI, include/ygg_b200.h); this package is its
Python host side, shaped as the reference's inference API (``Yggdrasil.load(path, backend="b200")``).
"""
from .inference import B200Yggdrasil, Yggdrasil  # noqa: F401

__all__ = ["Yggdrasil", "B200Yggdrasil"]   # without the operators: `import *` would import torch and their binding

_OPERATORS = {"token_logprobs": "logprobs", "TokenLogprobs": "logprobs",
              "int8_linear": "linear", "quantize_rows": "linear", "QuantizedRows": "linear",
              "StateCache": "cache"}


def __getattr__(name):   # the operators import torch; the package itself does not
    if name in _OPERATORS:
        from importlib import import_module
        value = getattr(import_module("." + _OPERATORS[name], __name__), name)
        globals()[name] = value
        return value
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
