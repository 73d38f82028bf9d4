"""What the channel-last operators share on the host: the compiled module
``_operators.so`` (``csrc/torch/operators.cpp``), which checks arguments,
allocates and calls the C ABI for autograd, and the activations' names.

Like the kernels' library it is loaded from this package only; there is no
fallback. Build both with ``python -m dynamicconvolutionoperator_b200._build``.
"""

from __future__ import annotations

import importlib

import torch

from . import _gradbuf, _lib

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}

_module = None


def activation_code(activation: str | None) -> int:
    try:
        return ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {sorted(k for k in ACTIVATIONS if k)} or "
                         f"None, got {activation!r}") from None


def _grad_buffer(param: torch.Tensor) -> torch.Tensor | None:
    view = _gradbuf.take_view(param)
    return None if view is None else view.view(param.shape)


def operators():
    """The compiled module (loaded once)."""
    global _module
    if _module is None:
        _lib.load()
        try:
            module = importlib.import_module("._operators", __package__)
        except ImportError as e:
            raise RuntimeError(
                "_operators.so is not built or does not load; run "
                f"`python -m dynamicconvolutionoperator_b200._build` ({e})") from e
        _gradbuf.observe(lambda attached: module.set_grad_buffer(_grad_buffer if attached else None))
        _module = module
    return _module


__all__ = ["ACTIVATIONS", "activation_code", "operators"]
