"""What the channel-last operators share on the host."""

from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _gradbuf
from ._kernels import _require_cuda

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def activation_code(activation: str | None) -> int:
    try:
        return ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {sorted(k for k in ACTIVATIONS if k)} or "
                         f"None, got {activation!r}") from None


def ptr(t: torch.Tensor | None) -> int | None:
    return t.data_ptr() if t is not None else None


def aligned(*pointers: int | None) -> bool:
    """Whether every address is on a 16-byte boundary."""
    bits = 0
    for p in pointers:
        bits |= p or 0
    return bits % 16 == 0


def param_grad(param: torch.Tensor) -> torch.Tensor:
    """Where the backward writes ``param``'s gradient (contiguous): an attached
    buffer, or a new tensor."""
    if _gradbuf.attached():
        return _gradbuf.grad_buffer(param, param.shape, param.dtype, param.device)
    return torch.empty_like(param, memory_format=torch.contiguous_format)


def on_one_device(x: torch.Tensor, *others: torch.Tensor | None) -> None:
    """Raise unless every tensor is on ``x``'s CUDA device."""
    if not x.is_cuda:
        _require_cuda(x)
    index = x.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            _require_cuda(x, t)


def workspace(nbytes: int, device: torch.device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def first_order(backward):
    """``once_differentiable`` (a second derivative raises), at no cost where
    the graph of the backward is not recorded."""
    recorded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


__all__ = ["ACTIVATIONS", "activation_code", "aligned", "first_order", "on_one_device",
           "param_grad", "ptr", "workspace"]
