"""Dropout from a counter-based generator (``ddpm_dropout`` in
``include/ddpm_b200.h``).

The mask is a function of the seed and of each value's position, so it is never
stored: the backward pass draws it again. There is no hidden generator state:
equal arguments give equal results, on every device and in every order.
"""

from __future__ import annotations

import torch

from . import _lib
from ._op import first_order, on_one_device, ptr

_U64 = (1 << 64) - 1


def _launch(x, residual, p, seed, offset):
    """``x`` (and ``residual``) contiguous; ``seed`` a number or a tensor."""
    out = torch.empty_like(x)
    number, held = (0, seed.data_ptr()) if isinstance(seed, torch.Tensor) else (seed, None)
    _lib.call_on(x.device, "ddpm_dropout", x.data_ptr(), ptr(residual), out.data_ptr(), x.numel(),
                 p, number, held, offset, _lib.dtype_code(x.dtype))
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        # a seed on the device is saved, so that writing to it before the
        # backward (which has to draw the same mask) raises
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)
            ctx.args = (p, None, offset)
        else:
            ctx.args = (p, seed, offset)
        return _launch(x, residual, p, seed, offset)

    @staticmethod
    @first_order
    def backward(ctx, grad_out):
        p, seed, offset = ctx.args
        gx = None
        if ctx.needs_input_grad[0]:
            if seed is None:
                seed, = ctx.saved_tensors
            gx = _launch(grad_out.contiguous(), None, p, seed, offset)
        return gx, grad_out if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int | torch.Tensor, offset: int = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """Zero each value of ``x`` with probability ``p``, scale the others by
    ``1 / (1 - p)`` and add ``residual``.

    The values are numbered in ``x``'s row-major order from ``offset`` on; value
    ``q`` is kept iff word ``q % 4`` of Philox-4x32-10 at counter ``q // 4``
    with key ``seed`` is at least ``round(p * 2**32)``. A call on a slice, with
    the slice's first position as ``offset``, draws the mask of the whole. A
    dropped infinity or NaN becomes 0.

    Args:
        x: CUDA tensor (float32, bfloat16 or float16) of any shape; one that is
            not contiguous is copied.
        p: Probability of dropping, between 0 and 1.
        seed: 64-bit key, or an int64 CUDA tensor of one element on ``x``'s
            device, read when the kernel runs: a captured graph draws a new
            mask on every replay once the tensor is written in between. It
            must not change between the forward and its backward.
        offset: Position of the first value (64 bits).
        residual: Added after the scaling; same shape, dtype and device as ``x``.
    """
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be between 0 and 1, got {p}")
    if isinstance(seed, torch.Tensor):
        if seed.numel() != 1 or seed.dtype != torch.int64:
            raise ValueError("a seed tensor must hold one int64 value, got "
                             f"{tuple(seed.shape)} of {seed.dtype}")
    else:
        seed = int(seed)
        if not -(1 << 63) <= seed <= _U64:
            raise ValueError(f"seed must fit 64 bits, got {seed}")
        seed &= _U64
    offset = int(offset)
    if not 0 <= offset <= _U64:
        raise ValueError(f"offset must fit 64 bits and not be negative, got {offset}")
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"residual must have x's shape and dtype, got {tuple(residual.shape)} "
                             f"of {residual.dtype} for {tuple(x.shape)} of {x.dtype}")
    on_one_device(x, seed if isinstance(seed, torch.Tensor) else None, residual)
    _lib.dtype_code(x.dtype)
    x = x.contiguous()
    residual = residual.contiguous() if residual is not None else None
    if torch.is_grad_enabled() and (x.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, p, seed, offset)
    return _launch(x, residual, p, seed, offset)


__all__ = ["dropout"]
