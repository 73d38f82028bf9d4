"""Dropout from a counter-based generator (``ddpm_dropout`` in
``include/ddpm_b200.h``).

The mask is a function of the seed and of each value's position, so it is never
stored: the backward pass draws it again. There is no hidden generator state:
equal arguments give equal results, on every device and in every order.
"""

from __future__ import annotations

import torch

from ._op import operators

_U64 = (1 << 64) - 1


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
        offset: Position of the first value; every position fits 64 bits.
        residual: Added after the scaling; same shape, dtype and device as ``x``.
    """
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be between 0 and 1, got {p}")
    held = None
    if isinstance(seed, torch.Tensor):
        seed, held = 0, seed
    else:
        seed = int(seed)
        if not -(1 << 63) <= seed <= _U64:
            raise ValueError(f"seed must fit 64 bits, got {seed}")
    offset = int(offset)
    if not 0 <= offset <= _U64:
        raise ValueError(f"offset must fit 64 bits and not be negative, got {offset}")
    return operators().dropout(x, p, seed & _U64, held, offset, residual)


__all__ = ["dropout"]
