"""Group norm with an activation over channel-last maps (``ddpm_group_norm_*``
in ``include/ddpm_b200.h``).

Statistics and sums are held in FP32 and the result is rounded once, after the
activation. The backward recomputes the normalised values from ``x`` and the
saved mean and reciprocal deviation; neither they nor the activation's argument
is stored.
"""

from __future__ import annotations

import torch

from ._op import activation_code, operators


def group_norm_act(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, eps: float = 1e-5,
                   activation: str | None = None) -> torch.Tensor:
    """``act(group_norm(x))`` for ``x`` [N, C, *] held channel-last.

    Mean and biased variance run over each sample's group of ``C // num_groups``
    channels and all further dimensions. The result has channel-last memory
    (``[N, *, C]`` contiguous, torch's ``channels_last`` for four dimensions);
    an ``x`` in another layout is copied first.

    Args:
        x: CUDA tensor (float32, bfloat16 or float16) of at least two dimensions.
        num_groups: Number of groups; divides C.
        weight: Scale per channel [C], in ``x``'s dtype or float32; None: ones.
        bias: Offset per channel [C], in the same dtype as ``weight``; None: zeros.
        eps: Added to the variance.
        activation: "relu", "silu", "gelu" (erf form), "gelu_tanh" or None.
    """
    act = activation_code(activation)
    return operators().group_norm_act(x, int(num_groups), weight, bias, float(eps), act)


__all__ = ["group_norm_act"]
