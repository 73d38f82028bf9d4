"""Matrix product with bias, activation and residual in its epilogue
(``ddpm_linear_*`` in ``include/ddpm_b200.h``): ``nn.Linear`` or a 1x1
convolution over channel-last rows, on the library's tensor-core kernel.

The backward keeps ``x`` and ``weight`` only: with an activation, its argument
is computed again by the same product.
"""

from __future__ import annotations

import torch

from ._op import activation_code, operators


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               activation: str | None = None,
               residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x weight^T + bias) + residual`` with one rounding.

    Sums are held in FP32; float32 data keeps its 24 bits (it is multiplied in
    three bf16 parts; an infinity in it gives a NaN in the row or column that it
    belongs to, but for the forward of up to eight rows, which multiplies in FP32
    and gives the infinity). 16-bit gradients round ``dz = grad * act'`` once, as an
    operand of the two products it enters.

    Args:
        x: CUDA tensor (float32, bfloat16 or float16) [..., k]. Rows may lie
            apart (a slice of wider rows is not copied); other layouts are copied.
        weight: [n, k], or a 1x1 convolution's [n, k, 1, 1].
        bias: [n] or None.
        activation: "relu", "silu", "gelu" (erf form), "gelu_tanh" or None.
        residual: [..., n] or None; added behind the activation.

    All tensors have one dtype and device. Returns [..., n], contiguous.
    """
    act = activation_code(activation)
    return operators().linear_act(x, weight, bias, act, residual)


__all__ = ["linear_act"]
