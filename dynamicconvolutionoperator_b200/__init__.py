"""B200-native (sm_100a) DDPM: a drop-in for lartpang/DynamicConvolutionOperator's
``triton_impl.DDPM`` and ``_triton_kernels`` GPU path.

Public surface:
  * ``DDPM`` — the module (reference ``triton_impl.py:247-392``).
  * ``fused_dynamic_cat`` / ``fused_generator_dynamic_cat`` — the differentiable
    kernel-level ops (reference ``_triton_kernels.py:869``, ``:1056``).
  * ``group_norm_act`` / ``linear_act`` / ``dropout`` — differentiable
    channel-last operators around the module: group norm with an activation,
    matrix product with bias, activation and residual, dropout from a
    counter-based generator.
  * ``data_parallel`` — batch-sharded training helpers over NCCL.
"""

from ._dropout import dropout
from ._kernels import fused_dynamic_cat, fused_generator_dynamic_cat
from ._linear import linear_act
from ._norm import group_norm_act
from .ddpm import DDPM

__all__ = ["DDPM", "dropout", "fused_dynamic_cat", "fused_generator_dynamic_cat",
           "group_norm_act", "linear_act"]
