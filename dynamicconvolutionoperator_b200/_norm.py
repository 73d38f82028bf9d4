"""Group norm with an activation over channel-last maps (``ddpm_group_norm_*``
in ``include/ddpm_b200.h``).

Statistics and sums are held in FP32 and the result is rounded once, after the
activation. The backward recomputes the normalised values from ``x`` and the
saved mean and reciprocal deviation; neither they nor the activation's argument
is stored.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._gradbuf import grad_buffer
from ._kernels import _require_cuda

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def activation_code(activation: str | None) -> int:
    try:
        return ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {sorted(k for k in ACTIVATIONS if k)} or "
                         f"None, got {activation!r}") from None


def _channel_last(t: torch.Tensor) -> torch.Tensor:
    """[N, C, *] as contiguous [N, *, C] (no copy for channel-last memory)."""
    return (t.movedim(1, -1) if t.ndim > 2 else t).contiguous()


def _channel_first(t: torch.Tensor) -> torch.Tensor:
    return t.movedim(-1, 1) if t.ndim > 2 else t


def _ptr(t: torch.Tensor | None):
    return t.data_ptr() if t is not None else None


def _sizes(xl: torch.Tensor) -> tuple[int, int, int]:
    n, c = xl.shape[0], xl.shape[-1]
    pixels = 1
    for d in xl.shape[1:-1]:
        pixels *= d
    return n, pixels, c


def _forward(xl, weight, bias, groups, eps, act):
    n, pixels, c = _sizes(xl)
    out = torch.empty_like(xl)
    stats = torch.empty((n, groups, 2), dtype=torch.float32, device=xl.device)
    code = _lib.dtype_code(xl.dtype)
    nbytes = int(_lib.load().ddpm_group_norm_workspace_bytes(n, pixels, c, groups, code, 0))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=xl.device)
    params = weight if weight is not None else bias
    _lib.call_on(xl.device, "ddpm_group_norm_fwd", xl.data_ptr(), _ptr(weight), _ptr(bias),
                 out.data_ptr(), stats.data_ptr(), ws.data_ptr(), nbytes, n, pixels, c, groups,
                 eps, act, code, code if params is None else _lib.dtype_code(params.dtype))
    return out, stats


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        xl = _channel_last(x)
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        out, stats = _forward(xl, w, b, groups, eps, act)
        ctx.save_for_backward(xl, w, b, stats)
        ctx.params = (weight, bias)  # gradient buffers are looked up by identity
        ctx.groups, ctx.act = groups, act
        return _channel_first(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        xl, w, b, stats = ctx.saved_tensors
        weight, bias = ctx.params
        n, pixels, c = _sizes(xl)
        need_x = ctx.needs_input_grad[0]
        need_w = weight is not None and ctx.needs_input_grad[1]
        need_b = bias is not None and ctx.needs_input_grad[2]
        gx = torch.empty_like(xl) if need_x else None
        gw = grad_buffer(weight, weight.shape, weight.dtype, xl.device) if need_w else None
        gb = grad_buffer(bias, bias.shape, bias.dtype, xl.device) if need_b else None
        if xl.numel() == 0:
            for g in (gw, gb):
                if g is not None:
                    g.zero_()
        else:
            g = _channel_last(grad_out)
            code = _lib.dtype_code(xl.dtype)
            nbytes = int(_lib.load().ddpm_group_norm_workspace_bytes(n, pixels, c, ctx.groups,
                                                                     code, 1))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=xl.device)
            params = w if w is not None else b
            _lib.call_on(xl.device, "ddpm_group_norm_bwd", xl.data_ptr(), g.data_ptr(), _ptr(w),
                         _ptr(b), stats.data_ptr(), _ptr(gx), _ptr(gw), _ptr(gb), ws.data_ptr(),
                         nbytes, n, pixels, c, ctx.groups, ctx.act, code,
                         code if params is None else _lib.dtype_code(params.dtype))
        return _channel_first(gx) if need_x else None, gw, gb, None, None, None


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
    if x.ndim < 2:
        raise ValueError(f"x must have at least two dimensions [N, C, *], got {tuple(x.shape)}")
    c, num_groups = x.shape[1], int(num_groups)
    if num_groups < 1 or c < 1 or c % num_groups:
        raise ValueError(f"num_groups must divide the channels, got {num_groups} for {c}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (c,):
            raise ValueError(f"{name} must have shape ({c},), got {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} must have x's dtype or float32, got {t.dtype} for {x.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")
    _require_cuda(x, *(t for t in (weight, bias) if t is not None))
    _lib.dtype_code(x.dtype)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, weight, bias)):
        return _GroupNormAct.apply(x, weight, bias, num_groups, float(eps), act)
    out, _ = _forward(_channel_last(x), weight.contiguous() if weight is not None else None,
                      bias.contiguous() if bias is not None else None, num_groups, float(eps), act)
    return _channel_first(out)


__all__ = ["ACTIVATIONS", "activation_code", "group_norm_act"]
