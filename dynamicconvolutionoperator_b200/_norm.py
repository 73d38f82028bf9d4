"""Group norm with an activation over channel-last maps (``ddpm_group_norm_*``
in ``include/ddpm_b200.h``).

Statistics and sums are held in FP32 and the result is rounded once, after the
activation. The backward recomputes the normalised values from ``x`` and the
saved mean and reciprocal deviation; neither they nor the activation's argument
is stored.
"""

from __future__ import annotations

import functools
import math

import torch

from . import _lib
from ._op import (activation_code, aligned, first_order, on_one_device, param_grad, ptr,
                  workspace)


def _channel_last(t: torch.Tensor) -> torch.Tensor:
    """[N, C, *] as contiguous [N, *, C] (no copy for channel-last memory)."""
    if t.ndim == 4:
        return t.permute(0, 2, 3, 1).contiguous()
    return (t.movedim(1, -1) if t.ndim > 2 else t).contiguous()


def _channel_first(t: torch.Tensor) -> torch.Tensor:
    if t.ndim == 4:
        return t.permute(0, 3, 1, 2)
    return t.movedim(-1, 1) if t.ndim > 2 else t


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(n, pixels, c, groups, code, bwd, is_aligned, index) -> int:
    """The plan's size on device ``index`` (it depends on the number of SMs)."""
    with torch.cuda.device(index):
        return int(_lib.load().ddpm_group_norm_workspace_bytes(n, pixels, c, groups, code, bwd,
                                                               is_aligned))


def _forward(xl, w, b, groups, eps, act):
    shape = xl.shape
    n, c = shape[0], shape[-1]
    pixels = math.prod(shape[1:-1])
    dev, code = xl.device, _lib.dtype_code(xl.dtype)
    out = torch.empty_like(xl)
    stats = torch.empty((n, groups, 2), dtype=torch.float32, device=dev)
    px, po = xl.data_ptr(), out.data_ptr()
    nbytes = _workspace_bytes(n, pixels, c, groups, code, 0, aligned(px, po), dev.index)
    ws = workspace(nbytes, dev)
    params = w if w is not None else b
    _lib.call_on(dev, "ddpm_group_norm_fwd", px, ptr(w), ptr(b), po, stats.data_ptr(), ptr(ws),
                 nbytes, n, pixels, c, groups, eps, act, code,
                 code if params is None else _lib.dtype_code(params.dtype))
    return out, stats


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        xl = _channel_last(x)
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        out, stats = _forward(xl, w, b, groups, eps, act)
        ctx.save_for_backward(xl, w, b)
        ctx.stats = stats
        ctx.params = (weight, bias)  # gradient buffers are looked up by identity
        ctx.args = (groups, act)
        return _channel_first(out)

    @staticmethod
    @first_order
    def backward(ctx, grad_out):
        xl, w, b = ctx.saved_tensors
        weight, bias = ctx.params
        groups, act = ctx.args
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dev = xl.device
        gx = torch.empty_like(xl) if need_x else None
        gw = param_grad(weight) if need_w else None
        gb = param_grad(bias) if need_b else None
        if xl.numel() == 0:
            for g in (gw, gb):
                if g is not None:
                    g.zero_()
        else:
            g = _channel_last(grad_out)
            shape = xl.shape
            n, c = shape[0], shape[-1]
            pixels = math.prod(shape[1:-1])
            code = _lib.dtype_code(xl.dtype)
            px, pg, po = xl.data_ptr(), g.data_ptr(), ptr(gx)
            nbytes = _workspace_bytes(n, pixels, c, groups, code, 1, aligned(px, pg, po), dev.index)
            ws = workspace(nbytes, dev)
            params = w if w is not None else b
            _lib.call_on(dev, "ddpm_group_norm_bwd", px, pg, ptr(w), ptr(b), ctx.stats.data_ptr(),
                         po, ptr(gw), ptr(gb), ptr(ws), nbytes, n, pixels, c, groups, act, code,
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
    for t in (weight, bias):
        if t is None:
            continue
        if t.shape != (c,):
            raise ValueError(f"{'weight' if t is weight else 'bias'} must have shape ({c},), "
                             f"got {tuple(t.shape)}")
        if t.dtype is not x.dtype and t.dtype is not torch.float32:
            raise ValueError(f"{'weight' if t is weight else 'bias'} must have x's dtype or "
                             f"float32, got {t.dtype} for {x.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")
    on_one_device(x, weight, bias)
    _lib.dtype_code(x.dtype)
    if torch.is_grad_enabled() and (x.requires_grad
                                    or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _GroupNormAct.apply(x, weight, bias, num_groups, float(eps), act)
    out, _ = _forward(_channel_last(x), weight.contiguous() if weight is not None else None,
                      bias.contiguous() if bias is not None else None, num_groups, float(eps), act)
    return _channel_first(out)


__all__ = ["group_norm_act"]
