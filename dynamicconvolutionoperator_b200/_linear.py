"""Matrix product with bias, activation and residual in its epilogue
(``ddpm_linear_*`` in ``include/ddpm_b200.h``): ``nn.Linear`` or a 1x1
convolution over channel-last rows, on the library's tensor-core kernel.

The backward keeps ``x`` and ``weight`` only: with an activation, its argument
is computed again by the same product.
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from ._op import (activation_code, aligned, first_order, on_one_device, param_grad, ptr,
                  workspace)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` [..., k] as [m, k] with unit column stride (a view where the
    leading dimensions fold into rows of one stride, else a copy)."""
    if x.ndim == 2 and x.is_contiguous():
        return x
    k = x.shape[-1]
    flat = x if x.ndim == 2 else x.reshape(-1, k)
    if flat.stride(1) == 1 or k == 1:
        if flat.shape[0] <= 1 or flat.stride(0) >= k:
            return flat
    return flat.contiguous()


def _matrix(t: torch.Tensor, shape: tuple[int, int]) -> torch.Tensor:
    """``t`` as a contiguous matrix."""
    return (t if t.ndim == 2 else t.reshape(shape)).contiguous()


def _row_stride(flat: torch.Tensor) -> int:
    return flat.stride(0) if flat.shape[0] > 1 else flat.shape[1]


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(m, n, k, ld, act, code, bwd, is_aligned, index) -> int:
    """The plan's size on device ``index`` (it depends on the number of SMs)."""
    with torch.cuda.device(index):
        return int(_lib.load().ddpm_linear_workspace_bytes(m, n, k, ld, act, code, bwd, is_aligned))


def _forward(flat, w, b, res, act):
    m, k = flat.shape
    n = w.shape[0]
    dev, code, ld = flat.device, _lib.dtype_code(flat.dtype), _row_stride(flat)
    out = torch.empty((m, n), dtype=flat.dtype, device=dev)
    px, pw, pb, pr, po = flat.data_ptr(), w.data_ptr(), ptr(b), ptr(res), out.data_ptr()
    nbytes = _workspace_bytes(m, n, k, ld, act, code, 0, aligned(px, pw, pb, pr, po), dev.index)
    ws = workspace(nbytes, dev)
    _lib.call_on(dev, "ddpm_linear_fwd", px, ld, pw, pb, pr, po, ptr(ws), nbytes, m, n, k, act,
                 code)
    return out


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        flat = _rows(x)
        n = weight.shape[0]
        w = _matrix(weight, (n, flat.shape[1]))
        b = bias.contiguous() if bias is not None else None
        res = _matrix(residual, (-1, n)) if residual is not None else None
        out = _forward(flat, w, b, res, act)
        ctx.save_for_backward(flat, w, b if act else None)
        ctx.params = (weight, bias)  # gradient buffers are looked up by identity
        ctx.act, ctx.shape = act, x.shape
        return out if x.ndim == 2 else out.reshape(*x.shape[:-1], n)

    @staticmethod
    @first_order
    def backward(ctx, grad_out):
        flat, w, b = ctx.saved_tensors
        weight, bias = ctx.params
        need_x, need_w, need_b, need_res = ctx.needs_input_grad[:4]
        m, k = flat.shape
        n = w.shape[0]
        dev, dt = flat.device, flat.dtype
        gx = torch.empty((m, k), dtype=dt, device=dev) if need_x else None
        gw = param_grad(weight) if need_w else None
        gb = param_grad(bias) if need_b else None
        if m == 0:
            for g in (gw, gb):
                if g is not None:
                    g.zero_()
        elif need_x or need_w or need_b:
            g = _matrix(grad_out, (m, n))
            code, ld = _lib.dtype_code(dt), _row_stride(flat)
            px, pw, pb, pg = flat.data_ptr(), w.data_ptr(), ptr(b), g.data_ptr()
            ox, ow, ob = ptr(gx), ptr(gw), ptr(gb)
            nbytes = _workspace_bytes(m, n, k, ld, ctx.act, code, 1,
                                      aligned(px, pw, pb, pg, ox, ow, ob), dev.index)
            ws = workspace(nbytes, dev)
            _lib.call_on(dev, "ddpm_linear_bwd", px, ld, pw, pb, pg, ox, ow, ob, ptr(ws), nbytes,
                         m, n, k, ctx.act, code)
        if need_x and len(ctx.shape) != 2:
            gx = gx.reshape(ctx.shape)
        return gx, gw, gb, grad_out if need_res else None, None


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               activation: str | None = None,
               residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x weight^T + bias) + residual`` with one rounding.

    Sums are held in FP32; float32 data keeps its 24 bits (it is multiplied in
    three bf16 parts, an infinity in it gives a NaN). 16-bit gradients round
    ``dz = grad * act'`` once, as an operand of the two products it enters.

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
    if x.ndim < 1:
        raise ValueError("x must have at least one dimension [..., k]")
    shape = weight.shape
    if not (len(shape) == 2 or (len(shape) == 4 and shape[2] == shape[3] == 1)) or shape[1] != x.shape[-1]:
        raise ValueError(f"weight must be [n, {x.shape[-1]}] or [n, {x.shape[-1]}, 1, 1], "
                         f"got {tuple(shape)}")
    n = shape[0]
    if n < 1 or shape[1] < 1:
        raise ValueError(f"weight must not be empty, got {tuple(shape)}")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"bias must have shape ({n},), got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], n):
        raise ValueError(f"residual must have shape {(*x.shape[:-1], n)}, got {tuple(residual.shape)}")
    needs_grad = x.requires_grad
    for t in (weight, bias, residual):
        if t is not None:
            if t.dtype is not x.dtype:
                raise ValueError(f"all tensors must have one dtype, got {x.dtype} and {t.dtype}")
            needs_grad = needs_grad or t.requires_grad
    on_one_device(x, weight, bias, residual)
    _lib.dtype_code(x.dtype)
    if needs_grad and torch.is_grad_enabled():
        return _LinearAct.apply(x, weight, bias, residual, act)
    flat = _rows(x)
    out = _forward(flat, _matrix(weight, (n, flat.shape[1])),
                   bias.contiguous() if bias is not None else None,
                   _matrix(residual, (-1, n)) if residual is not None else None, act)
    return out if x.ndim == 2 else out.reshape(*x.shape[:-1], n)


__all__ = ["linear_act"]
