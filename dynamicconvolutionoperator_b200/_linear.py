"""Matrix product with bias, activation and residual in its epilogue
(``ddpm_linear_*`` in ``include/ddpm_b200.h``): ``nn.Linear`` or a 1x1
convolution over channel-last rows, on the library's tensor-core kernel.

The backward keeps ``x`` and ``weight`` only: with an activation, its argument
is computed again by the same product.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._gradbuf import grad_buffer
from ._kernels import _require_cuda
from ._norm import _ptr, activation_code


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` [..., k] as [m, k] with unit column stride (a view where the
    leading dimensions fold into rows of one stride, else a copy)."""
    k = x.shape[-1]
    flat = x if x.ndim == 2 else x.reshape(-1, k)
    if flat.stride(1) == 1 or k == 1:
        if flat.shape[0] <= 1 or flat.stride(0) >= k:
            return flat
    return flat.contiguous()


def _row_stride(flat: torch.Tensor) -> int:
    return flat.stride(0) if flat.shape[0] > 1 else flat.shape[1]


def _workspace(flat, n, act, bwd, tensors):
    m, k = flat.shape
    aligned = not any(t is not None and t.data_ptr() % 16 for t in tensors)
    nbytes = int(_lib.load().ddpm_linear_workspace_bytes(
        m, n, k, _row_stride(flat), act, _lib.dtype_code(flat.dtype), bwd, aligned))
    return torch.empty(nbytes, dtype=torch.uint8, device=flat.device), nbytes


def _forward(flat, w, b, res, act):
    m, k = flat.shape
    n = w.shape[0]
    out = torch.empty((m, n), dtype=flat.dtype, device=flat.device)
    ws, nbytes = _workspace(flat, n, act, 0, (flat, w, b, res, out))
    _lib.call_on(flat.device, "ddpm_linear_fwd", flat.data_ptr(), _row_stride(flat), w.data_ptr(),
                 _ptr(b), _ptr(res), out.data_ptr(), ws.data_ptr(), nbytes, m, n, k, act,
                 _lib.dtype_code(flat.dtype))
    return out


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        flat = _rows(x)
        n = weight.shape[0]
        w = weight.reshape(n, -1).contiguous()
        b = bias.contiguous() if bias is not None else None
        res = residual.reshape(-1, n).contiguous() if residual is not None else None
        out = _forward(flat, w, b, res, act)
        ctx.save_for_backward(flat, w, b if act else None)
        ctx.params = (weight, bias)  # gradient buffers are looked up by identity
        ctx.act, ctx.shape = act, x.shape
        return out.reshape(*x.shape[:-1], n)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        flat, w, b = ctx.saved_tensors
        weight, bias = ctx.params
        m, k = flat.shape
        n = w.shape[0]
        dev, dt = flat.device, flat.dtype
        need_w = ctx.needs_input_grad[1]
        need_b = bias is not None and ctx.needs_input_grad[2]
        gx = torch.empty((m, k), dtype=dt, device=dev) if ctx.needs_input_grad[0] else None
        gw = grad_buffer(weight, weight.shape, dt, dev) if need_w else None
        gb = grad_buffer(bias, bias.shape, dt, dev) if need_b else None
        if m == 0:
            for g in (gw, gb):
                if g is not None:
                    g.zero_()
        elif gx is not None or need_w or need_b:
            g = grad_out.reshape(m, n).contiguous()
            ws, nbytes = _workspace(flat, n, ctx.act, 1, (flat, w, b, g, gx, gw, gb))
            _lib.call_on(dev, "ddpm_linear_bwd", flat.data_ptr(), _row_stride(flat), w.data_ptr(),
                         _ptr(b), g.data_ptr(), _ptr(gx), _ptr(gw), _ptr(gb), ws.data_ptr(),
                         nbytes, m, n, k, ctx.act, _lib.dtype_code(dt))
        if gx is not None:
            gx = gx.reshape(ctx.shape)
        return gx, gw, gb, grad_out if ctx.needs_input_grad[3] else None, None


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
    shape = tuple(weight.shape)
    if not (len(shape) == 2 or (len(shape) == 4 and shape[2:] == (1, 1))) or shape[1] != x.shape[-1]:
        raise ValueError(f"weight must be [n, {x.shape[-1]}] or [n, {x.shape[-1]}, 1, 1], got {shape}")
    n = shape[0]
    if n < 1 or shape[1] < 1:
        raise ValueError(f"weight must not be empty, got {shape}")
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"bias must have shape ({n},), got {tuple(bias.shape)}")
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], n):
        raise ValueError(f"residual must have shape {(*x.shape[:-1], n)}, got {tuple(residual.shape)}")
    given = [t for t in (weight, bias, residual) if t is not None]
    for t in given:
        if t.dtype != x.dtype:
            raise ValueError(f"all tensors must have one dtype, got {x.dtype} and {t.dtype}")
    _require_cuda(x, *given)
    _lib.dtype_code(x.dtype)
    if torch.is_grad_enabled() and (x.requires_grad or any(t.requires_grad for t in given)):
        return _LinearAct.apply(x, weight, bias, residual, act)
    out = _forward(_rows(x), weight.reshape(n, -1).contiguous(),
                   bias.contiguous() if bias is not None else None,
                   residual.reshape(-1, n).contiguous() if residual is not None else None, act)
    return out.reshape(*x.shape[:-1], n)


__all__ = ["linear_act"]
