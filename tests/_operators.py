"""Plain float64 forms of the channel-last operators and the error bounds their
tests use.

Bounds: an output rounded once to type t is off by at most half a step,
``finfo(t).eps / 2`` relative to its value; what is computed in FP32 before
that is off by a small multiple of 2^-24 of the terms it is made of. Each test
passes those terms (``scale``) and the multiple (``steps``).
"""

from __future__ import annotations

import math

import torch

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def slope(z, name):
    z = z.detach().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(act(z, name).sum(), z)[0] if name else torch.ones_like(z)


def bound(ref, scale, steps, dtype, act_steps=0.0):
    """Elementwise error bound: half a step of ``dtype`` at the (slightly wrong)
    value plus ``steps`` FP32 roundings of ``scale``."""
    err = scale * steps * 2.0 ** -24
    half = torch.finfo(dtype).eps / 2
    # below the smallest normal number a half step is absolute
    return (ref.abs() + err) * half + err + torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def check(name, got, ref, tol):
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    got = got.double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - ref).abs() / tol
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: error {worst:.3g} times its bound"


def group_norm(x, groups, weight, bias, eps, name, dy=None):
    """(out, scale of out, [(gradient, its scale)...]) in float64 for x [N, C, *]."""
    n, c = x.shape[:2]
    xs = x.double().reshape(n, groups, -1)
    var, mean = torch.var_mean(xs, 2, correction=0, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    view = (1, c) + (1,) * (x.ndim - 2)
    w = torch.ones(c, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    w, b = w.reshape(view), b.reshape(view)
    xhat = ((xs - mean) * rstd).reshape(x.shape)
    # terms of z: the subtraction's operands in units of the deviation
    parts = ((xs.abs() + mean.abs() + (xs - mean).abs()) * rstd).reshape(x.shape)
    z = xhat * w + b
    out = act(z, name)
    zscale = parts * w.abs() + b.abs()
    if dy is None:
        return out, zscale * 1.2 + out.abs(), []
    g = dy.double()
    s = slope(z, name)
    dz = g * s
    # |act''| <= 1.2 for every activation here; relu's slope is exact away from 0
    dzs = g.abs() * (s.abs() + (0 if name in (None, "relu") else 1.2) * zscale)
    dims = (0,) + tuple(range(2, x.ndim))
    gw, gb = (dz * xhat).sum(dims), dz.sum(dims)
    gws = (dzs * xhat.abs() + dz.abs() * parts).sum(dims)
    gbs = dzs.sum(dims)

    def fold(v):
        v = v.reshape(n, groups, -1)
        return v.mean(2, keepdim=True).expand(v.shape).reshape(x.shape)

    r = rstd.expand(xs.shape).reshape(x.shape)
    dx = r * (w * dz - fold(w * dz) - xhat * fold(w * dz * xhat))
    dxs = r * (w.abs() * dzs + fold(w.abs() * dzs)
               + (xhat.abs() + parts) * fold(w.abs() * dzs * (xhat.abs() + parts)))
    return out, zscale * 1.2 + out.abs(), [(dx, dxs), (gw, gws), (gb, gbs)]


def philox(counter: int, key: int) -> list[int]:
    """Philox-4x32-10 (Salmon et al. 2011) on Python integers."""
    c = [counter & 0xFFFFFFFF, (counter >> 32) & 0xFFFFFFFF, 0, 0]
    k = [key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF]
    return philox_words(c, k)


def philox_words(c, k):
    c, k = list(c), list(k)
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(size: int, p: float, seed: int, offset: int) -> torch.Tensor:
    least = math.floor(p * 2 ** 32 + 0.5)
    words, at = [], offset // 4
    while len(words) < size + offset % 4:
        words += philox(at % 2 ** 62, seed)
        at += 1
    return torch.tensor([w >= least for w in words[offset % 4:][:size]], dtype=torch.bool)


def linear(x, w, b, name, res, dy=None):
    """(out, scale of out, z's scale, gradients with their scales) in float64
    for x [m, k], w [n, k]. A gradient's scales: (terms rounded in FP32, terms
    holding dz rounded to the data's type)."""
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    zscale = xd.abs() @ wd.abs().t()
    if b is not None:
        z = z + b.double()
        zscale = zscale + b.double().abs()
    out = act(z, name)
    # |act'| <= 1.13 for every activation here
    scale = 1.2 * zscale + out.abs()
    if res is not None:
        out = out + res.double()
        scale = scale + res.double().abs()
    if dy is None:
        return out, scale, zscale, None
    g = dy.double()
    s = slope(z, name)
    dz = g * s
    wobble = 0 if name in (None, "relu") else 1.2 * zscale  # |act''| <= 1.2
    dzs = g.abs() * (s.abs() + wobble)
    return out, scale, zscale, {
        "x": (dz @ wd, dzs @ wd.abs(), dz.abs() @ wd.abs()),
        "weight": (dz.t() @ xd, dzs.t() @ xd.abs(), dz.abs().t() @ xd.abs()),
        "bias": (dz.sum(0), dzs.sum(0), torch.zeros_like(dz.sum(0))),
    }


def linear_choice(m, n, k, dtype, product, name=None):
    """How a product of ``linear_act`` runs: {"forward", "x", "weight"} as (tile
    columns, blocks, epilogue warps, splits, stages, fits)."""
    import ctypes

    from dynamicconvolutionoperator_b200 import _lib
    from dynamicconvolutionoperator_b200._op import activation_code

    out = (ctypes.c_int * 6)()
    _lib.call("ddpm_test_linear_choice", m, n, k, activation_code(name), _lib.dtype_code(dtype),
              ["forward", "x", "weight"].index(product), out)
    return tuple(out)
