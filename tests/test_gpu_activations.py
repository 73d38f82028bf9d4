"""The activations of the channel-last operators value by value, over the whole range
of their argument: 16-bit data takes fitted and approximate functions."""

from __future__ import annotations

import pytest
import torch

from tests import _operators as ops

pytestmark = pytest.mark.gpu

HALVES = [torch.bfloat16, torch.float16]


def _ndtr(z):
    """Phi with its relative digits below zero too (torch.special.ndtr is
    (1 + erf) / 2 and has none of them at -8)."""
    return 0.5 * torch.special.erfc(-z * 0.7071067811865476)


def _sweep(dtype):
    """Every value of the type in +-14, and a few far beyond."""
    z = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    z = z[(z.double().abs() <= 14)]
    far = torch.tensor([-6e4, -1000., -90., 15., 90., 1000., 6e4], dtype=dtype)
    z = torch.cat([z, far])
    return torch.cat([z, z.new_zeros(-len(z) % 8)]).view(-1, 8).cuda()


def _through_linear(z, name, rows):
    """act(z) and act'(z): the product with the identity is exact."""
    from dynamicconvolutionoperator_b200 import linear_act

    eye = torch.eye(8, dtype=z.dtype, device="cuda")
    outs, slopes = [], []
    for part in z.split(rows):
        p = part.detach().requires_grad_()
        out = linear_act(p, eye, activation=name)
        outs.append(out.detach())
        slopes.append(torch.autograd.grad(out, p, torch.ones_like(out))[0])
    return torch.cat(outs).double(), torch.cat(slopes).double()


@pytest.mark.parametrize("rows", [8, 512])
@pytest.mark.parametrize("dtype", HALVES)
def test_gelu_keeps_its_digits_over_the_whole_range(dtype, rows):
    """The stated errors of the fitted Phi(-|z|): 1.7e-5 of it down to -13.2 and 0 beyond;
    then one rounding. The slope is Phi(z) + z phi(z), whose second term adds FP32
    roundings (z^2 / 2 in the exponent, 2^-24 each, and the hardware's 2^-22)."""
    z = _sweep(dtype) if rows > 8 else _sweep(dtype)[::16].contiguous()
    out, slope = _through_linear(z, "gelu", rows)
    zd = z.double()
    phi, density = _ndtr(zd), torch.exp(-zd * zd / 2) * 0.3989422804014327
    err = 1.8e-5 * _ndtr(-zd.abs()) + torch.where(zd < -13.2, phi, 0.0)
    half = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # half a subnormal step and one more

    def check(name, got, ref, err):
        over = (got - ref).abs() / ((ref.abs() + err) * half + err + least)
        at = over.argmax()
        assert over.max() <= 1, (name, zd.flatten()[at].item(), over.max().item())

    check("gelu", out, zd * phi, zd.abs() * err)
    # beyond 13.2 the exponential is 0 in the slope's second term too
    wobble = (zd * density).abs() * torch.where(zd < -13.2, 1.0, (zd * zd + 8) * 2.0 ** -22)
    check("slope", slope, phi + zd * density, err + wobble)


@pytest.mark.parametrize("dtype", HALVES)
def test_gelu_of_a_norm_keeps_its_digits(dtype):
    """The norm kernels' activation: a constant group leaves the bias as its argument."""
    from dynamicconvolutionoperator_b200 import group_norm_act

    z = _sweep(dtype).flatten()[:2048]
    for side in (1, 20):  # a cluster's kernel, and the ring's
        x = torch.full((3, side, side, 2048), 1.5, dtype=dtype, device="cuda").permute(0, 3, 1, 2)
        out = group_norm_act(x, 32, torch.ones_like(z), z, activation="gelu")[0, :, 0, 0].double()
        zd = z.double()
        ref = zd * _ndtr(zd)
        err = zd.abs() * 1.8e-5 * _ndtr(-zd.abs()) + torch.where(zd < -13.2, ref.abs(), 0.0)
        half = torch.finfo(dtype).eps / 2
        tol = (ref.abs() + err) * half + err + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        assert ((out - ref).abs() <= tol).all()


@pytest.mark.parametrize("rows", [4, 200])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("name", ["relu", "silu", "gelu", "gelu_tanh"])
def test_infinities(name, dtype, rows):
    from dynamicconvolutionoperator_b200 import linear_act

    one = torch.ones(1, 1, dtype=dtype, device="cuda")
    big = torch.tensor([float("inf"), float("nan")], device="cuda", dtype=dtype)
    out = linear_act(big.repeat(rows // 2)[:, None], one, activation=name).view(-1, 2)
    assert (out[:, 0] == float("inf")).all() and out[:, 1].isnan().all()


@pytest.mark.parametrize("rows", [4, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ops.ACTS)
def test_slopes_of_large_values(name, dtype, rows):
    """Far out an activation is z or 0 and its slope 1 or 0, also where z^2 overflows."""
    from dynamicconvolutionoperator_b200 import linear_act

    z = torch.tensor([1e20, -1e20, 3e38, -3e38, 1e10, -1e10, 150., -150.], device="cuda", dtype=dtype)
    x = z.repeat(rows)[:, None].requires_grad_()
    out = linear_act(x, torch.ones(1, 1, dtype=dtype, device="cuda"), activation=name)
    slope, = torch.autograd.grad(out, x, torch.ones_like(out))
    want = torch.ones_like(z) if name is None else (z > 0).to(dtype)
    assert torch.equal(slope.view(-1, 8), want.expand(rows, 8))
    assert torch.equal(out.detach().view(-1, 8), (z * want).expand(rows, 8))
