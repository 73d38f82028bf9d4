"""linear_act over sums so long that they are split: 16-bit data, every product.

A tensor-core addition cuts off what lies below the last bit of the running sum:
up to 2^-23 of it for 16 values of k. On data of one sign these add up, so the
length of a chain has to be bounded for the sum to be an FP32 sum.
"""

from __future__ import annotations

import pytest
import torch

from tests import _operators as ops
from tests.test_gpu_linear_act import _case, _run, _steps

pytestmark = pytest.mark.gpu

CHAIN = 16384  # values of k in a chain


def _close(name, got, ref, terms):
    """All terms positive: ``terms`` / 16 additions of at most CHAIN / 16 to a
    chain lose up to 2^-23 of the sum each; the chains' sums are added in FP32
    (2^-24 each); one rounding to the type."""
    half = torch.finfo(got.dtype).eps / 2
    lost = min(terms, CHAIN) / 16 * 2.0 ** -23 + (terms // CHAIN + 8) * 2.0 ** -24
    rel = ((got.double() - ref) / ref).abs().max().item()
    assert rel <= half * (1 + lost) + lost, f"{name}: {rel:.3g}"


def _positive(rows, cols, dtype, scale, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.empty(rows, cols, dtype=dtype, device="cuda")
    for at in range(0, rows, 1 << 16):
        part = t[at:at + (1 << 16)]
        part.copy_((torch.rand(part.shape, generator=g, device="cuda") + 0.5) * scale)
    return t


@pytest.mark.parametrize("dtype,rows", [(torch.float16, 1 << 18), (torch.bfloat16, (1 << 20) - 5)])
@pytest.mark.parametrize("n,k", [(2560, 1024), (64, 64)])
def test_weight_gradient_of_many_rows_of_one_sign(dtype, rows, n, k):
    from dynamicconvolutionoperator_b200 import linear_act

    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    x = _positive(rows, k, dtype, 1.0, 1)
    dy = _positive(rows, n, dtype, 2.0 ** -10, 2)
    w = torch.zeros(n, k, dtype=dtype, device="cuda", requires_grad=True)
    gw, = torch.autograd.grad(linear_act(x, w), w, dy)
    for cols in (slice(0, 40), slice(n - 40, n)):
        ref = sum(dy[i:i + (1 << 16), cols].double().t() @ x[i:i + (1 << 16)].double()
                  for i in range(0, rows, 1 << 16))
        _close("weight", gw[cols], ref, rows)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_rows_of_one_sign(dtype):
    """The forward over 2^20 columns, and the data gradient over 2^20 outputs."""
    from dynamicconvolutionoperator_b200 import linear_act

    long = (1 << 20) + 24
    x, w = _positive(40, long, dtype, 1.0, 3), _positive(72, long, dtype, 2.0 ** -10, 4)
    _close("out", linear_act(x, w), x.double() @ w.double().t(), long)
    w, dy = _positive(long, 72, dtype, 1.0, 5), _positive(40, long, dtype, 2.0 ** -10, 6)
    x = torch.zeros(40, 72, dtype=dtype, device="cuda", requires_grad=True)
    gx, = torch.autograd.grad(linear_act(x, w), x, dy)
    _close("x", gx, dy.double() @ w.double(), long)


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("m,n,k", [(9, 33, 40_001), (300, 520, 16_400), (130, 32_776, 24),
                                   (33, 17_001, 17)])
def test_split_sums_match_float64(m, n, k, dtype):
    """Every epilogue of a split product, ragged sizes, rows that TMA cannot address."""
    x, w, b, res, dy = _case(m, n, k, dtype, seed=6)
    _run(x, w, b, res, dy, "silu")
    _run(x, w, b, None, dy, None)
    _run(x, w, None, res, dy, "gelu")


def test_split_sums_captured_and_repeated():
    from dynamicconvolutionoperator_b200 import linear_act

    x, w, b, res, dy = _case(70, 40, 50_000, torch.bfloat16, seed=9)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def once():
        out = linear_act(*leaves, "silu", res)
        return [out.detach(), *torch.autograd.grad(out, leaves, dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(held, once()))


def test_partials_of_a_weight_gradient_in_several_parts():
    """64 splits of 5000 x 1024 partials would take 1.3 GB: 4096 rows of them at a time."""
    from dynamicconvolutionoperator_b200 import linear_act

    if torch.cuda.mem_get_info()[0] < 32 << 30:
        pytest.skip("needs 32 GB")
    rows, n, k = (1 << 20) - 5, 5000, 1024
    x = _positive(rows, k, torch.bfloat16, 1.0, 11)
    dy = _positive(rows, n, torch.bfloat16, 2.0 ** -10, 12)
    w = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    out = linear_act(x, w)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    gw, = torch.autograd.grad(out, w, dy)
    assert torch.cuda.max_memory_allocated() - before < 1.1 * 2 ** 30
    for cols in (slice(0, 20), slice(4086, 4106), slice(n - 20, n)):
        ref = sum(dy[i:i + (1 << 16), cols].double().t() @ x[i:i + (1 << 16)].double()
                  for i in range(0, rows, 1 << 16))
        _close("weight", gw[cols], ref, rows)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_partials_of_a_forward_in_several_parts(dtype):
    """Two splits of 33001 x 4096 partials: 32768 rows at a time, in the forward and in
    the product that makes dz."""
    from dynamicconvolutionoperator_b200 import linear_act

    if torch.cuda.mem_get_info()[0] < 32 << 30:
        pytest.skip("needs 32 GB")
    m, n, k = 33_001, 4096, 16_400
    x, w, b, res, dy = _case(m, n, k, dtype, seed=13)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    out = linear_act(*leaves, "silu", res)
    gx, gw, gb = torch.autograd.grad(out, leaves, dy)
    half = torch.finfo(dtype).eps / 2
    for cols in (slice(0, 24), slice(n - 24, n)):
        ref, scale, _, grads = ops.linear(x.detach(), w.detach()[cols], b.detach()[cols], "silu",
                                          res[:, cols], dy[:, cols])
        ops.check("out", out.detach()[:, cols], ref, ops.bound(ref, scale, _steps(k, dtype), dtype))
        for key, got in (("weight", gw[cols]), ("bias", gb[cols])):
            r, s, rounded = grads[key]
            tol = ops.bound(r, s, _steps(m, dtype) + _steps(k, dtype), dtype)
            tol = tol + half * rounded * (1 + half) + torch.finfo(dtype).tiny * half * m * 8
            ops.check(key, got, r, tol)
    # the rows around the seam as a call of their own: the same sums in the same order
    seam = slice(32_700, m)
    part = x.detach()[seam].requires_grad_()
    again = linear_act(part, w.detach(), b.detach(), "silu", res[seam])
    assert torch.equal(again, out[seam])
    gp, = torch.autograd.grad(again, part, dy[seam])
    assert torch.equal(gp, gx[seam])
