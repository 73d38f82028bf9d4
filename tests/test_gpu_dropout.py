"""dropout against Philox on Python integers and the float64 form."""

from __future__ import annotations

import pytest
import torch

from tests import _operators as ops

pytestmark = pytest.mark.gpu


def _case(size, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(size, generator=g, device="cuda").to(dtype) for _ in range(3)]


def _expect(x, mask, p, res):
    out = torch.where(mask.to(x.device), x.double() / (1 - p), torch.zeros_like(x.double()))
    return out if res is None else out + res.double()


def _tol(ref, x, p, res, dtype):
    # 1 / (1 - p) and the product are each rounded once in FP32, the sum once
    scale = x.double().abs() / (1 - p) + (0 if res is None else res.double().abs())
    return ops.bound(ref, scale, 4, dtype)


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("size", [1, 3, 4, 7, 8, 9, 255, 4099])
@pytest.mark.parametrize("offset", [0, 1, 4, 2 ** 32 + 6, 2 ** 40 - 3, 2 ** 63 + 8])
def test_mask_and_values(size, offset, dtype):
    from dynamicconvolutionoperator_b200 import dropout

    p, seed = 0.3, 0x1234_5678_9ABC_DEF1
    x, res, dy = _case(size, dtype)
    mask = ops.kept(size, p, seed, offset)
    for r in (None, res):
        xa = x.detach().requires_grad_()
        ra = None if r is None else r.detach().requires_grad_()
        out = dropout(xa, p, seed, offset, residual=ra)
        want = _expect(x, mask, p, r)
        ops.check("out", out.detach(), want, _tol(want, x, p, r, dtype))
        if r is None:
            assert torch.equal(out != 0, mask.cuda() & (x != 0))
        grads = torch.autograd.grad(out, [xa] + ([] if r is None else [ra]), dy)
        want = _expect(dy, mask, p, None)
        ops.check("x", grads[0], want, _tol(want, dy, p, None, dtype))
        if r is not None:
            assert torch.equal(grads[1], dy)


def test_pieces_draw_the_mask_of_the_whole():
    from dynamicconvolutionoperator_b200 import dropout

    x = torch.ones(10_007, device="cuda", dtype=torch.bfloat16)
    whole = dropout(x, 0.5, 77, 1000)
    cuts = [0, 1, 2, 9, 4000, 4001, 10_007]
    for a, b in zip(cuts, cuts[1:]):
        assert torch.equal(dropout(x[a:b], 0.5, 77, 1000 + a), whole[a:b])


def test_share_of_kept_values():
    from dynamicconvolutionoperator_b200 import dropout

    n = 1 << 24
    x = torch.ones(n, device="cuda")
    for p in (0.1, 0.5, 0.9):
        share = (dropout(x, p, 5) != 0).double().mean().item()
        assert abs(share - (1 - p)) < 6 * (p * (1 - p) / n) ** 0.5
    a, b = (dropout(x, 0.5, s) != 0 for s in (1, 2))
    assert abs((a == b).double().mean().item() - 0.5) < 6 * 0.5 / n ** 0.5


@pytest.mark.parametrize("dtype", ops.DTYPES)
def test_zero_and_one(dtype):
    from dynamicconvolutionoperator_b200 import dropout

    x, res, _ = _case(1003, dtype)
    assert torch.equal(dropout(x, 0.0, 3), x)
    assert not dropout(x, 1.0, 3).any()
    assert torch.equal(dropout(x, 1.0, 3, residual=res), res)
    assert dropout(x[:0], 0.5, 3).shape == (0,)


def test_dropped_infinities_do_not_reach_the_output():
    from dynamicconvolutionoperator_b200 import dropout

    mask = ops.kept(64, 0.5, 11, 0).cuda()
    x = torch.where(mask, torch.ones(64, device="cuda"), torch.full((64,), float("nan"), device="cuda"))
    assert torch.equal(dropout(x, 0.5, 11), 2.0 * mask)
    x = torch.where(mask, x, torch.full_like(x, float("inf")))
    assert torch.equal(dropout(x, 0.5, 11, residual=torch.ones_like(x)), 1 + 2.0 * mask)


def test_seed_on_the_device():
    from dynamicconvolutionoperator_b200 import dropout

    x, res, dy = _case(5000, torch.float32)
    for value in (0, 9, -1, 2 ** 63 - 1):
        seed = torch.tensor([value], device="cuda")
        assert torch.equal(dropout(x, 0.4, seed), dropout(x, 0.4, value))
    xa = x.requires_grad_()
    out = dropout(xa, 0.4, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(dy)


def test_strided_input_follows_its_row_major_order():
    from dynamicconvolutionoperator_b200 import dropout

    x = torch.randn(6, 10, device="cuda").t()
    assert torch.equal(dropout(x, 0.5, 4), dropout(x.contiguous(), 0.5, 4))
    x = torch.randn(2, 8, 4, 4, device="cuda").contiguous(memory_format=torch.channels_last)
    assert torch.equal(dropout(x, 0.5, 4), dropout(x.contiguous(), 0.5, 4))


def test_replayed_graph_draws_by_the_seed_tensor():
    from dynamicconvolutionoperator_b200 import dropout

    x = torch.randn(4096, device="cuda", requires_grad=True)
    dy = torch.randn(4096, device="cuda")
    seed = torch.tensor([5], device="cuda")

    def once():
        out = dropout(x, 0.5, seed)
        return [out.detach(), *torch.autograd.grad(out, x, dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for value in (6, 7):
        seed.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, once()))
        assert torch.equal(held[0] != 0, held[1] != 0)


def test_more_values_than_32_bits_count():
    from dynamicconvolutionoperator_b200 import dropout

    n = (1 << 32) + 4099
    if torch.cuda.mem_get_info()[0] < 5 * n:
        pytest.skip("needs 22 GB")
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    out = dropout(x, 0.5, 3)
    for at in (0, 1 << 31, (1 << 32) - 500, n - 1001):
        assert torch.equal(out[at:at + 1000], dropout(x[at:at + 1000], 0.5, 3, at))


def test_seed_on_another_device_is_refused():
    from dynamicconvolutionoperator_b200 import dropout

    with pytest.raises(RuntimeError, match="CUDA"):
        dropout(torch.ones(4, device="cuda"), 0.5, torch.tensor([1]))


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(requires_grad):
    from torch.autograd import forward_ad

    from dynamicconvolutionoperator_b200 import dropout

    x = torch.randn(40, device="cuda", requires_grad=requires_grad)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            dropout(forward_ad.make_dual(x, torch.ones_like(x)), 0.5, 1)
        if requires_grad:  # forward over reverse
            out = dropout(x, 0.5, 1)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, forward_ad.make_dual(torch.ones_like(x), x.detach()))


@pytest.mark.parametrize("size", [1, 6, 4099])
def test_last_positions(size):
    from dynamicconvolutionoperator_b200 import dropout

    x = torch.ones(size, device="cuda")
    offset = (1 << 64) - size
    assert torch.equal(dropout(x, 0.5, 9, offset) != 0, ops.kept(size, 0.5, 9, offset).cuda())
