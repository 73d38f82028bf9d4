"""group_norm_act against a float64 form: values, gradients, layouts, streams,
graphs, empty inputs."""

from __future__ import annotations

import pytest
import torch

from tests import _operators as ops

pytestmark = pytest.mark.gpu

# FP32 roundings on the way to a value: the statistics are folded in three
# levels (a thread's, a block's, a sample's partial sums; at most 64 + 12 + 20
# roundings of a running sum each), the value itself takes about ten more.
STEPS = 128


def _case(shape, dtype, groups, seed=0, mean=0.5, channels_last=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = shape[1]
    x = torch.randn(shape, generator=g, device="cuda") * 1.5 + mean
    x = x.to(dtype)
    if channels_last and x.ndim > 2:
        x = x.movedim(1, -1).contiguous().movedim(-1, 1)
    w = (1 + 0.2 * torch.randn(c, generator=g, device="cuda")).to(dtype)
    b = (0.2 * torch.randn(c, generator=g, device="cuda")).to(dtype)
    dy = torch.randn(shape, generator=g, device="cuda").to(dtype)
    return x, w, b, dy


def _run(x, groups, w, b, dy, name, eps=1e-5, steps=STEPS):
    from dynamicconvolutionoperator_b200 import _lib, group_norm_act

    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    xa = next(it)
    wa = next(it) if w is not None else None
    ba = next(it) if b is not None else None
    out = group_norm_act(xa, groups, wa, ba, eps, activation=name)
    grads = torch.autograd.grad(out, leaves, dy)
    with torch.no_grad():
        again = group_norm_act(x, groups, w, b, eps, activation=name)
    assert torch.equal(out, again)
    ref, scale, gref = ops.group_norm(x, groups, w, b, eps, name, dy)
    ops.check("out", out.detach(), ref, ops.bound(ref, scale, steps, x.dtype))
    names = ["x"] + ["weight"] * (w is not None) + ["bias"] * (b is not None)
    want = [gref[0]] + [gref[1]] * (w is not None) + [gref[2]] * (b is not None)
    for nm, got, (r, s) in zip(names, grads, want):
        ops.check(nm, got, r, ops.bound(r, s, steps, got.dtype))
    assert _lib.device_status() == 0
    return out, grads


SHAPES = [
    ((1, 8, 1), 1),               # one pixel
    ((1, 64, 16, 16), 8),
    ((3, 60, 37, 53), 5),         # 4-channel loads, ragged rows
    ((2, 18, 9, 7), 3),           # 2-channel loads
    ((5, 7, 11, 3), 7),           # one channel a load, one channel a group
    ((2, 33, 130), 1),            # one group, odd channels
    ((4, 96), 4),                 # rows without pixels
    ((1, 64, 256, 256), 8),       # one sample over the whole grid
    ((300, 16, 5, 3), 2),         # more samples than blocks
    ((2, 2304, 6, 5), 9),         # channels of several tiles, groups across them
    ((2, 515, 17), 5),            # several tiles of single channels
    ((3000, 24), 3),              # rows without pixels, more than blocks
    ((1500, 40, 6), 5),
    ((1, 8, 3, 4, 5), 4),         # three spatial dimensions
]


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_matches_float64(shape, groups, dtype):
    x, w, b, dy = _case(shape, dtype, groups)
    _run(x, groups, w, b, dy, "silu")


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("name", ops.ACTS)
def test_activations(name, dtype):
    x, w, b, dy = _case((2, 32, 19, 23), dtype, 4, seed=3)
    if name == "relu":
        # away from the kink, where a rounding turns the slope on or off
        z = ops.group_norm(x, 4, w, b, 1e-5, None)[0]
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    _run(x, 4, w, b, dy, name)


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("shape,groups", [
    ((3, 64, 512, 300), 8),    # a sample of more chunks than a block can hold
    ((2, 64, 256, 257), 8),    # samples held between the phases
    ((7, 256, 60, 61), 64),    # many groups, four channels each
    ((40, 24, 100, 71), 1),    # 48-byte rows (96 in float32), one group
    ((5, 2048, 20, 33), 32),   # few rows a block
    ((1000, 32, 9, 15), 4),    # more samples than blocks
    ((1, 16, 1024, 1024), 4),
])
def test_large(shape, groups, dtype):
    x, w, b, dy = _case(shape, dtype, groups, seed=5)
    _run(x, groups, w, b, dy, "silu", steps=256)


@pytest.mark.parametrize("name", ops.ACTS)
@pytest.mark.parametrize("dtype", ops.DTYPES)
def test_large_activations(name, dtype):
    x, w, b, dy = _case((4, 64, 100, 120), dtype, 8, seed=6, mean=3.0)
    if name == "relu":
        z = ops.group_norm(x, 8, w, b, 1e-5, None)[0]
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    _run(x, 8, w, b, dy, name)


@pytest.mark.parametrize("mean", [0.0, 300.0])
def test_mean_far_from_zero(mean):
    """The variance is summed about values of the data: a mean of 200
    deviations costs its own digits and no others."""
    x, w, b, dy = _case((2, 16, 64, 64), torch.float32, 4, mean=mean)
    _run(x, 4, w, b, dy, None)


def test_constant_input_gives_the_bias():
    from dynamicconvolutionoperator_b200 import group_norm_act

    x = torch.full((2, 8, 5, 5), 3.25, device="cuda").contiguous(memory_format=torch.channels_last)
    b = torch.arange(8.0, device="cuda")
    out = group_norm_act(x, 2, torch.ones(8, device="cuda"), b)
    assert torch.equal(out, b.reshape(1, 8, 1, 1).expand_as(out))


def test_without_weight_and_bias_and_mixed_types():
    x, w, b, dy = _case((2, 24, 10, 9), torch.bfloat16, 4)
    _run(x, 4, None, None, dy, "silu")
    _run(x, 4, w, None, dy, "silu")
    _run(x, 4, None, b.float(), dy, "silu")
    out, grads = _run(x, 4, w.float(), b.float(), dy, "gelu")
    assert grads[1].dtype == torch.float32 and out.dtype == torch.bfloat16


@pytest.mark.parametrize("shape", [(0, 8, 4, 4), (2, 8, 0, 4)])
def test_empty(shape):
    from dynamicconvolutionoperator_b200 import group_norm_act

    x = torch.empty(shape, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    out = group_norm_act(x, 2, w)
    assert out.shape == x.shape
    gx, gw = torch.autograd.grad(out, (x, w), torch.empty_like(out))
    assert gx.shape == x.shape and not gw.any()


def test_layouts_agree_and_output_is_channel_last():
    from dynamicconvolutionoperator_b200 import group_norm_act

    x, w, b, dy = _case((2, 24, 12, 10), torch.float32, 3)
    want = group_norm_act(x, 3, w, b, activation="silu")
    assert want.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(group_norm_act(x.contiguous(), 3, w, b, activation="silu"), want)
    wide = torch.zeros(2, 24, 12, 20, device="cuda")
    wide[..., ::2] = x
    assert torch.equal(group_norm_act(wide[..., ::2], 3, w, b, activation="silu"), want)
    # an address that allows no vector loads
    flat = torch.empty(x.numel() + 1, device="cuda")
    off = flat[1:].view(2, 12, 10, 24)
    off.copy_(x.permute(0, 2, 3, 1))
    got = group_norm_act(off.permute(0, 3, 1, 2), 3, w, b, activation="silu")
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("side", [8, 300])
def test_only_the_asked_gradients(side):
    from dynamicconvolutionoperator_b200 import group_norm_act

    x, w, b, dy = _case((2, 16, side, side), torch.float32, 4)
    full = _run(x, 4, w, b, dy, "silu")[1]
    for i in range(3):
        args = [x, w, b]
        args[i] = args[i].detach().requires_grad_()
        got, = torch.autograd.grad(group_norm_act(args[0], 4, args[1], args[2], activation="silu"),
                                   args[i], dy)
        assert torch.equal(got, full[i])


def test_gradient_matches_differences():
    x, w, b, dy = _case((1, 4, 3, 5), torch.float32, 2, seed=9)
    _, grads = _run(x, 2, w, b, dy, "gelu")
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).cuda()
    h = 1e-4
    up, down = (ops.group_norm(x.double() + s * h * d.double(), 2, w, b, 1e-5, "gelu")[0]
                for s in (1, -1))
    want = ((up - down) * dy.double()).sum() / (2 * h)
    # differences: h^2 times a third derivative of order 10
    assert abs((grads[0].double() * d).sum() - want) < 1e-5 * (1 + abs(want))


def test_same_bits_every_time_and_on_other_streams():
    from dynamicconvolutionoperator_b200 import group_norm_act

    x, w, b, dy = _case((4, 64, 96, 96), torch.bfloat16, 8)
    xa = x.detach().requires_grad_()
    wa = w.detach().requires_grad_()

    def once():
        out = group_norm_act(xa, 8, wa, b, activation="silu")
        return (out.detach(), *torch.autograd.grad(out, (xa, wa), dy))

    want = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for _ in range(5):
        for s in streams:  # calls of several streams in flight at once
            with torch.cuda.stream(s):
                results.append(once())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, e) for a, e in zip(got, want))


@pytest.mark.parametrize("shape", [(4, 64, 96, 96), (3, 63, 96, 96), (3, 60, 20, 20)])
def test_calls_of_one_stream_overlap_with_another_kernels(shape):
    """Blocks that wait for one another beside other work on the device."""
    from dynamicconvolutionoperator_b200 import group_norm_act, linear_act

    x, w, b, _ = _case(shape, torch.float16, 3 if shape[1] % 3 == 0 else 4)
    groups = 3 if shape[1] % 3 == 0 else 4
    want = group_norm_act(x, groups, w, b)
    a, wa = (torch.randn(4096, 512, device="cuda").bfloat16() for _ in range(2))
    other = linear_act(a, wa)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            outs.append((group_norm_act(x, groups, w, b), want))
        with torch.cuda.stream(s2):
            outs.append((linear_act(a, wa), other))
    torch.cuda.synchronize()
    assert all(torch.equal(g, e) for g, e in outs)


def test_more_values_than_32_bits_count():
    from dynamicconvolutionoperator_b200 import group_norm_act

    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    x = torch.randn(36, 1000, 1000, 64, device="cuda", dtype=torch.bfloat16).permute(0, 3, 1, 2)
    assert x.numel() > 2 ** 31
    xa = x.requires_grad_()
    out = group_norm_act(xa, 8, activation="silu")
    last = x[-1:].detach().requires_grad_()
    want = group_norm_act(last, 8, activation="silu")
    # the same sums in other chunks: the last digit of the rounding may differ
    torch.testing.assert_close(out[-1:], want, rtol=2 ** -7, atol=1e-5)
    dy = torch.randn_like(last)
    g = torch.zeros_like(x)
    g[-1:] = dy
    gx, = torch.autograd.grad(out, xa, g)
    gl, = torch.autograd.grad(want, last, dy)
    torch.testing.assert_close(gx[-1:], gl, rtol=2 ** -7, atol=1e-5)
    assert not gx[0].any()


def test_second_derivative_is_refused():
    from dynamicconvolutionoperator_b200 import group_norm_act

    x = torch.randn(2, 8, 4, 4, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(group_norm_act(x, 2).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|not require grad"):
        g.sum().backward()


@pytest.mark.parametrize("shape", [(2, 64, 64, 64), (2, 64, 200, 200), (2, 63, 200, 200)])
def test_captured_and_replayed(shape):
    """A kernel of each kind: clusters, the ring, blocks that wait for one another."""
    from dynamicconvolutionoperator_b200 import group_norm_act

    groups = 8 if shape[1] == 64 else 7
    x, w, b, dy = _case(shape, torch.bfloat16, groups)
    xa, wa, ba = (t.clone().requires_grad_() for t in (x, w, b))

    def once():
        out = group_norm_act(xa, groups, wa, ba, activation="silu")
        return [out.detach(), *torch.autograd.grad(out, (xa, wa, ba), dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for seed in (1, 2):
        x2 = _case(shape, torch.bfloat16, groups, seed=seed)[0]
        with torch.no_grad():
            xa.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        want = once()
        assert all(torch.equal(a, e) for a, e in zip(held, want))


def test_nan_stays_in_its_group():
    from dynamicconvolutionoperator_b200 import group_norm_act

    x, w, b, _ = _case((2, 8, 6, 6), torch.float32, 2)
    want = group_norm_act(x, 2, w, b, activation="relu")
    x[0, 1, 2, 3] = float("nan")
    x[1, 6, 0, 0] = float("inf")
    got = group_norm_act(x, 2, w, b, activation="relu")
    assert got[0, :4].isnan().all() and got[1, 4:].isnan().all()
    assert torch.equal(got[0, 4:], want[0, 4:]) and torch.equal(got[1, :4], want[1, :4])


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(requires_grad):
    from torch.autograd import forward_ad

    from dynamicconvolutionoperator_b200 import group_norm_act

    x = torch.randn(2, 8, 4, 4, device="cuda", requires_grad=requires_grad)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            group_norm_act(forward_ad.make_dual(x, torch.ones_like(x)), 2)
        if requires_grad:  # forward over reverse
            out = group_norm_act(x, 2)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, forward_ad.make_dual(torch.ones_like(x), x.detach()))


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("shape,groups", [
    ((5000, 64, 4, 4), 8),     # many small samples
    ((70_000, 64), 8),
    ((2000, 24, 7, 9), 3),
    ((129, 64, 32, 32), 8),    # clusters of fewer blocks than eight
    ((300, 64, 48, 48), 8),    # the ring: more samples than blocks
    ((1, 64, 100, 103), 8),    # and one small sample
    ((2, 512, 33, 32), 32),
])
def test_small_and_many_samples(shape, groups, dtype):
    x, w, b, dy = _case(shape, dtype, groups, seed=15)
    _run(x, groups, w, b, dy, "silu", steps=256)
