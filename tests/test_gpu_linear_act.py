"""linear_act against a float64 form: values, gradients, ragged sizes, strides,
alignment, streams, graphs."""

from __future__ import annotations

import pytest
import torch

from tests import _operators as ops

pytestmark = pytest.mark.gpu

SHAPES = [  # m, n, k
    (1, 1, 1), (1, 5, 3), (2, 40, 1000), (4, 130, 64), (8, 100, 72), (5, 9, 7),  # dot products
    (9, 1, 1), (9, 64, 64), (17, 333, 200), (128, 64, 256), (129, 257, 65),
    (300, 1728, 64), (130, 24, 1100), (2049, 128, 8), (1000, 255, 16), (77, 72, 2048),
    (4000, 3, 5), (640, 512, 512),
]


def _case(m, n, k, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    return (normal(m, k).to(dtype), (normal(n, k) / k ** 0.5).to(dtype), (0.3 * normal(n)).to(dtype),
            normal(m, n).to(dtype), normal(m, n).to(dtype))


def _steps(terms, dtype):
    """FP32 roundings of a sum of ``terms`` products, none kinder than a
    truncation (two half steps): one per 16 products and bf16 part product, the
    epilogue's and the split's partial sums, and for FP32 data the products of
    parts that are left out (below 4 * 2^-24 of the product)."""
    return 2 * ((6 if dtype == torch.float32 else 1) * (terms / 16 + 1) + 16) + 8


def _run(x, w, b, res, dy, name):
    from dynamicconvolutionoperator_b200 import _lib, linear_act

    dt = x.dtype
    m, k = x.shape
    n = w.shape[0]
    given = {"x": x, "weight": w, "bias": b, "residual": res}
    leaf = {i: None if t is None else t.detach().requires_grad_() for i, t in given.items()}
    out = linear_act(leaf["x"], leaf["weight"], leaf["bias"], name, leaf["residual"])
    ref, scale, zscale, grads = ops.linear(x, w, b, name, res, dy)
    ops.check("out", out.detach(), ref, ops.bound(ref, scale, _steps(k, dt), dt))
    with torch.no_grad():
        assert torch.equal(linear_act(x, w, b, name, res), out)
    names = [i for i, t in leaf.items() if t is not None]
    got = dict(zip(names, torch.autograd.grad(out, [leaf[i] for i in names], dy)))
    if res is not None:
        assert torch.equal(got["residual"], dy)
    half = torch.finfo(dt).eps / 2
    for i, terms in (("x", n), ("weight", m), ("bias", m)):
        if i not in got:
            continue
        r, s, rounded = grads[i]
        # dz's own error: its product over k terms; for 16-bit data its rounding
        tol = ops.bound(r, s, _steps(terms, dt) + _steps(k, dt), dt)
        if dt != torch.float32:
            tol = tol + half * rounded * (1 + half)
            # products of fp16's smallest dz values: below the type's normal
            # range a rounding is absolute
            tol = tol + torch.finfo(dt).tiny * half * terms * 8
        ops.check(i, got[i], r, tol)
    assert _lib.device_status() == 0
    return out, got


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matches_float64(m, n, k, dtype):
    x, w, b, res, dy = _case(m, n, k, dtype)
    _run(x, w, b, res, dy, "silu")
    _run(x, w, b, None, dy, None)


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("name", ops.ACTS)
@pytest.mark.parametrize("m", [3, 200])
def test_activations(m, name, dtype):
    x, w, b, res, dy = _case(m, 96, 80, dtype, seed=2)
    if name == "relu":  # away from the kink, where a rounding turns the slope
        z = ops.linear(x, w, b, None, None)[0]
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    _run(x, w, b, res, dy, name)
    _run(x, w, None, None, dy, name)


@pytest.mark.parametrize("dtype", ops.DTYPES)
def test_long_sums(dtype):
    """Many rows (the weight gradient's axis, split over the SMs) and long rows."""
    _run(*_case(40_000, 64, 72, dtype, seed=4), "gelu")
    _run(*_case(200, 72, 6000, dtype, seed=5), "gelu")


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("m,n,k", [(5000, 1500, 300), (2600, 2049, 96), (20_000, 256, 264)])
def test_several_tiles_a_block(m, n, k, dtype):
    """Tiles of pairs of blocks, blocks with several tiles, ragged last tiles."""
    x, w, b, res, dy = _case(m, n, k, dtype, seed=8)
    _run(x, w, b, res, dy, "gelu")
    _run(x, w, None, None, dy, None)


def test_float32_keeps_its_digits():
    """The 2-norm of the error stays near a single-precision product's, not at
    the 2^-17 of two bf16 parts."""
    x, w, b, res, dy = _case(2048, 256, 1024, torch.float32)
    out, got = _run(x, w, b, res, dy, None)
    ref, _, _, grads = ops.linear(x, w, b, None, res, dy)
    for name, a, e in [("out", out, ref)] + [(i, got[i], grads[i][0]) for i in ("x", "weight")]:
        rel = ((a.double() - e).norm() / e.norm()).item()
        assert rel < 1e-6, (name, rel)


def test_float32_range():
    """Values near the type's limits split without overflow."""
    from dynamicconvolutionoperator_b200 import linear_act

    x = torch.full((16, 8), 3.4e38, device="cuda")
    w = torch.zeros(8, 8, device="cuda")
    w.fill_diagonal_(1.0)
    assert torch.equal(linear_act(x, w), x)
    x = torch.full((16, 8), 1.2e-30, device="cuda")
    torch.testing.assert_close(linear_act(x, w), x, rtol=2 ** -22, atol=0)


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("m", [4, 150])
def test_strides_and_alignment(m, dtype):
    from dynamicconvolutionoperator_b200 import linear_act

    x, w, b, res, dy = _case(m, 48, 64, dtype)
    want = linear_act(x, w, b, "silu", res)
    wide = torch.zeros(m, 3, 64, dtype=dtype, device="cuda")
    wide[:, 1] = x
    assert torch.equal(linear_act(wide[:, 1], w, b, "silu", res), want)
    assert torch.equal(linear_act(x.t().contiguous().t(), w, b, "silu", res), want)
    assert torch.equal(linear_act(x, w.t().contiguous().t(), b, "silu", res), want)
    shaped = linear_act(x.view(2, m // 2, 64), w.view(48, 64, 1, 1), b, "silu", res.view(2, m // 2, 48))
    assert torch.equal(shaped.view(m, 48), want)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    ref, scale, _, _ = ops.linear(x, w, b, "silu", res)
    tol = ops.bound(ref, scale, _steps(64, dtype), dtype)
    ops.check("out", linear_act(shifted(x), shifted(w), shifted(b), "silu", shifted(res)), ref, tol)
    if m > 8:
        _run(shifted(x), shifted(w), shifted(b), shifted(res), shifted(dy), "silu")
        _run(wide[:, 1], w, b, None, dy, None)


def test_broadcast_and_shared_inputs():
    from dynamicconvolutionoperator_b200 import linear_act

    x, w, b, res, dy = _case(1, 32, 16, torch.float32)
    xa = x.requires_grad_()
    out = linear_act(xa.expand(40, 16), w, b)
    gx, = torch.autograd.grad(out, xa, torch.ones_like(out))
    torch.testing.assert_close(gx, 40 * w.sum(0, keepdim=True), rtol=1e-5, atol=1e-4)
    # one tensor as x and residual
    sq = torch.randn(40, 16, device="cuda", requires_grad=True)
    wq = torch.randn(16, 16, device="cuda")
    gs, = torch.autograd.grad(linear_act(sq, wq, None, None, sq).sum(), sq)
    torch.testing.assert_close(gs, wq.sum(0) + torch.ones_like(sq), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", ops.DTYPES)
def test_empty_rows(dtype):
    from dynamicconvolutionoperator_b200 import linear_act

    x, w, b, res, _ = _case(0, 8, 16, dtype)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    out = linear_act(x, w, b, "gelu", res)
    assert out.shape == (0, 8)
    gx, gw, gb = torch.autograd.grad(out, (x, w, b), torch.empty_like(out))
    assert gx.shape == x.shape and not gw.any() and not gb.any()


def test_only_the_asked_gradients():
    from dynamicconvolutionoperator_b200 import linear_act

    x, w, b, res, dy = _case(70, 40, 24, torch.bfloat16)
    for name in (None, "silu"):
        full = _run(x, w, b, res, dy, name)[1]
        for i, key in enumerate(("x", "weight", "bias", "residual")):
            args = [x, w, b, res]
            args[i] = args[i].detach().requires_grad_()
            out = linear_act(args[0], args[1], args[2], name, args[3])
            got, = torch.autograd.grad(out, args[i], dy)
            assert torch.equal(got, full[key]), key


def test_gradient_matches_differences():
    x, w, b, res, dy = _case(20, 12, 10, torch.float32, seed=7)
    _, got = _run(x, w, b, res, dy, "gelu")
    g = torch.Generator(device="cuda").manual_seed(1)
    h = 1e-4
    for key, i in (("x", 0), ("weight", 1), ("bias", 2)):
        args = [x, w, b]
        d = torch.randn(args[i].shape, generator=g, device="cuda").double()
        ends = []
        for s in (1, -1):
            moved = [t.double() for t in args]
            moved[i] = moved[i] + s * h * d
            ends.append((ops.linear(*moved, "gelu", res)[0] * dy.double()).sum())
        want = (ends[0] - ends[1]) / (2 * h)
        # h^2 times a third derivative of order 10^2, and FP32 gradients
        assert abs((got[key].double() * d).sum() - want) < 1e-5 * (10 + abs(want))


def test_row_offsets_beyond_32_bits():
    """Rows far apart: the last row's values lie past 2^32 bytes and 2^31 elements."""
    from dynamicconvolutionoperator_b200 import linear_act

    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    ld = 1 << 23
    wide = torch.empty(300 * ld, dtype=torch.bfloat16, device="cuda").view(300, ld)
    x, w, b, _, _ = _case(300, 40, 64, torch.bfloat16)
    wide[:, -64:] = x
    assert torch.equal(linear_act(wide[:, -64:], w, b), linear_act(x, w, b))
    assert torch.equal(linear_act(wide[-4:, -64:], w, b), linear_act(x[-4:], w, b))


def test_same_bits_every_time_and_on_other_streams():
    from dynamicconvolutionoperator_b200 import linear_act

    x, w, b, res, dy = _case(3000, 192, 128, torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]

    def once():
        out = linear_act(*leaves, "silu", res)
        return (out.detach(), *torch.autograd.grad(out, leaves, dy))

    want = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(once())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, e) for a, e in zip(got, want))


def test_calls_from_new_threads():
    """A thread whose first CUDA call is the operator's, once everything that is
    looked up once has been looked up."""
    import threading

    from dynamicconvolutionoperator_b200 import linear_act

    x, w, b, _, _ = _case(300, 64, 64, torch.bfloat16)
    want = linear_act(x, w, b)
    torch.cuda.synchronize()
    got = []
    threads = [threading.Thread(target=lambda: got.append(linear_act(x, w, b))) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(got) == 3 and all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_captured_and_replayed(dtype):
    from dynamicconvolutionoperator_b200 import linear_act

    x, w, b, res, dy = _case(500, 72, 56, dtype)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]

    def once():
        out = linear_act(*leaves, "gelu", res)
        return [out.detach(), *torch.autograd.grad(out, leaves, dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):  # two graphs over the same leaves
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = once()
        graphs.append((graph, held))
    for seed in (1, 2):
        with torch.no_grad():
            leaves[0].copy_(_case(500, 72, 56, dtype, seed=seed)[0])
        for graph, held in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = once()
        for _, held in graphs:
            assert all(torch.equal(a, e) for a, e in zip(held, want))


def test_gradients_land_in_attached_buffers():
    from dynamicconvolutionoperator_b200 import _gradbuf, linear_act

    x, w, b, _, dy = _case(64, 24, 16, torch.float32)
    w, b = torch.nn.Parameter(w.view(24, 16, 1, 1)), torch.nn.Parameter(b)
    flat = torch.zeros(w.numel() + b.numel() + 1, device="cuda")
    views = flat[1:25 * 16 - 15].view(24, 16, 1, 1), flat[25 * 16 - 15:]  # not 16-byte aligned
    for p, v in zip((w, b), views):
        _gradbuf.attach(p, v)
    try:
        linear_act(x, w, b, "silu").backward(dy)
        assert w.grad.data_ptr() == views[0].data_ptr() and b.grad.data_ptr() == views[1].data_ptr()
        ref = ops.linear(x, w.detach().view(24, 16), b.detach(), "silu", None, dy)[3]
        for got, key in ((w.grad.view(24, 16), "weight"), (b.grad, "bias")):
            r, s, _ = ref[key]
            ops.check(key, got, r, ops.bound(r, s, _steps(64, x.dtype) + _steps(16, x.dtype), x.dtype))
    finally:
        _gradbuf.detach(w), _gradbuf.detach(b)


def test_more_outputs_than_32_bits_count():
    from dynamicconvolutionoperator_b200 import linear_act

    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    m = 1 << 20
    x, w, b, _, _ = _case(m, 2056, 16, torch.bfloat16)
    out = linear_act(x, w, b, "silu")
    assert out.numel() > 2 ** 31
    assert torch.equal(out[-300:], linear_act(x[-300:], w, b, "silu"))
    xa = x[-300:].clone().requires_grad_()
    gy = torch.zeros_like(out)
    gy[-300:] = torch.randn(300, 2056, device="cuda").bfloat16()
    xb = x.requires_grad_()
    gx, = torch.autograd.grad(linear_act(xb, w, b, "silu"), xb, gy)
    ga, = torch.autograd.grad(linear_act(xa, w, b, "silu"), xa, gy[-300:])
    assert torch.equal(gx[-300:], ga) and not gx[:1000].any()


def test_vectors_and_batches():
    from dynamicconvolutionoperator_b200 import linear_act

    x, w, b, res, _ = _case(12, 24, 40, torch.float32)
    want = linear_act(x, w, b, "gelu", res)
    got = linear_act(x.view(3, 2, 2, 40), w, b, "gelu", res.view(3, 2, 2, 24))
    assert torch.equal(got.view(12, 24), want)
    v = x[0].clone().requires_grad_()
    out = linear_act(v, w, b)
    assert out.shape == (24,)
    g, = torch.autograd.grad(out.sum(), v)
    torch.testing.assert_close(g, w.sum(0), rtol=1e-5, atol=1e-5)


def test_second_derivative_is_refused():
    from dynamicconvolutionoperator_b200 import linear_act

    x, w, _, _, _ = _case(12, 24, 40, torch.float32)
    x.requires_grad_()
    g, = torch.autograd.grad(linear_act(x, w, None, "silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|not require grad"):
        g.sum().backward()


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(requires_grad):
    from torch.autograd import forward_ad

    from dynamicconvolutionoperator_b200 import linear_act

    x, w, _, _, dy = _case(12, 24, 40, torch.float32)
    x.requires_grad_(requires_grad)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            linear_act(forward_ad.make_dual(x, torch.ones_like(x)), w)
        if requires_grad:  # forward over reverse
            out = linear_act(x, w, None, "silu")
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, forward_ad.make_dual(dy, torch.ones_like(dy)))


@pytest.mark.parametrize("dtype", ops.DTYPES)
@pytest.mark.parametrize("m", [3, 8, 9, 300])
def test_infinities_stay_in_their_row_or_column(m, dtype):
    from dynamicconvolutionoperator_b200 import linear_act

    x, w, b, res, _ = _case(m, 40, 24, dtype)
    want = linear_act(x, w, b, "silu", res)
    x[1, 5], w[7, 3] = float("inf"), float("-inf")
    got = linear_act(x, w, b, "silu", res)
    hit = torch.zeros(m, 40, dtype=torch.bool, device="cuda")
    hit[1], hit[:, 7] = True, True
    assert torch.equal(got[~hit], want[~hit]) and not got[hit].isfinite().all()
    z = linear_act(x, w, b)[1]
    keep = torch.arange(40, device="cuda") != 7
    if dtype == torch.float32 and m > 8:  # three bf16 parts: as documented
        assert z.isnan().all()
    else:
        assert torch.equal(z[keep], float("inf") * w[keep, 5].sign())
