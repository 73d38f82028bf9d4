"""The DDPM with its optional head (group norm + activation, dropout, 1x1
projection, residual) against the float64 oracle with the same head, and the
parts of the head called one after the other."""

from __future__ import annotations

import pytest
import torch

from oracle import ddpm_oracle as orc
from tests import _operators as ops
from tests._parity import compare

pytestmark = pytest.mark.gpu

HEADS = [
    dict(norm_groups=4, activation="silu"),
    dict(norm_groups=2, activation="gelu", dropout=0.25, out_dim=16, residual=True),
    dict(dropout=0.5, residual=True),
    dict(out_dim=24),
    dict(residual=True),
]


def _gold(m, ref, x, y, grad, seed):
    """Output and gradients in float64 on the CPU."""
    ref = ref.double()
    head = {n: p.detach().double().cpu().requires_grad_() for n, p in m.named_parameters()
            if n.startswith(("norm.", "project."))}
    xd, yd = x.double().requires_grad_(), y.double().requires_grad_()
    out = ref(xd, yd)
    if m.norm is not None:
        out = torch.nn.functional.group_norm(out, m.norm.num_groups, head["norm.weight"],
                                             head["norm.bias"], m.norm.eps)
        out = ops.act(out, m.activation)
    if m.dropout and m.training:
        cl = out.permute(0, 2, 3, 1)
        mask = ops.kept(cl.numel(), m.dropout, seed, 0).view(cl.shape)
        out = torch.where(mask, cl / (1 - m.dropout), torch.zeros_like(cl)).permute(0, 3, 1, 2)
    if m.project is not None:
        out = torch.nn.functional.conv2d(out, head["project.weight"], head["project.bias"])
    if m.residual:
        out = out + xd
    leaves = {"x": xd, "y": yd, **dict(ref.named_parameters()), **head}
    grads = torch.autograd.grad(out, list(leaves.values()), grad.double())
    return out.detach(), dict(zip(leaves, grads))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("head", HEADS)
def test_matches_float64(head, dtype):
    from dynamicconvolutionoperator_b200 import DDPM, _lib

    seed = 1234
    ref = orc.make_model(16, 3, dtype=dtype, seed=3)
    m = DDPM(16, 3, **head)
    m.load_state_dict(ref.state_dict(), strict=False)
    if m.norm is not None:
        torch.nn.init.uniform_(m.norm.weight, 0.5, 1.5)
        torch.nn.init.uniform_(m.norm.bias, -0.5, 0.5)
    m = m.cuda().to(dtype)
    shape = (2, 16, 11, 13)
    x, y, _ = orc.make_inputs(shape, dtype=dtype, seed=5)
    oc = head.get("out_dim") or 16
    grad = torch.randn((2, oc, 11, 13), generator=torch.Generator().manual_seed(6)).to(dtype)
    xd, yd = (t.cuda().requires_grad_() for t in (x, y))
    out = m(xd, yd, seed=seed)
    assert out.shape == grad.shape
    named = dict(m.named_parameters())
    got = torch.autograd.grad(out, [xd, yd, *named.values()], grad.cuda())
    got = {k: v.cpu() for k, v in zip(["x", "y", *named], got)}
    gold, want = _gold(m, ref, x, y, grad, seed)
    stats, fails = compare(out.detach().cpu(), got, gold, want, dtype)
    assert not fails, "\n".join(fails) + f"\n{stats}"
    assert _lib.device_status() == 0


def test_without_a_head_nothing_changes():
    from dynamicconvolutionoperator_b200 import DDPM

    m = DDPM(16, 3).cuda()
    assert set(m.state_dict()) == {"generator.weight", "generator.bias", "fuse.weight", "fuse.bias"}
    x, y = torch.randn(2, 2, 16, 9, 10, device="cuda")
    assert torch.equal(m(x, y), m._body(x, y))


def test_head_is_its_operators_in_a_row():
    from dynamicconvolutionoperator_b200 import DDPM, dropout, group_norm_act, linear_act

    m = DDPM(16, 3, norm_groups=4, activation="gelu", dropout=0.3, out_dim=16, residual=True).cuda()
    x, y = torch.randn(2, 2, 16, 20, 24, device="cuda")
    body = m._body(x, y)
    z = group_norm_act(body, 4, m.norm.weight, m.norm.bias, m.norm.eps, activation="gelu")
    z = dropout(z.permute(0, 2, 3, 1), 0.3, 99)
    z = linear_act(z, m.project.weight, m.project.bias, residual=x.permute(0, 2, 3, 1))
    assert torch.equal(m(x, y, seed=99), z.permute(0, 3, 1, 2))
    m.eval()
    assert torch.equal(m(x, y, seed=1), m(x, y, seed=2))


def test_drawn_seeds_follow_the_default_generator():
    from dynamicconvolutionoperator_b200 import DDPM

    m = DDPM(16, 3, dropout=0.5).cuda()
    x, y = torch.randn(2, 1, 16, 8, 8, device="cuda")
    torch.manual_seed(5)
    a, b = m(x, y), m(x, y)
    torch.manual_seed(5)
    assert torch.equal(m(x, y), a) and not torch.equal(a, b)


def test_autocast_runs_the_head_in_the_autocast_type():
    from dynamicconvolutionoperator_b200 import DDPM

    m = DDPM(16, 3, norm_groups=4, activation="silu", out_dim=8).cuda()
    x, y = torch.randn(2, 1, 16, 12, 16, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = m(x, y)
    assert out.dtype == torch.bfloat16
    out.float().square().mean().backward()
    for p in m.parameters():
        assert p.grad is not None and p.grad.dtype == torch.float32 and p.grad.isfinite().all()


def test_training_step_with_the_head_captured_and_replayed():
    from dynamicconvolutionoperator_b200 import DDPM

    m = DDPM(16, 3, norm_groups=4, activation="silu", dropout=0.2, out_dim=16, residual=True,
             fused_generator_training=True).cuda().to(torch.bfloat16)
    x, y, g = torch.randn(3, 2, 16, 16, 24, device="cuda").to(torch.bfloat16)
    seed = torch.tensor([7], device="cuda")
    params = list(m.parameters())

    def once():
        out = m(x, y, seed=seed)
        return [out.detach(), *torch.autograd.grad(out, params, g)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for value in (7, 8):
        seed.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        # the generator's backward adds with FP32 atomics, whose order is free
        for a, b in zip(held, once()):
            scale = b.float().abs().max() + 1e-6
            assert ((a.float() - b.float()).abs().max() / scale).item() < 2e-2
        assert torch.equal(held[0], m(x, y, seed=seed))
    with pytest.raises(RuntimeError, match="seed"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            m(x, y)


def test_tracing_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx

    from dynamicconvolutionoperator_b200 import DDPM, linear_act

    x, y = torch.randn(2, 1, 16, 9, 10, device="cuda")
    m = DDPM(16, 3, norm_groups=4, activation="silu", out_dim=8).cuda().eval()
    with torch.no_grad(), pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(m, (x, y), check_trace=False)
    # a backward on its own
    a, w = torch.randn(2, 12, 12, device="cuda", requires_grad=True)
    out = linear_act(a, w, None, "silu")
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda g: torch.autograd.grad(out, a, g))(torch.ones_like(out))


def _head_of(dtype=torch.float32, **kwargs):
    from dynamicconvolutionoperator_b200 import DDPM

    m = DDPM(16, 3, norm_groups=4, activation="silu", out_dim=16, residual=True, **kwargs).cuda()
    x, y = torch.randn(2, 2, 16, 10, 12, device="cuda").to(dtype)
    return m.to(dtype), x, y


def test_hooks_of_the_heads_layers_run():
    m, x, y = _head_of()
    want = m(x, y)
    seen = []
    for name in ("norm", "project"):
        layer = getattr(m, name)
        layer.register_forward_pre_hook(lambda mod, args, name=name: seen.append(name))
        layer.register_forward_hook(lambda mod, args, out, name=name: seen.append((name, out)))
    got = m(x, y)
    assert [s if isinstance(s, str) else s[0] for s in seen] == ["norm", "norm", "project", "project"]
    body = m._body(x, y)
    z = m.project(torch.nn.functional.silu(m.norm(body)))
    assert torch.equal(got, z + x)
    # the library's convolution may round its operands to TF32 (2^-11 each)
    assert (got - want).abs().max() < 2 ** -9 * want.abs().max()
    # hooks that make the weight: a step on their parameters reaches the result
    m, x, y = _head_of()
    torch.nn.utils.weight_norm(m.project)
    before = m(x, y) - x
    with torch.no_grad():
        m.project.weight_g.mul_(2)
        m.project.bias.mul_(2)
    assert ((m(x, y) - x) - 2 * before).abs().max() < 2 ** -9 * before.abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layers_without_parameters_of_their_own(dtype):
    from dynamicconvolutionoperator_b200 import group_norm_act, linear_act

    m, x, y = _head_of(dtype)
    m.norm = torch.nn.GroupNorm(4, 16, affine=False)
    m.project = torch.nn.Conv2d(16, 16, 1, bias=False).cuda().to(dtype)
    z = group_norm_act(m._body(x, y), 4, activation="silu").permute(0, 2, 3, 1)
    want = linear_act(z, m.project.weight, residual=x.permute(0, 2, 3, 1)).permute(0, 3, 1, 2)
    assert torch.equal(m(x, y), want)


@pytest.mark.parametrize("layer", [
    lambda: torch.nn.Conv2d(16, 8, 1, stride=2),
    lambda: torch.nn.Conv2d(16, 8, 3, padding=1),
    lambda: torch.nn.Conv2d(16, 8, 1, groups=4),
    lambda: torch.nn.Conv2d(16, 8, 1, padding=1),
    lambda: torch.nn.Sequential(torch.nn.Conv2d(16, 8, 1), torch.nn.ReLU()),
])
def test_replaced_projections_run_their_own_forward(layer):
    m, x, y = _head_of()
    m.residual, m.project = False, layer().cuda()
    m.norm = torch.nn.BatchNorm2d(16).cuda().eval()
    want = m.project(torch.nn.functional.silu(m.norm(m._body(x, y))))
    got = m(x, y)
    assert got.shape == want.shape and torch.equal(got, want)
    # FP32 layers behind a 16-bit body
    m.generator.bfloat16(), m.fuse.bfloat16()
    out = m(x.bfloat16(), y.bfloat16())
    assert out.dtype == torch.bfloat16 and out.shape == want.shape
    with torch.autocast("cuda", dtype=torch.float16):
        assert m.float()(x, y).dtype == torch.float16


def test_shards_draw_the_whole_batchs_mask():
    from dynamicconvolutionoperator_b200 import DDPM

    m = DDPM(16, 3, norm_groups=4, dropout=0.5).cuda()
    x, y = torch.randn(2, 4, 16, 9, 7, device="cuda")
    whole = m(x, y, seed=3) != 0
    for first, last in ((0, 1), (1, 4)):
        part = m(x[first:last], y[first:last], seed=3, offset=first * 9 * 7 * 16)
        assert torch.equal(part != 0, whole[first:last])
    assert not torch.equal(m(x[1:], y[1:], seed=3) != 0, whole[1:])


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("head", HEADS)
def test_memory_of_the_output(head, training):
    from dynamicconvolutionoperator_b200 import DDPM

    m = DDPM(16, 3, **head).cuda().train(training)
    x, y = torch.randn(2, 2, 16, 9, 7, device="cuda")
    wrote = "norm_groups" in head or "out_dim" in head or ("dropout" in head and training)
    assert m(x, y, seed=1).is_contiguous(memory_format=torch.channels_last) == wrote
