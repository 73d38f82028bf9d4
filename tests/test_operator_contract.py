"""Argument checks of the channel-last operators (CPU: nothing is launched)."""

from __future__ import annotations

import pytest
import torch

from dynamicconvolutionoperator_b200 import _lib, dropout, group_norm_act, linear_act
from tests import _operators as ops


def test_philox_known_answers():
    """The published test vectors of Philox-4x32-10 (Random123 ``kat_vectors``)."""
    assert ops.philox_words([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert ops.philox_words([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [
        0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("call", [
    lambda x: group_norm_act(x, 2),
    lambda x: dropout(x, 0.5, 1),
    lambda x: linear_act(x, torch.randn(5, 3)),
])
def test_cpu_tensors_fail_loudly(call):
    with pytest.raises(RuntimeError, match="CUDA"):
        call(torch.randn(2, 4, 3, 3))


@pytest.mark.parametrize("kwargs,match", [
    (dict(num_groups=3), "num_groups"),
    (dict(num_groups=0), "num_groups"),
    (dict(num_groups=2, activation="tanh"), "activation"),
    (dict(num_groups=2, activation=["relu"]), "activation"),
    (dict(num_groups=2, eps=-1.0), "eps"),
    (dict(num_groups=2, eps=float("nan")), "eps"),
    (dict(num_groups=2, weight=torch.ones(3)), "weight must have shape"),
    (dict(num_groups=2, bias=torch.ones(1, 4)), "bias must have shape"),
    (dict(num_groups=2, weight=torch.ones(4, dtype=torch.float64)), "dtype"),
    (dict(num_groups=2, weight=torch.ones(4, dtype=torch.bfloat16)), "dtype"),
])
def test_group_norm_refusals(kwargs, match):
    with pytest.raises(ValueError, match=match):
        group_norm_act(torch.randn(2, 4, 3, 3), **kwargs)


def test_group_norm_refuses_one_dimension_and_mixed_parameters():
    with pytest.raises(ValueError, match="two dimensions"):
        group_norm_act(torch.randn(4), 1)
    with pytest.raises(ValueError, match="one dtype"):
        group_norm_act(torch.randn(2, 4).bfloat16(), 1, torch.ones(4), torch.ones(4).bfloat16())


@pytest.mark.parametrize("kwargs,match", [
    (dict(p=-0.1, seed=1), "between 0 and 1"),
    (dict(p=1.5, seed=1), "between 0 and 1"),
    (dict(p=float("nan"), seed=1), "between 0 and 1"),
    (dict(p=0.5, seed=1 << 64), "64 bits"),
    (dict(p=0.5, seed=torch.tensor([1, 2])), "one int64"),
    (dict(p=0.5, seed=torch.tensor([1], dtype=torch.int32)), "one int64"),
    (dict(p=0.5, seed=1, offset=-1), "offset"),
    (dict(p=0.5, seed=1, offset=1 << 64), "offset"),
    (dict(p=0.5, seed=1, residual=torch.zeros(5)), "residual"),
    (dict(p=0.5, seed=1, residual=torch.zeros(4, dtype=torch.float16)), "residual"),
])
def test_dropout_refusals(kwargs, match):
    with pytest.raises(ValueError, match=match):
        dropout(torch.randn(4), **kwargs)


@pytest.mark.parametrize("kwargs,match", [
    (dict(weight=torch.ones(5, 4)), "weight must be"),
    (dict(weight=torch.ones(3)), "weight must be"),
    (dict(weight=torch.ones(5, 3, 3, 3)), "weight must be"),
    (dict(weight=torch.ones(0, 3)), "empty"),
    (dict(weight=torch.ones(5, 3), bias=torch.ones(3)), "bias must have shape"),
    (dict(weight=torch.ones(5, 3), residual=torch.ones(2, 3)), "residual must have shape"),
    (dict(weight=torch.ones(5, 3), residual=torch.ones(5)), "residual must have shape"),
    (dict(weight=torch.ones(5, 3).half()), "one dtype"),
    (dict(weight=torch.ones(5, 3), bias=torch.ones(5).half()), "one dtype"),
    (dict(weight=torch.ones(5, 3), activation="swish"), "activation"),
])
def test_linear_refusals(kwargs, match):
    with pytest.raises(ValueError, match=match):
        linear_act(torch.randn(2, 3), **kwargs)


def test_linear_abi_argument_errors_without_gpu():
    lib = _lib.load()

    def fwd(m=64, n=8, k=8, ldx=8, act=0, dt=1, x=16, ws=256, nbytes=1 << 20):
        return lib.ddpm_linear_fwd(x, ldx, 16, None, None, 16, ws, nbytes, m, n, k, act, dt, None)

    assert fwd(ldx=7) == -1 and b"stride" in lib.ddpm_last_error()
    assert fwd(n=0) == -1 and fwd(k=0) == -1 and fwd(m=-1) == -1
    assert fwd(act=9) == -1 and b"activation" in lib.ddpm_last_error()
    assert fwd(dt=3) == -1 and b"dtype" in lib.ddpm_last_error()
    assert fwd(x=None) == -1 and b"null" in lib.ddpm_last_error()
    assert fwd(x=17) == -1 and b"misaligned" in lib.ddpm_last_error()
    assert fwd(ws=8) == -1 and b"workspace" in lib.ddpm_last_error()
    assert fwd(dt=0, x=20, nbytes=64) == -4 and b"workspace" in lib.ddpm_last_error()
    assert fwd(x=18, nbytes=64) == -4  # rows that TMA cannot address are copied
    assert fwd(m=1 << 33) == -2
    assert fwd(m=0) == 0
    size = lib.ddpm_linear_workspace_bytes
    assert size(64, 8, 8, 8, 0, 1, 0, 1) == 0 and size(64, 8, 8, 8, 0, 1, 0, 0) > 0
    assert size(64, 8, 8, 7, 0, 1, 0, 1) == 0  # refused shapes
    for bwd in (0, 1):
        for act in (0, 2):
            for dt in (0, 1, 2):
                assert size(1999, 333, 200, 200, act, dt, bwd, 0) >= size(
                    1999, 333, 200, 200, act, dt, bwd, 1)


def test_abi_argument_errors_without_gpu():
    lib = _lib.load()

    def norm(n=1, px=4, c=8, g=2, act=0, dt=0, pdt=0, x=16, ws=256, nbytes=1 << 20):
        return lib.ddpm_group_norm_fwd(x, None, None, 16, 16, ws, nbytes, n, px, c, g, 1e-5, act,
                                       dt, pdt, None)

    assert norm(g=3) == -1 and b"num_groups" in lib.ddpm_last_error()
    assert norm(dt=7) == -1 and b"dtype" in lib.ddpm_last_error()
    assert norm(act=5) == -1 and b"activation" in lib.ddpm_last_error()
    assert norm(dt=1, pdt=2) == -1 and b"fp32" in lib.ddpm_last_error()
    assert norm(x=None) == -1 and b"null" in lib.ddpm_last_error()
    assert norm(x=18) == -1 and b"misaligned" in lib.ddpm_last_error()
    assert norm(ws=128) == -1 and b"misaligned" in lib.ddpm_last_error()
    assert norm(px=1 << 20, nbytes=16) == -4 and b"workspace" in lib.ddpm_last_error()
    assert norm(px=1 << 20, ws=None) == -4
    assert norm(c=1 << 17) == -2
    assert norm(n=0) == 0 and norm(px=0) == 0

    def drop(n=8, p=0.5, dt=0, x=16, seed=None):
        return lib.ddpm_dropout(x, None, 16, n, p, 1, seed, 0, dt, None)

    assert drop(p=2.0) == -1 and b"between" in lib.ddpm_last_error()
    assert drop(dt=9) == -1 and b"dtype" in lib.ddpm_last_error()
    assert drop(x=None) == -1 and b"null" in lib.ddpm_last_error()
    assert drop(x=17) == -1 and b"misaligned" in lib.ddpm_last_error()
    assert drop(seed=4) == -1 and b"misaligned" in lib.ddpm_last_error()
    assert drop(n=-1) == -1 and drop(n=0) == 0


@pytest.mark.parametrize("bwd", [0, 1])
def test_group_norm_workspace_covers_every_alignment(bwd):
    lib = _lib.load()
    size = lib.ddpm_group_norm_workspace_bytes
    assert size(0, 4, 8, 2, 0, bwd, 0) == 0 and size(4, 4, 9, 2, 0, bwd, 0) == 0
    for c, g in ((64, 8), (60, 5), (515, 5), (4096, 32)):
        for n, px in ((3, 1000), (5, 100_000)):
            assert size(n, px, c, g, 1, bwd, 0) >= size(n, px, c, g, 1, bwd, 1)
        assert size(5, 100_000, c, g, 1, bwd, 1) > 0


@pytest.mark.parametrize("kwargs,match", [
    (dict(norm_groups=3), "norm_groups"),
    (dict(norm_groups=0), "norm_groups"),
    (dict(activation="relu"), "needs norm_groups"),
    (dict(norm_groups=2, activation="swish"), "activation"),
    (dict(dropout=1.5), "dropout"),
    (dict(out_dim=0), "out_dim"),
    (dict(out_dim=5, residual=True), "residual"),
])
def test_ddpm_head_refusals(kwargs, match):
    from dynamicconvolutionoperator_b200 import DDPM

    with pytest.raises(ValueError, match=match):
        DDPM(4, 3, **kwargs)


def _calls():
    """Every operator as a function of one argument that may carry a derivative."""
    x, w, v = torch.randn(2, 4, 3, 3), torch.randn(5, 3), torch.randn(4)
    return {
        "norm x": (lambda t: group_norm_act(t, 2), x),
        "norm weight": (lambda t: group_norm_act(x, 2, t), v),
        "norm bias": (lambda t: group_norm_act(x, 2, None, t), v),
        "linear x": (lambda t: linear_act(t, w), x),
        "linear weight": (lambda t: linear_act(x, t), w),
        "linear bias": (lambda t: linear_act(x, w, t), torch.randn(5)),
        "linear residual": (lambda t: linear_act(x, w, None, "relu", t), torch.randn(2, 4, 3, 5)),
        "dropout x": (lambda t: dropout(t, 0.5, 1), x),
        "dropout residual": (lambda t: dropout(x, 0.5, 1, residual=t), x),
    }


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name", list(_calls()))
def test_forward_mode_derivatives_are_refused(name, requires_grad):
    """An output without a tangent would pass for one with a zero derivative."""
    from torch.autograd import forward_ad

    call, t = _calls()[name]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t.requires_grad_(requires_grad), torch.ones_like(t))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            call(dual)


def _jit(call, t):
    torch.jit.trace(call, (t,), check_trace=False)


def _fx(call, t):
    from torch.fx.experimental.proxy_tensor import make_fx

    make_fx(call)(t)


def _fake(call, t):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=True):
        call(torch.empty(t.shape))


@pytest.mark.parametrize("tracer", [_jit, _fx, _fake])
@pytest.mark.parametrize("name", ["norm x", "linear x", "dropout x"])
def test_tracing_is_refused(name, tracer):
    """A trace would hold the output's allocation without the kernel."""
    with pytest.raises(RuntimeError, match="cannot be traced"):
        tracer(*_calls()[name])


def test_dropout_positions_past_64_bits_are_refused():
    """The generator's counter would leave the 2^64 positions that a seed has."""
    x, most = torch.randn(8), (1 << 64) - 1
    for offset in (most, most - 6):
        with pytest.raises(ValueError, match="fit 64 bits"):
            dropout(x, 0.5, 1, offset)
    for offset in (most - 7, 0):
        with pytest.raises(RuntimeError, match="CUDA"):
            dropout(x, 0.5, 1, offset)
    with pytest.raises(RuntimeError, match="CUDA"):
        dropout(x[:0], 0.5, 1, most)
    lib = _lib.load()
    assert lib.ddpm_dropout(16, None, 16, 8, 0.5, 1, None, most - 6, 0, None) == -1
    assert b"64 bits" in lib.ddpm_last_error()


@pytest.mark.parametrize("channels", [65544, 2 ** 31, 2 ** 32 + 8])
def test_too_many_channels_are_refused(channels):
    """2^32 + 8 channels must not pass for 8."""
    x = torch.zeros(1).expand(1, channels)
    with pytest.raises(RuntimeError, match="C <= 65536"):
        group_norm_act(x, 8)
    with pytest.raises(RuntimeError, match="C <= 65536"):
        group_norm_act(x[..., None].requires_grad_(), channels)


@pytest.mark.parametrize("dtype", ops.DTYPES)
def test_every_product_has_a_ring_of_two_stages(dtype):
    """With one stage a copy would wait for the product before it."""
    sizes = (1, 16, 64, 200, 512, 1024, 4000, 19_000, 25_600, 40_000, 300_000)
    seen = set()
    for m in sizes:
        for n in sizes:
            for k in sizes:
                for product in ("forward", "x", "weight"):
                    bn, cg, ew, splits, stages, fits = ops.linear_choice(m, n, k, dtype, product)
                    assert stages >= 2 and fits and splits >= 1, (m, n, k, product)
                    seen.add((bn, cg, ew))
    # 16 epilogue warps for a short K loop only
    assert ops.linear_choice(65536, 1728, 256, torch.bfloat16, "forward")[:3] == (256, 2, 16)
    assert ops.linear_choice(65536, 1728, 320, torch.bfloat16, "forward")[:3] == (256, 2, 8)
    assert seen == ({(64, 1, 8), (128, 1, 8)} if dtype == torch.float32 else
                    {(64, 1, 8), (128, 1, 8), (256, 1, 8), (256, 2, 8), (256, 2, 16)})


def test_modules_pickled_without_a_head_load():
    import pickle

    from dynamicconvolutionoperator_b200 import DDPM

    m = DDPM(4, 3)
    for name in ("norm", "project", "activation", "dropout", "residual"):
        del m.__dict__[name]
    old = pickle.loads(pickle.dumps(m))
    old._body = lambda x, y: x + y
    x = torch.ones(1, 4, 2, 2)
    assert torch.equal(old(x, x), 2 * x)
    assert set(old.state_dict()) == set(m.state_dict())
    new = pickle.loads(pickle.dumps(DDPM(4, 3, norm_groups=2, activation="silu", out_dim=4)))
    assert new.norm.num_groups == 2 and new.project.out_channels == 4 and new.activation == "silu"


def test_another_torch_builds_the_operators_again(tmp_path, monkeypatch):
    """_operators.so fits one torch; file times do not show a change of it."""
    import subprocess

    from dynamicconvolutionoperator_b200 import _build

    made = []

    def run(cmd, **kwargs):
        out = _build.Path(cmd[cmd.index("-o") + 1])
        out.write_text("")
        made.append(out.name)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(_build.subprocess, "run", run)
    monkeypatch.setattr(_build, "BUILD_DIR", tmp_path)
    monkeypatch.setattr(_build, "OPERATORS_PATH", tmp_path / "_operators.so")

    def build():
        made.clear()
        _build._build_operators(False, False)
        return list(made)

    assert build() == ["operators.o", "_operators.so.tmp"]
    assert build() == []
    monkeypatch.setattr(torch, "__version__", "0.0.0")
    assert build() == ["operators.o", "_operators.so.tmp"]
    assert build() == []


def test_each_wait_of_the_operators_has_its_own_status_code():
    """A code names the wait that ran out, so no two kernels may record the same one."""
    import re
    from collections import Counter

    from dynamicconvolutionoperator_b200 import _build

    codes = Counter()
    for name in ("groupnorm.cu", "linear.cu"):
        text = (_build.CSRC / name).read_text()
        codes.update(re.findall(r"(?:fail\(|status, 0, |p\.status, )(\d+)\)", text))
    assert len(codes) == 13 and max(codes.values()) == 1, codes


def test_small_samples_need_no_workspace_however_many_there_are():
    """They go to the kernel without counters in global memory: a step of the other
    ones costs a microsecond however little it holds."""
    size = _lib.load().ddpm_group_norm_workspace_bytes
    for n, pixels, c in ((16_357, 64, 64), (1_000_000, 1, 64), (129, 1024, 64), (64, 256, 512)):
        for dtype in (1, 2):
            assert size(n, pixels, c, 8, dtype, 0, 1) == 0, (n, pixels, c)
    for n, pixels, c in ((32, 4096, 64), (1, 10_300, 64), (64, 65536, 64)):
        assert size(n, pixels, c, 8, 1, 0, 1) > 0


def test_partials_of_long_sums_take_a_gigabyte_at_most():
    size = _lib.load().ddpm_linear_workspace_bytes
    m, n, k = 1 << 20, 16_384, 16_400  # two splits of it: 137 GB
    assert size(m, n, k, k, 0, 1, 0, 1) <= 1 << 30
    extra = -(-m // 64) * n  # column sums for the bias
    assert size(m, n, k, k, 0, 1, 1, 1) <= (1 << 30) + extra * 4
    assert size(300, 520, 16_400, 16_400, 0, 1, 0, 1) == -(-2 * 300 * 520 * 4 // 256) * 256
