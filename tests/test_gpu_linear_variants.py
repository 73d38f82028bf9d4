"""linear_act on every tile that the planner chooses: ragged last tiles, residual and an
activation's backward, with operands and results that TMA can address and cannot."""

from __future__ import annotations

import pytest
import torch

from tests import _operators as ops
from tests.test_gpu_linear_act import _case, _run

pytestmark = pytest.mark.gpu

# m, n, k; product; tile columns, blocks that share a tile, epilogue warps
HALF = [
    ((4000, 4100, 1100), "forward", (256, 2, 8)),
    ((4001, 4104, 1104), "weight", (256, 2, 8)),
    ((9000, 1600, 520), "x", (256, 2, 8)),
    ((100, 25601, 512), "forward", (256, 1, 8)),
    ((100, 25600, 512), "weight", (256, 2, 16)),
    ((128, 30_000, 1000), "forward", (256, 1, 8)),
    ((5001, 1504, 240), "forward", (256, 2, 16)),
    ((20_000, 256, 264), "x", (256, 2, 16)),
    ((4000, 1200, 1104), "weight", (256, 1, 8)),
    ((1000, 2304, 700), "forward", (128, 1, 8)),
    ((300, 3000, 520), "x", (64, 1, 8)),
]
SINGLE = [
    ((4000, 1200, 1100), "forward", (128, 1, 8)),
    ((3333, 5000, 264), "x", (64, 1, 8)),
    ((300, 3000, 520), "forward", (64, 1, 8)),
    ((7000, 1000, 260), "weight", (128, 1, 8)),
]


@pytest.mark.parametrize("dtype,shape,product,tile",
                         [(t, *c) for t in (torch.bfloat16, torch.float16) for c in HALF]
                         + [(torch.float32, *c) for c in SINGLE])
def test_tile(dtype, shape, product, tile):
    assert ops.linear_choice(*shape, dtype, product, "silu")[:3] == tile
    x, w, b, res, dy = _case(*shape, dtype, seed=12)
    _run(x, w, b, res, dy, "silu")
    _run(x, w, b, None, dy, None)
