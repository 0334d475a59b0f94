"""Sigmoid gates far below zero.

Tolerances: those of the operator's own test, and where e^g is below the normal range of FP32 two steps of it, 2^-149
each, times what it multiplies: one of the exponential, one of the product with the reciprocal; the product with
block_scale keeps them.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_ops_norm as norm  # noqa: E402
from strix_trellis import runtime  # noqa: E402

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


@pytest.mark.parametrize("shape", ["full", "rows"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_sigmoid_over_its_whole_range(ctx, shape, name):
    dtype = norm.TYPES[name]
    width = 600
    steps = torch.linspace(-104.0, 104.0, 417)
    rows = 417 if shape == "rows" else 7
    gate = steps[:, None] if shape == "rows" else torch.linspace(-104.0, 104.0, rows * width).view(rows, width)
    gate = gate.to(dtype).to(DEV)
    g = torch.Generator().manual_seed(5)
    for size in (1.0, 1e6, 1e30):
        block = ((torch.rand(rows, width, generator=g) + 0.5) * size).to(dtype).to(DEV)
        hidden = torch.zeros_like(block)
        runtime.block_norm(ctx, block=block, gate=gate, gate_activation="sigmoid", hidden=hidden, block_scale=0.5)
        u, m, _, _ = norm.reference(block, None, gate, "sigmoid", {}, False, 1e-6, 0.0, 1.0, 0.5)
        m = m + (2 * 2.0 ** -149 * block.cpu().double().abs() + 2.0 ** -149) / norm.TOL
        norm.check(hidden, u, m, (shape, name, size))


def test_extreme_gates(ctx):
    inf, nan = float("inf"), float("nan")
    block = torch.full((1, 6), 3.0, device=DEV)
    gate = torch.tensor([[-inf, inf, nan, -3.4e38, 3.4e38, 0.0]], device=DEV)
    hidden = torch.zeros_like(block)
    runtime.block_norm(ctx, block=block, gate=gate, gate_activation="sigmoid", hidden=hidden)
    h = hidden[0].cpu()
    assert h[[0, 3]].tolist() == [0.0, 0.0] and h[[1, 4]].tolist() == [3.0, 3.0] and h[5] == 1.5
    assert bool(torch.isnan(h[2]))
