"""Every core of the 8-bit layer on long sums over inputs: bit for bit the same rows in calls of 16, which another core
serves, and sampled rows against the definition in 64 bits with the tolerances of the layer's own test."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_ops_int8 as int8  # noqa: E402
from int8_cores import CALLS  # noqa: E402
from strix_trellis import runtime  # noqa: E402

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


@pytest.mark.parametrize("core,rows,I,N", CALLS)
@pytest.mark.parametrize("kind", ["f32", "i8"])
def test_long_sums(ctx, core, rows, I, N, kind):
    g = torch.Generator(device=DEV).manual_seed(rows + I + N)
    w = torch.randint(-128, 128, (N, I), generator=g, device=DEV, dtype=torch.int8)
    t = torch.rand(N, generator=g, device=DEV) * 0.01 + 1e-4
    bias = torch.randn(N, generator=g, device=DEV)
    if kind == "i8":
        x = torch.randint(-128, 128, (rows, I), generator=g, device=DEV, dtype=torch.int8)
        xs = torch.rand(rows, generator=g, device=DEV) + 0.1
    else:
        x, xs = torch.randn(rows, I, generator=g, device=DEV), None
    weights = runtime.Int8Weights(ctx, w, t, bias=bias)
    y = torch.full((rows + 1, N), 7.0, device=DEV)
    runtime.int8_linear(weights, x, y[:rows], x_scales=xs)
    assert bool((y[rows] == 7.0).all())
    # the same rows sixteen at a time (one at a time in the cores of so few)
    step = 16 if rows > 16 else 1
    part = torch.full((rows, N), float("nan"), device=DEV)
    for r in range(0, rows, step):
        at = slice(r, min(r + step, rows))
        runtime.int8_linear(weights, x[at], part[at], x_scales=None if xs is None else xs[at])
    assert torch.equal(y[:rows], part), (core, int((y[:rows] != part).sum()))
    pick = torch.unique(torch.tensor([0, rows // 3, rows // 2, rows - 1], device=DEV))
    ref = int8.reference(x[pick], None if xs is None else xs[pick], w, t, bias, 1.0, 0.0, None)
    int8.check(y[pick], *ref, (core, rows, I, N, kind))
    weights.destroy()
