"""The 8-bit layer where the integer sum times the token's scale leaves the range of FP32 although the output does not:
rows of huge values in front of small channel scales, given scales below the normal range in front of large ones,
channels of scale zero.

Tolerances are those of the layer's own test: a power of two between the factors rounds nothing, and no output here
is below the normal range.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_ops_int8 as int8  # noqa: E402
from strix_trellis import runtime  # noqa: E402

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


def check(y, ref, what):
    assert bool(torch.isfinite(y).all()), what
    int8.check(y, *ref, what)


# the core of a few rows, of sixteen, the small tiles, the large ones
@pytest.mark.parametrize("rows,N", [(1, 70), (4, 70), (16, 70), (40, 70), (300, 70), (640, 8200)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_huge_rows_before_small_channel_scales(ctx, rows, N, kind):
    I = 500
    g = torch.Generator().manual_seed(rows)
    w = torch.randint(-127, 128, (N, I), generator=g, dtype=torch.int8)
    t = torch.rand(N, generator=g) * 1e-12 + 1e-14
    t[5] = 0.0
    bias = torch.randn(N, generator=g)
    # rows in the direction of a channel's weights, so that its sum is as large as can be, from 1e30 to 3e38
    most = 10.0 ** (30 + 8.47 * torch.arange(rows) / max(rows - 1, 1)) if rows > 1 else torch.tensor([3e38])
    x = (w[torch.arange(rows) % N].float() / 127 * most[:, None]).to(int8.TYPES[kind])
    assert bool(torch.isfinite(x).all())
    weights = runtime.Int8Weights(ctx, w.to(DEV), t.to(DEV), bias=bias.to(DEV))
    y = torch.zeros(rows, N, device=DEV)
    runtime.int8_linear(weights, x.to(DEV), y)
    check(y, int8.reference(x, None, w, t, bias, 1.0, 0.0, None), (rows, N, kind))
    assert torch.equal(y[:, 5].cpu(), bias[5].expand(rows))
    weights.destroy()


@pytest.mark.parametrize("rows", [1, 4, 16, 40, 300])
@pytest.mark.parametrize("token,channel", [(2.0 ** 120, 2.0 ** -80), (2.0 ** -130, 2.0 ** 60), (2.0 ** -149, 2.0 ** 100),
                                           (2.0 ** 96, 2.0 ** -149), (-2.0 ** 127, 2.0 ** -60), (2.0 ** -126, 2.0 ** 30)])
def test_given_scales(ctx, rows, token, channel):
    I, N = 300, 45
    g = torch.Generator().manual_seed(rows)
    w = torch.randint(-128, 128, (N, I), generator=g, dtype=torch.int8)
    t = torch.full((N,), channel)
    x = torch.randint(-128, 128, (rows, I), generator=g, dtype=torch.int8)
    x[0] = w[0]
    xs = torch.full((rows,), token)
    weights = runtime.Int8Weights(ctx, w.to(DEV), t.to(DEV))
    for alpha in (1.0, -0.75):
        y = torch.zeros(rows, N, device=DEV)
        runtime.int8_linear(weights, x.to(DEV), y, x_scales=xs.to(DEV), alpha=alpha)
        check(y, int8.reference(x, xs, w, t, None, alpha, 0.0, None), (rows, token, channel))
    weights.destroy()


def test_what_has_no_finite_value(ctx):
    """An output past FP32 is infinite, with its sign; scales that are not finite stay in their row and channel."""
    inf = float("inf")
    I, N = 64, 40
    w = torch.ones(N, I, dtype=torch.int8)
    w[1] = -1
    t = torch.ones(N)
    t[2] = float("nan")
    x = torch.full((20, I), 100, dtype=torch.int8)
    xs = torch.ones(20)
    xs[3], xs[4], xs[5] = 2.0 ** 127, inf, float("nan")
    weights = runtime.Int8Weights(ctx, w.to(DEV), t.to(DEV))
    y = torch.zeros(20, N, device=DEV)
    runtime.int8_linear(weights, x.to(DEV), y, x_scales=xs.to(DEV))
    y = y.cpu()
    assert bool(torch.isnan(y[:, 2]).all()) and bool(torch.isnan(y[5]).all())
    for row in (3, 4):
        assert float(y[row, 0]) == inf and float(y[row, 1]) == -inf
    assert bool((y[6:, 3:] == 6400.0).all()) and bool((y[6:, 1] == -6400.0).all())
    weights.destroy()
