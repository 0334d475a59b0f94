"""Norms of rows whose sums or squares pass the range of FP32 while their values do not: RMS and LAYER, before and
behind the residual sum, at every share of a row that a thread can hold.

Tolerances are those of the operator's own test: such a row is summed again after a multiplication by a power of two,
which rounds nothing that counts: the values themselves stay as they are, but for one rounding with the mean.
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


def rows_of(width, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda: torch.randn(width, generator=g)  # noqa: E731
    most = torch.finfo(dtype).max
    ends = torch.tensor([most, -most, -most / 2]).repeat(width // 3 + 1)[:width]
    return torch.stack([
        r(),                                    # an ordinary row
        r() * 1e19,                             # squares past the range
        r() * 1e30,
        r() * 2e37,                             # the sum too, for many channels
        (3.0 + 0.1 * r()) * 1e37,               # a mean far from zero
        ends,                                   # values whose distance from the mean is past the range
        -ends,
        r() * 1e17,                             # squares inside the range for few channels, past it for many
    ]).to(dtype).to(DEV), lambda: torch.randn(width, generator=g).to(DEV)


@pytest.mark.parametrize("width", [3, 200, 1000, 2047, 4099, 5121, 8195, 12289, 16385, 24577, 30001])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_sums_past_the_range(ctx, width, kind, name):
    x, vec = rows_of(width, norm.TYPES[name], width)
    layer = kind == "layer"
    # the first norm, whose result is added to an ordinary residual
    residual = torch.randn(x.shape, device=DEV).to(x.dtype)
    for p in ({"post_weight": vec()}, {"post_weight": vec(), "post_bias": vec()}):
        hidden = torch.zeros_like(x)
        runtime.block_norm(ctx, block=x, residual=residual, hidden=hidden, kind=kind, weight_offset=1.0, **p)
        u, m, _, _ = norm.reference(x, residual, None, "linear", p, layer, 1e-6, 1.0, 1.0, 1.0)
        norm.check(hidden, u, m, (width, kind, name, "post"))
    # the second norm, of a sum that is as large
    for p in ({"pre_weight": vec()}, {"pre_weight": vec(), "pre_bias": vec(), "channel_scale": vec()}):
        hidden, normed = torch.zeros_like(x), torch.zeros_like(x)
        runtime.block_norm(ctx, block=residual, residual=x, hidden=hidden, normed=normed, kind=kind,
                           residual_scale=0.5, **p)
        _, _, n, m = norm.reference(residual, x, None, "linear", p, layer, 1e-6, 0.0, 0.5, 1.0)
        norm.check(normed, n, m, (width, kind, name, "pre"))
    # both norms in one call
    p = {"post_weight": vec(), "pre_weight": vec()}
    normed = torch.zeros_like(x)
    runtime.block_norm(ctx, block=x, residual=x, normed=normed, kind=kind, residual_scale=0.25, **p)
    _, _, n, m = norm.reference(x, x, None, "linear", p, layer, 1e-6, 0.0, 0.25, 1.0)
    norm.check(normed, n, m, (width, kind, name, "both"))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_epsilon_counts_beside_such_squares(ctx, kind):
    for width, eps in ((300, 1e38), (5000, 1e36), (300, 3e38)):
        x, vec = rows_of(width, torch.float32, 1)
        w = vec()
        normed = torch.zeros_like(x)
        runtime.block_norm(ctx, block=x, normed=normed, pre_weight=w, kind=kind, eps=eps)
        _, _, n, m = norm.reference(x, None, None, "linear", {"pre_weight": w}, kind == "layer", eps, 0.0, 1.0, 1.0)
        norm.check(normed, n, m, (width, kind, eps))


def test_infinite_and_nan_values(ctx):
    """RMS divides the finite values of a row by an infinite norm; a LAYER row has no mean."""
    width = 700
    x = torch.randn(3, width, device=DEV)
    x[1, 5] = float("inf")
    x[2, 6] = float("nan")
    w, b = torch.randn(width, device=DEV), torch.randn(width, device=DEV)
    for kind in ("rms", "layer"):
        normed = torch.zeros_like(x)
        runtime.block_norm(ctx, block=x, normed=normed, pre_weight=w, pre_bias=b, kind=kind)
        assert bool(torch.isfinite(normed[0]).all()) and bool(torch.isnan(normed[2]).all())
        assert bool(torch.isnan(normed[1, 5]))
        rest = torch.arange(width, device=DEV) != 5
        if kind == "rms":
            assert torch.equal(normed[1][rest], b[rest])
        else:
            assert bool(torch.isnan(normed[1]).all())
