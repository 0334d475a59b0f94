"""Blocks whose scale has every bit of its mantissa set: s = 2^k (2 - 2^-23), of which 1 / s is a hair above the middle of
two floats, so that an inverse computed in steps may end on the lower one.  Elements stand at 2 (q + half a step) 2^k, with q
an even e4m3 value: times the lower inverse they are ties and go to q, times the rounded one they are above the tie.

Each test has the wrong answer a step of e4m3 off, 2^-4 of the value at least, and holds equality with the definition in
64 bits or, for sums, FP32's roundings of one product.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import fp8_ref as ref  # noqa: E402
from strix_trellis import runtime  # noqa: E402

DEV = ref.DEV
MOST = float.fromhex("0x1.bffffep+9")       # / 448 = 2 - 2^-23 in float32


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


def block(n, by):
    """`n` float32 values: the largest, and elements at ties, times `by` (a power of two)."""
    ties = torch.tensor([1.0625, 1.3125, 1.5625, 1.8125], dtype=torch.float64)
    v = torch.cat([2.0 * ties * 2.0 ** e for e in range(-6, 8)])
    v = torch.cat([v, -v]).repeat(n // (2 * v.numel()) + 1)[:n]
    v[n // 2] = MOST
    return (v * by).to(torch.float32).to(DEV)


def test_the_values_are_what_they_are_meant_to_be(ctx):
    for by in (1.0, 2.0 ** -20, 2.0 ** 20):
        x = block(128, by)[None]
        q, s = ref.round_rows(x)
        assert float(s) == (2.0 - 2.0 ** -23) * by
        low = (x.double() * (0.5 / by)).float().to(ref.E4M3)
        assert int((low.float() != q.float()).sum()) >= 100


@pytest.mark.parametrize("rows", [1, 2, 4, 6, 16, 40, 150, 300, 1100])
@pytest.mark.parametrize("by", [1.0, 2.0 ** -20, 2.0 ** 20])
def test_rows(ctx, rows, by):
    """Rows rounded in the call, through unit weights: a channel has one element of its row."""
    I = 256
    x = torch.cat([block(128, by), block(128, 4.0 * by)])[None].repeat(rows, 1)
    q, s = ref.round_rows(x)
    w = torch.eye(I, device=DEV).to(ref.E4M3)
    handle = runtime.Fp8Weights(ctx, w, torch.ones(2, 2, device=DEV))
    y = torch.zeros(rows, I, device=DEV)
    runtime.fp8_linear(handle, x, y)
    torch.cuda.synchronize()
    handle.destroy()
    want = q.double() * ref.spread(s.double(), rows, I)
    assert bool(((y.double() - want).abs() <= 2.0 ** -22 * want.abs()).all())


@pytest.mark.parametrize("by", [1.0, 2.0 ** -20])
def test_weights(ctx, by):
    """Weights rounded in preparation, read out by unit rows."""
    I, N = 256, 128
    # one element a channel in each block, the largest among them
    w = torch.zeros(N, I, device=DEV)
    n = torch.arange(N, device=DEV)
    w[n, n] = block(128, by)
    w[n, 128 + n] = block(128, 8.0 * by)
    q, t = ref.round_weights(w)
    assert bool((t == (2.0 - 2.0 ** -23) * by * torch.tensor([[1.0, 8.0]], device=DEV)).all())
    handle = runtime.Fp8Weights(ctx, w)
    x = torch.eye(I, device=DEV).to(ref.E4M3)
    y = torch.zeros(I, N, device=DEV)
    runtime.fp8_linear(handle, x, y, x_scales=torch.ones(I, 2, device=DEV))
    torch.cuda.synchronize()
    handle.destroy()
    want = (q.double() * ref.spread(t.double(), N, I)).t()
    assert bool(((y.double() - want).abs() <= 2.0 ** -22 * want.abs()).all())


@pytest.mark.parametrize("rows,N", [(1, 128), (9, 256), (200, 256), (2048, 8192), (4096, 4096)])
def test_hidden_rows(ctx, rows, N):
    """Hidden rows rounded behind the products, in a launch of their own or in the tile: silu(32) is 32 in FP32, and the up
    projection's biases are the elements over 32."""
    I = 128
    zero, one = torch.zeros(N, I, device=DEV).to(ref.E4M3), torch.ones(N // 128, 1, device=DEV)
    h = block(128, 1.0).repeat(N // 128)
    handle = runtime.Fp8Weights(ctx, zero, one, bias=torch.full((N,), 32.0, device=DEV), up=zero, up_scales=one,
                                up_bias=h / 32.0)
    x = torch.ones(rows, I, device=DEV)
    plain = torch.zeros(rows, N, device=DEV)
    runtime.fp8_gated(handle, x, plain)
    y, s = torch.zeros(rows, N, device=DEV, dtype=ref.E4M3), torch.zeros(rows, N // 128, device=DEV)
    runtime.fp8_gated(handle, x, y, y_scales=s)
    torch.cuda.synchronize()
    handle.destroy()
    assert bool((plain == h).all())
    q, want = ref.round_rows(h[None])
    assert bool((s == want).all()) and bool((y.float() == q.float()).all())
