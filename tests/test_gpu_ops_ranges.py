"""The operators where a rule picks another kernel or another launch: every number of rows and width of input that
the 8-bit layer tells apart, and more rows than one launch or one pass takes.

No tolerances of their own: the integer sums are exact and a row's bits do not depend on the others, so every way to
compute a row has to leave the same bits; one way is held to the definition with the tolerances of the operators'
own tests.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_ops_int8 as int8  # noqa: E402
import test_gpu_ops_logprobs as logprobs  # noqa: E402
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


def rows_of(rows, I, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "i8":
        return torch.randint(-128, 128, (rows, I), generator=g, dtype=torch.int8).to(DEV), \
            (torch.rand(rows, generator=g) + 0.1).to(DEV)
    return torch.randn(rows, I, generator=g).to(int8.TYPES[kind]).to(DEV), None


@pytest.mark.parametrize("I", [3, 255, 256, 1000, 2048, 2049, 2176, 4096, 4097, 5120, 5121, 8192, 8193, 12001])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "i8"])
def test_few_rows_of_every_width(ctx, I, kind):
    rows, N = 20, 50
    w, t, bias = int8.layer(I, N, I)
    x, xs = rows_of(rows, I, kind, I)
    weights = runtime.Int8Weights(ctx, w, t, bias=bias)
    every = torch.zeros(rows, N, device=DEV)
    runtime.int8_linear(weights, x, every, x_scales=xs)
    int8.check(every, *int8.reference(x, xs, w, t, bias, 1.0, 0.0, None), (I, kind))
    for m in (1, 2, 3, 4, 5, 8, 9, 16):
        y = torch.full((m, N), float("nan"), device=DEV)
        runtime.int8_linear(weights, x[rows - m:], y, x_scales=None if xs is None else xs[rows - m:])
        assert torch.equal(y, every[rows - m:]), (I, kind, m)
    weights.destroy()


def test_every_number_of_rows(ctx):
    rows, I, N = 2100, 200, 10000
    w, t, bias = int8.layer(I, N, 4)
    x, _ = rows_of(rows, I, "bf16", 5)
    weights = runtime.Int8Weights(ctx, w, t, bias=bias)
    every = torch.zeros(rows, N, device=DEV)
    runtime.int8_linear(weights, x, every)
    pick = torch.randperm(rows, generator=torch.Generator().manual_seed(6))[:60]
    ref, mag = int8.reference(x[pick.to(DEV)], None, w, t, bias, 1.0, 0.0, None)
    int8.check(every[pick.to(DEV)], ref, mag, "2100 rows")
    for m in (1, 7, 16, 17, 33, 64, 65, 97, 130, 257, 400, 513, 900, 1281):
        y = torch.full((m, N), float("nan"), device=DEV)
        runtime.int8_linear(weights, x[rows - m:], y)
        assert torch.equal(y, every[rows - m:]), m
    weights.destroy()
    # few channels: the small tiles at many rows
    for N in (1, 40, 700):
        w, t, bias = int8.layer(I, N, N)
        weights = runtime.Int8Weights(ctx, w, t, bias=bias)
        every = torch.zeros(rows, N, device=DEV)
        runtime.int8_linear(weights, x, every)
        int8.check(every, *int8.reference(x, None, w, t, bias, 1.0, 0.0, None), N)
        for m in (20, 300, 1000):
            y = torch.full((m, N), float("nan"), device=DEV)
            runtime.int8_linear(weights, x[:m], y)
            assert torch.equal(y, every[:m]), (N, m)
        weights.destroy()


def test_more_rows_than_one_pass(ctx):
    """65536 rows a pass; the last one of a single row, of nine, of twenty."""
    I, N = 70, 33
    w, t, bias = int8.layer(I, N, 7)
    weights = runtime.Int8Weights(ctx, w, t, bias=bias)
    for kind, extra in (("f32", 1), ("bf16", 9), ("i8", 20)):
        rows = 65536 + extra
        x, xs = rows_of(rows, I, kind, extra)
        y = torch.zeros(rows + 1, N, device=DEV)
        runtime.int8_linear(weights, x, y[:rows], x_scales=xs)
        int8.check(y[:rows], *int8.reference(x, xs, w, t, bias, 1.0, 0.0, None), kind)
        assert not y[rows].any()
    weights.destroy()


def test_more_channels_than_one_launch(ctx):
    """2^20 rows a launch of the preparation."""
    I, N = 5, 2 ** 20 + 37
    w, t, bias = int8.layer(I, N, 8)
    weights = runtime.Int8Weights(ctx, w, t, bias=bias)
    for m in (2, 40):
        x, _ = rows_of(m, I, "f32", m)
        y = torch.zeros(m, N, device=DEV)
        runtime.int8_linear(weights, x, y)
        int8.check(y, *int8.reference(x, None, w, t, bias, 1.0, 0.0, None), m)
    weights.destroy()


def test_more_rows_than_one_launch(ctx):
    """2^20 rows a launch of the norms and of the log probabilities."""
    rows, width = 2 ** 20 + 5, 7
    g = torch.Generator().manual_seed(9)
    x = torch.randn(rows + 1, width, generator=g).to(DEV)
    gate = torch.randn(rows, 1, generator=g).to(DEV)
    weight = torch.randn(width, generator=g).to(DEV)
    hidden, normed = torch.zeros_like(x), torch.zeros_like(x)
    runtime.block_norm(ctx, block=x[:rows], residual=x[:rows], gate=gate, hidden=hidden[:rows], normed=normed[:rows],
                       pre_weight=weight)
    h, n = torch.zeros(50, width, device=DEV), torch.zeros(50, width, device=DEV)
    at = slice(rows - 50, rows)
    runtime.block_norm(ctx, block=x[at], residual=x[at], gate=gate[at], hidden=h, normed=n, pre_weight=weight)
    assert torch.equal(hidden[at], h) and torch.equal(normed[at], n)
    u = x[:rows].double() * (1 + gate.double())
    assert (hidden[:rows].double() - u).abs().max() <= norm.TOL * 8 * (1 + float(gate.abs().max()))
    assert not hidden[rows].any() and not normed[rows].any()

    tokens = torch.randint(0, width, (rows,), generator=g, dtype=torch.int32).to(DEV)
    out, part = logprobs.outputs(rows, 3), logprobs.outputs(50, 3)
    runtime.token_logprobs(ctx, x[:rows], tokens=tokens, **out)
    runtime.token_logprobs(ctx, x[at], tokens=tokens[at], **part)
    for k in out:
        assert torch.equal(out[k][at], part[k]), k
    logprobs.check(x[:1000], tokens[:1000], {k: v[:1000] for k, v in out.items()}, 1.0, "first")
    logprobs.check(x[at], tokens[at], part, 1.0, "last")
