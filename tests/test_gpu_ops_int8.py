"""8-bit integer linear layer (strix_amd_int8_*) against its definition in 64 bits.

Tolerances.  The integer sum is exact; float(sum), * s, * t, + bias, * alpha,
beta * old and the last addition are one rounding each, off by at most half a
step, 2^-24 of the value it rounds.  So |y - exact| <= 2^-24 (1 + 2^-20) times
(5 |alpha s t sum| + 3 |alpha bias| + 2 |beta old|), and for 16-bit outputs half
a step of the type (eps / 2 of the value, or half the least subnormal) more.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from strix_trellis import abi, runtime  # noqa: E402

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24 * (1 + 2.0 ** -20)


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


def quantize(x):
    """(q, s) of rows in float64: s = max(RN32(max / 127), 2^-126), q = RNE(x / s).  The float64 quotient of two
    float32 values lies on a tie only where the exact one does (their distance is at least 2^-25 of a step)."""
    x = x.double()
    s = (x.abs().amax(1) / 127.0).float().clamp(min=2.0 ** -126).double()
    return torch.round(x / s[:, None]), s


def reference(x, x_scales, w, t, bias, alpha, beta, old):
    """(y, the magnitude its tolerance counts), float64 on the CPU."""
    q, s = quantize(x.cpu()) if x_scales is None else (x.cpu().double(), x_scales.cpu().double())
    core = alpha * (q @ w.cpu().double().t()) * s[:, None] * t.cpu().double()
    b = torch.zeros(1, dtype=torch.float64) if bias is None else alpha * bias.cpu().double()
    o = beta * old.cpu().double() if beta else torch.zeros(1, dtype=torch.float64)
    return core + b + o, 5 * core.abs() + 3 * b.abs() + 2 * o.abs()


def check(y, ref, mag, what):
    got = y.cpu().double()
    tol = U * mag
    if y.dtype != torch.float32:
        info = torch.finfo(y.dtype)
        tol = tol * (1 + info.eps) + (ref.abs() + tol) * (info.eps / 2) + info.smallest_normal * info.eps / 2
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got - ref).abs().max()))


def layer(I, N, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-128, 128, (N, I), generator=g, dtype=torch.int8)
    t = torch.rand(N, generator=g) * 0.01 + 1e-4
    b = torch.randn(N, generator=g) if bias else None
    return w.to(DEV), t.to(DEV), None if b is None else b.to(DEV)


# one row to several tiles; inputs and channels on and off every block, tile and piece boundary
SHAPES = [(1, 64, 16), (1, 1, 1), (2, 15, 17), (3, 4096, 33), (8, 5119, 129), (15, 128, 255), (16, 1000, 512),
          (17, 129, 31), (33, 640, 100), (64, 5120, 96), (65, 300, 257), (127, 2049, 128), (128, 128, 384),
          (129, 5121, 130), (200, 77, 515), (256, 1152, 256), (333, 511, 259), (700, 192, 640), (4, 6200, 65),
          (1, 40000, 40), (20, 17000, 48), (9, 9000, 1031)]


@pytest.mark.parametrize("rows,I,N", SHAPES)
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "i8"])
def test_against_definition(ctx, rows, I, N, kind):
    w, t, bias = layer(I, N, rows * 7 + I + N)
    g = torch.Generator().manual_seed(rows + I)
    if kind == "i8":
        x = torch.randint(-128, 128, (rows, I), generator=g, dtype=torch.int8).to(DEV)
        xs = (torch.rand(rows, generator=g) + 0.1).to(DEV)
    else:
        x, xs = torch.randn(rows, I, generator=g).to(TYPES[kind]).to(DEV), None
    weights = runtime.Int8Weights(ctx, w, t, bias=bias)
    out = {"f32": "f32", "f16": "bf16", "bf16": "f16", "i8": "f32"}[kind]
    y = torch.full((rows, N), float("nan"), device=DEV, dtype=TYPES[out])
    runtime.int8_linear(weights, x, y, x_scales=xs)
    ref, mag = reference(x, xs, w, t, bias, 1.0, 0.0, None)
    check(y, ref, mag, (rows, I, N, kind))
    weights.destroy()


@pytest.mark.parametrize("rows", [1, 5, 16, 40, 130])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_alpha_beta_and_strided_rows(ctx, rows, out):
    I, N = 777, 203
    w, t, bias = layer(I, N, 5)
    weights = runtime.Int8Weights(ctx, w, t, bias=bias)
    wide_x = torch.randn(rows + 2, I + 13, device=DEV)
    wide_y = torch.randn(rows + 2, N + 7, device=DEV).to(TYPES[out])
    before = wide_y.clone()
    x, y = wide_x[1:1 + rows, 5:5 + I], wide_y[1:1 + rows, 3:3 + N]
    old = y.clone()
    runtime.int8_linear(weights, x, y, alpha=0.5, beta=-2.0)
    ref, mag = reference(x, None, w, t, bias, 0.5, -2.0, old)
    check(y, ref, mag, (rows, out))
    # what lies beside the rows and behind the last one is as it was
    inside = torch.zeros_like(wide_y, dtype=torch.bool)
    inside[1:1 + rows, 3:3 + N] = True
    assert torch.equal(wide_y[~inside].view(-1), before[~inside].view(-1))
    # beta == 0 reads nothing of the old output
    y.fill_(float("nan"))
    runtime.int8_linear(weights, x, y, alpha=0.5)
    ref, mag = reference(x, None, w, t, bias, 0.5, 0.0, None)
    check(y, ref, mag, (rows, out, "beta 0"))
    weights.destroy()


@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_rounding_of_rows(ctx, rows, kind):
    """Identity weights with scale 1 show q * s itself: ties to even, the largest value, zeros, tiny rows."""
    I = 160
    weights = runtime.Int8Weights(ctx, torch.eye(I, dtype=torch.int8, device=DEV), torch.ones(I, device=DEV))
    g = torch.Generator().manual_seed(9)
    x = torch.randn(rows, I, generator=g)
    x[0] = (torch.arange(I) % 254 - 127).float() * 0.5          # s = 1/2 exactly below: quotients j and j + 1/2
    x[0, 0] = 63.5
    x[0, 1:130] = (torch.arange(129) - 64).float() * 0.25       # every tie of that scale
    if rows > 1:
        x[1] = 0.0
        x[2] = 0.0
        x[2, 5] = -3.0                                          # one value: q = -127
        x[3] *= 1e-4 if kind == "f16" else 1e-30
        if kind != "f16":
            x[4] = 2.0 ** -130                                  # below the least scale: q = 0 or 1
            x[5] = 2.0 ** -126 * 1.5                            # ties on the least scale
            x[6] *= 1e37
    x = x.to(TYPES[kind]).to(DEV)
    y = torch.full((rows, I), float("nan"), device=DEV)
    runtime.int8_linear(weights, x, y)
    q, s = quantize(x.cpu())
    assert bool((q.abs() <= 127).all())
    assert torch.equal(y.cpu(), (q * s[:, None]).float())       # one rounding of an exact product
    weights.destroy()


def test_weights_rounded_per_channel(ctx):
    g = torch.Generator().manual_seed(3)
    for kind, dtype in TYPES.items():
        for N, I in ((40, 333), (17, 6000), (1, 64)):
            w = (torch.randn(N, I, generator=g) * torch.rand(N, 1, generator=g)).to(dtype)
            weights = runtime.Int8Weights(ctx, w.to(DEV))
            x = torch.randint(-128, 128, (21, I), generator=g, dtype=torch.int8)
            xs = torch.rand(21, generator=g) + 0.5
            y = torch.empty((21, N), device=DEV)
            runtime.int8_linear(weights, x.to(DEV), y, x_scales=xs.to(DEV))
            q, t = quantize(w)
            ref, mag = reference(x, xs, q, t, None, 1.0, 0.0, None)
            check(y, ref, mag, (kind, N, I))
            weights.destroy()


@pytest.mark.parametrize("rows", [3, 40, 140])
def test_non_finite_values_stay_in_their_row(ctx, rows):
    I, N = 500, 70
    w, t, bias = layer(I, N, 8)
    weights = runtime.Int8Weights(ctx, w, t, bias=bias)
    x = torch.randn(rows, I, device=DEV)
    clean = torch.empty((rows, N), device=DEV)
    runtime.int8_linear(weights, x, clean)
    bad = x.clone()
    bad[0, 499] = float("inf")
    bad[2, 0] = float("nan")
    y = torch.empty((rows, N), device=DEV)
    runtime.int8_linear(weights, bad, y)
    assert bool(torch.isnan(y[[0, 2]]).all())
    keep = [r for r in range(rows) if r not in (0, 2)]
    assert torch.equal(y[keep], clean[keep])
    # a weight that is not finite: its channel alone
    wf = torch.randn(N, I, device=DEV)
    wf[3, 7] = float("-inf")
    other = runtime.Int8Weights(ctx, wf)
    runtime.int8_linear(other, x, y)
    assert bool(torch.isnan(y[:, 3]).all()) and bool(torch.isfinite(y[:, [c for c in range(N) if c != 3]]).all())
    other.destroy()
    weights.destroy()


def test_bits_of_a_row_do_not_depend_on_the_others(ctx):
    for I, N in ((1153, 300), (5120, 1152)):
        w, t, bias = layer(I, N, 4)
        weights = runtime.Int8Weights(ctx, w, t, bias=bias)
        x = torch.randn(400, I, device=DEV)
        whole = torch.empty((400, N), device=DEV)
        runtime.int8_linear(weights, x, whole)
        for rows in (1, 2, 7, 8, 9, 16, 17, 32, 33, 64, 65, 100, 128, 129, 257):
            y = torch.empty((rows, N), device=DEV)
            runtime.int8_linear(weights, x[:rows], y)
            assert torch.equal(y, whole[:rows]), (I, N, rows)
        weights.destroy()


def test_plans_streams_and_graphs(ctx):
    """Plans on another stream and captured into a graph, replayed with new inputs and eager work in between."""
    stream = torch.cuda.Stream()
    cases = [(1, 5120, 640), (8, 1000, 77), (40, 512, 300), (200, 700, 513)]
    made = []
    for rows, I, N in cases:
        w, t, bias = layer(I, N, rows)
        weights = runtime.Int8Weights(ctx, w, t, bias=bias)
        xs = [torch.randn(rows, I, device=DEV) for _ in range(3)]
        want = []
        for x in xs:
            y = torch.empty((rows, N), device=DEV)
            want.append(runtime.int8_linear(weights, x, y))
        x, y = torch.zeros(rows, I, device=DEV), torch.empty((rows, N), device=DEV)
        made.append((weights, xs, want, x, y, runtime.Int8LinearPlan(weights, x, y, stream=stream)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for *_, plan in made:
            plan.submit()
    torch.cuda.synchronize()
    for rep in range(6):
        for weights, xs, want, x, y, plan in made:
            x.copy_(xs[rep % 3])
            y.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay() if rep != 2 else [m[-1].submit() for m in made]
        torch.cuda.synchronize()
        for weights, xs, want, x, y, plan in made:
            assert torch.equal(y, want[rep % 3]), rep
            runtime.int8_linear(weights, xs[0], torch.empty_like(y))
    for weights, *_, plan in made:
        with pytest.raises(abi.StrixError):
            weights.destroy()       # a plan holds them
        plan.destroy()
        weights.destroy()


def test_refusals(ctx):
    w, t, bias = layer(64, 32, 1)
    weights = runtime.Int8Weights(ctx, w, t, bias=bias)
    x, y = torch.randn(4, 64, device=DEV), torch.zeros(4, 32, device=DEV)

    def status(*args, **kw):
        with pytest.raises(abi.StrixError) as e:
            runtime.int8_linear(weights, *args, **kw)
        return e.value.name

    assert status(torch.randn(4, 63, device=DEV), y) == "UNSUPPORTED_FORMAT"
    assert status(x, torch.zeros(3, 32, device=DEV)) == "UNSUPPORTED_FORMAT"
    assert status(x, torch.zeros(4, 32, device=DEV, dtype=torch.int8)) == "UNSUPPORTED_FORMAT"
    assert status(x, y, x_scales=torch.ones(4, device=DEV)) == "INVALID_ARGUMENT"
    assert status(x.to(torch.int8), y) == "INSUFFICIENT_BUFFER"
    assert status(x.to(torch.int8), y, x_scales=torch.ones(3, device=DEV)) == "INSUFFICIENT_BUFFER"
    assert status(x, y, alpha=float("inf")) == "INVALID_ARGUMENT"
    many = torch.randn(20, 64, device=DEV), torch.zeros(20, 32, device=DEV)
    assert status(*many, workspace=torch.zeros(256, dtype=torch.uint8, device=DEV)) == "INSUFFICIENT_BUFFER"
    assert status(x.cpu(), y, workspace=torch.zeros(1 << 16, dtype=torch.uint8, device=DEV)) == "INVALID_ARGUMENT"
    both = torch.zeros(4, 96, device=DEV)
    assert status(both[:, :64], both[:, 32:64]) == "INVALID_ARGUMENT"
    with pytest.raises(abi.StrixError):
        runtime.Int8Weights(ctx, w)                                     # int8 without scales
    with pytest.raises(abi.StrixError):
        runtime.Int8Weights(ctx, w.float(), t)                          # scales of weights that are not int8
    empty = torch.empty(0, 32, device=DEV)
    runtime.int8_linear(weights, torch.empty(0, 64, device=DEV), empty)  # no rows: nothing to do
    torch.cuda.synchronize()
    weights.destroy()
