"""Block-scaled e4m3 linear layer (strix_amd_fp8_*) against its definition in 64 bits (tests/fp8_ref.py, where the
tolerances are derived)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import fp8_ref as ref  # noqa: E402
from strix_trellis import abi, runtime  # noqa: E402

DEV = ref.DEV
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


def run(ctx, w, t, bias, x, out, x_scales=None, alpha=1.0, beta=0.0, old=None):
    handle = runtime.Fp8Weights(ctx, w, t, bias=bias)
    y = torch.full((x.shape[0], w.shape[0]), NAN, device=DEV, dtype=out) if old is None else old.clone()
    runtime.fp8_linear(handle, x, y, x_scales=x_scales, alpha=alpha, beta=beta)
    torch.cuda.synchronize()
    handle.destroy()
    return y


def held(ctx, I, N, rows, dtype, out, bias, given, seed=0):
    w, t, b = ref.weights(I, N, seed, bias)
    x = ref.rows_of(rows, I, seed + 1, dtype)
    q, s = ref.round_rows(x)
    y = run(ctx, w, t, b, q if given else x, out, s if given else None)
    z, mag = ref.product(q, s, w, t, b)
    ref.check(y, z, ref.unit(I, out) * mag, (I, N, rows, dtype, out, given))
    if out != torch.float32 and I * N >= 1000:
        ref.typical(y, z, (I, N, rows, dtype, out, given))
    return y


# inputs and channels at and off the grids of 16, 32, 64 and 128; fewer blocks than waves, many batches of them
SHAPES = [(1, 1), (3, 5), (127, 33), (128, 128), (129, 16), (300, 70), (1000, 1027), (2048, 272), (4100, 200),
          (5119, 100), (12288, 48), (44000, 17)]


@pytest.mark.parametrize("I,N", SHAPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 7, 16, 17, 33, 65])
def test_shapes(ctx, I, N, rows):
    held(ctx, I, N, rows, torch.float32, torch.float32, True, False, seed=I + N)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 4, 8, 12, 40])
def test_types(ctx, dtype, out, rows):
    given = dtype == "e4m3"
    held(ctx, 1153, 259, rows, ref.TYPES.get(dtype, torch.bfloat16), ref.TYPES[out], rows % 3 == 0, given)


@pytest.mark.parametrize("I,N,rows", [(4096, 1024, 200), (515, 2307, 333), (4096, 640, 700), (256, 300, 2049),
                                      (1152, 5120, 511), (2304, 1290, 1030), (130, 96, 4500)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_many_rows(ctx, I, N, rows, out):
    held(ctx, I, N, rows, torch.bfloat16, ref.TYPES[out], True, False)


def test_more_rows_than_a_pass(ctx):
    held(ctx, 100, 40, 66000, torch.float16, torch.float32, True, False)


def test_every_number_of_rows(ctx):
    """1..80 rows of one input: a row's own tolerance, whatever tile it falls into."""
    I, N = 640, 200
    w, t, b = ref.weights(I, N, 3)
    x = ref.rows_of(80, I, 4)
    q, s = ref.round_rows(x)
    z, mag = ref.product(q, s, w, t, b)
    for rows in range(1, 81):
        y = run(ctx, w, t, b, x[:rows], torch.float32)
        ref.check(y, z[:rows], ref.unit(I) * mag[:rows], rows)


@pytest.mark.parametrize("rows", [1, 4, 9, 30, 100, 300])
def test_rounding_in_the_call(ctx, rows):
    """Rows rounded in the call give the bits that the same values and scales give when they come rounded."""
    I, N = 1411, 160
    w, t, b = ref.weights(I, N, 5)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x = ref.rows_of(rows, I, 6, dtype)
        # magnitudes over the whole range of a block, ties of e4m3 among them, and blocks of zeros
        x[:, ::7] *= 2.0 ** -9
        x[:, 128:256] = 0
        x[0, 256:384] = torch.arange(128, device=DEV).to(dtype) * 3.5   # its scale is 444.5 / 448
        x[-1, 384:512] = 448.0
        x[-1, 384:510] = (17.0 + 2.0 * (torch.arange(126, device=DEV) % 7)).to(dtype)   # ties at scale 1
        q, s = ref.round_rows(x)
        assert torch.equal(run(ctx, w, t, b, x, torch.float32), run(ctx, w, t, b, q, torch.float32, s)), dtype


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("I,N", [(5, 3), (300, 261), (128, 16)])
def test_weights_rounded_in_preparation(ctx, dtype, I, N):
    w = ref.rows_of(N, I, 7, ref.TYPES[dtype]) * 0.02
    q, t = ref.round_weights(w)
    x = ref.rows_of(5, I, 8)
    assert torch.equal(run(ctx, w, None, None, x, torch.float32), run(ctx, q, t, None, x, torch.float32))


@pytest.mark.parametrize("rows", [2, 20, 70])
@pytest.mark.parametrize("alpha,beta", [(0.5, 0.0), (-1.25, 1.0), (0.0, -0.75)])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_alpha_beta(ctx, rows, alpha, beta, out):
    I, N = 200, 75
    w, t, b = ref.weights(I, N, 9)
    x = ref.rows_of(rows, I, 10)
    old = ref.rows_of(rows, N, 11, ref.TYPES[out])
    if beta == 0.0:
        old[:] = NAN   # not read
    q, s = ref.round_rows(x)
    z, mag = ref.product(q, s, w, t, b)
    o = beta * old.double() if beta else torch.zeros_like(z)
    y = run(ctx, w, t, b, x, ref.TYPES[out], alpha=alpha, beta=beta, old=old)
    ref.check(y, alpha * z + o, ref.unit(I, y.dtype) * (abs(alpha) * mag + o.abs()), (alpha, beta))


@pytest.mark.parametrize("rows", [1, 3, 16, 50, 260])
def test_strides(ctx, rows):
    """Rows inside wider ones, at odd offsets; what lies around the output stays."""
    I, N = 333, 131
    w, t, b = ref.weights(I, N, 12)
    for dtype, out in ((torch.float32, torch.float16), (torch.bfloat16, torch.float32), (ref.E4M3, torch.bfloat16)):
        wide = ref.rows_of(rows, I + 9, 13, torch.float32).to(dtype)
        x = wide[:, 5:5 + I]
        s = None
        if dtype == ref.E4M3:
            s = torch.rand(rows, 3, device=DEV) * 0.01 + 0.001
        y_wide = torch.full((rows, N + 6), 7.0, device=DEV, dtype=out)
        handle = runtime.Fp8Weights(ctx, w, t, bias=b)
        runtime.fp8_linear(handle, x, y_wide[:, 3:3 + N], x_scales=s)
        torch.cuda.synchronize()
        handle.destroy()
        q, s = (x, s) if s is not None else ref.round_rows(x)
        z, mag = ref.product(q, s, w, t, b)
        ref.check(y_wide[:, 3:3 + N], z, ref.unit(I, out) * mag, (rows, dtype))
        assert bool((y_wide[:, :3] == 7).all()) and bool((y_wide[:, 3 + N:] == 7).all())


def test_strided_weights(ctx):
    I, N = 140, 50
    w, t, b = ref.weights(I + 3, N, 14)
    w = w[:, 2:2 + I]
    x = ref.rows_of(4, I, 15)
    assert torch.equal(run(ctx, w, t, b, x, torch.float32), run(ctx, w.contiguous(), t, b, x, torch.float32))


@pytest.mark.parametrize("rows", [3, 14, 40, 270])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_bad_values_stay_in_their_row(ctx, rows, bad):
    I, N = 700, 180
    w, t, b = ref.weights(I, N, 16)
    for dtype in (torch.float32, torch.bfloat16):
        x = ref.rows_of(rows, I, 17, dtype)
        clean = run(ctx, w, t, b, x, torch.float32)
        x[1, 400] = bad
        y = run(ctx, w, t, b, x, torch.float32)
        assert bool(y[1].isnan().all())
        keep = torch.arange(rows, device=DEV) != 1
        assert torch.equal(y[keep], clean[keep])


def test_bad_weights_stay_in_their_channels(ctx):
    I, N = 300, 200
    w, t, b = ref.weights(I, N, 18)
    x = ref.rows_of(6, I, 19)
    clean = run(ctx, w, t, b, x, torch.float32)
    codes = w.clone().view(torch.uint8)
    codes[77, 200] = 0x7F   # NaN
    y = run(ctx, codes.view(ref.E4M3), t, b, x, torch.float32)
    keep = torch.arange(N, device=DEV) != 77
    assert bool(y[:, 77].isnan().all()) and torch.equal(y[:, keep], clean[:, keep])
    f = w.float()
    f[10, 5] = INF   # its 128 x 128 block has no finite scale
    y = run(ctx, f, None, b, x, torch.float32)
    assert bool(y[:, :128].isnan().all()) and not bool(y[:, 128:].isnan().any())


@pytest.mark.parametrize("size", [2.0 ** -149, 1e-36, 1e-30, 1e30, 3e38])
@pytest.mark.parametrize("rows", [2, 40])
def test_extreme_rows(ctx, size, rows):
    """Rows whose scales stand at the ends of float32."""
    I, N = 256, 64
    w, t, _ = ref.weights(I, N, 20, bias=False)
    x = (ref.rows_of(rows, I, 21).clamp(-1, 1) * size)
    q, s = ref.round_rows(x)
    z, mag = ref.product(q, s, w, t)
    y = run(ctx, w, t, None, x, torch.float32)
    # a term whose scales' product, or which itself, lies below 2^-126 is off by steps of 2^-149
    small = 2.0 ** -149 * (448.0 * 448.0 * 128 + I)
    # sums are FP32: outputs of which a block's term or the sum of the two passes its range are not asked for
    parts = [ref.product(q[:, k:k + 128], s[:, k // 128:k // 128 + 1], w[:, k:k + 128], t[:, k // 128:k // 128 + 1])[0] for k in (0, 128)]
    inside = torch.stack([v.abs() for v in (*parts, z)]).amax(0) < torch.finfo(torch.float32).max * (1 - 2.0 ** -10)
    assert bool(inside.any())
    ref.check(y[inside], z[inside], (ref.unit(I) * mag + small)[inside], size)


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
def test_codes_of_every_value(ctx, rows):
    """Every e4m3 code against every other one (subnormals among them)."""
    codes = torch.arange(256, device=DEV, dtype=torch.uint8)
    codes = codes[(codes & 0x7F) != 0x7F]
    q = codes[(torch.arange(rows, device=DEV)[:, None] + torch.arange(254, device=DEV)) % 254].view(ref.E4M3)
    w = codes[(3 * torch.arange(64, device=DEV)[:, None] + torch.arange(254, device=DEV)) % 254].view(ref.E4M3)
    s = torch.ones(rows, 2, device=DEV)
    t = torch.ones(1, 2, device=DEV)
    z, mag = ref.product(q, s, w, t)
    ref.check(run(ctx, w, t, None, q, torch.float32, s), z, ref.unit(254) * mag, rows)
    # one input alone: the product itself is exact
    for i in (0, 1, 7, 100, 253):
        one = torch.zeros_like(q.view(torch.uint8))
        one[:, i] = q.view(torch.uint8)[:, i]
        one = one.view(ref.E4M3)
        assert torch.equal(run(ctx, w, t, None, one, torch.float32, s).double(), ref.product(one, s, w, t)[0]), i


@pytest.mark.parametrize("rows", [1, 3, 12, 60, 300])
def test_graph_on_another_stream(ctx, rows):
    """A captured plan on a stream of its own, replayed with new rows, against the eager call."""
    I, N = 1025, 140
    w, t, b = ref.weights(I, N, 22)
    stream = torch.cuda.Stream()
    handle = runtime.Fp8Weights(ctx, w, t, bias=b)
    x = ref.rows_of(rows, I, 23)
    y = torch.zeros(rows, N, device=DEV)
    torch.cuda.synchronize()
    plan = runtime.Fp8LinearPlan(handle, x, y, stream=stream)
    with torch.cuda.stream(stream):
        plan.submit()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        plan.submit()
    for seed in range(4):
        x.copy_(ref.rows_of(rows, I, 30 + seed))
        y.fill_(NAN)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(y)
        runtime.fp8_linear(handle, x, want)
        torch.cuda.synchronize()
        assert torch.equal(y, want), seed
    plan.destroy()
    handle.destroy()


def test_no_rows(ctx):
    w, t, b = ref.weights(64, 32, 24)
    handle = runtime.Fp8Weights(ctx, w, t, bias=b)
    runtime.fp8_linear(handle, torch.zeros(0, 64, device=DEV), torch.zeros(0, 32, device=DEV))
    handle.destroy()


def test_rows_far_apart(ctx):
    """Rows whose offsets pass 32 bits, in and out."""
    I, N, rows = 130, 40, 5
    stride = (1 << 31) // 4 + 4096   # elements of 4 bytes: the third row lies past 2^32 bytes
    w, t, b = ref.weights(I, N, 25)
    far = torch.empty(rows * stride, device=DEV)
    x, y = far.view(rows, stride)[:, :I], far.view(rows, stride)[:, 1024:1024 + N]
    x.copy_(ref.rows_of(rows, I, 26))
    out = torch.empty(rows * stride, device=DEV).view(rows, stride)[:, :N]
    handle = runtime.Fp8Weights(ctx, w, t, bias=b)
    near = torch.zeros(rows, N, device=DEV)
    runtime.fp8_linear(handle, x.contiguous(), near)
    runtime.fp8_linear(handle, x, out)
    torch.cuda.synchronize()
    assert torch.equal(out, near) and y.shape == near.shape
    handle.destroy()


def test_refusals(ctx):
    w, t, b = ref.weights(256, 64, 27)
    handle = runtime.Fp8Weights(ctx, w, t, bias=b)
    pair = runtime.Fp8Weights(ctx, w, t, up=w, up_scales=t)
    x, y = ref.rows_of(4, 256, 28), torch.zeros(4, 64, device=DEV)
    q, s = ref.round_rows(x)

    def refused(name, call, *args, **kw):
        with pytest.raises(abi.StrixError) as e:
            call(*args, **kw)
        assert e.value.name == name

    refused("INVALID_ARGUMENT", runtime.fp8_linear, pair, x, y)
    refused("INVALID_ARGUMENT", runtime.fp8_linear, handle, x, y, x_scales=s)
    refused("INSUFFICIENT_BUFFER", runtime.fp8_linear, handle, q, y)
    refused("INSUFFICIENT_BUFFER", runtime.fp8_linear, handle, q, y, x_scales=s[:, :1].contiguous())
    refused("UNSUPPORTED_FORMAT", runtime.fp8_linear, handle, x[:, :255], y)
    refused("UNSUPPORTED_FORMAT", runtime.fp8_linear, handle, x, y[:3])
    refused("INVALID_ARGUMENT", runtime.fp8_linear, handle, x, y, alpha=NAN)
    refused("INVALID_ARGUMENT", runtime.fp8_linear, handle, x, x[:, :64])
    refused("INSUFFICIENT_BUFFER", runtime.Fp8Weights, ctx, w)
    refused("INVALID_ARGUMENT", runtime.Fp8Weights, ctx, w.float(), t)
    refused("INVALID_ARGUMENT", runtime.Fp8Weights, ctx, w, t, up_scales=t)
    refused("INVALID_ARGUMENT", runtime.Fp8Weights, ctx, w, t, bias=b, up=w, up_scales=t)
    refused("UNSUPPORTED_FORMAT", runtime.Fp8Weights, ctx, w, t, up=w[:32], up_scales=t)
    plan = runtime.Fp8LinearPlan(handle, x, y)
    refused("INVALID_ARGUMENT", handle.destroy)   # the plan holds it
    plan.destroy()
    for h in (handle, pair):
        h.destroy()
    with pytest.raises(ValueError):
        runtime.int8_linear(handle, q, y)
    with pytest.raises(ValueError):
        runtime.fp8_linear(handle, x, y.to(ref.E4M3))
