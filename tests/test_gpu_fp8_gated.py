"""The gated half of a feed-forward block on e4m3 weights (strix_amd_fp8_gated) against its definition in 64 bits.

Tolerances.  g and u are products with tolerances dg and du (tests/fp8_ref.py).  |act'| is at most 1.13 for both
activations, and act's own evaluation is within 2^-19 of its value (an exponential of a few steps, a reciprocal of
one, and, for gelu, a polynomial whose rounding, 3 steps of its argument z <= 100, the exponential passes on as a
relative error; beyond, the factor is 0 or 1).  So |h - exact| <= (1.13 dg)(|u| + du) + |act(g)| du + 2^-19 |h|, where the last is
taken at the largest |h| that the other two allow.  e4m3: the scale is that of the largest |h| of the block, and q s is within half a
step of h, 2^-4 of |h| or 2^-10 s, beside the rounding of h / s and the scale.
"""
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


def pair_of(I, N, seed, bias=True):
    return ref.weights(I, N, seed, bias), ref.weights(I, N, seed + 100, bias)


def handle_of(ctx, layers):
    (w, t, b), (u, ut, ub) = layers
    return runtime.Fp8Weights(ctx, w, t, bias=b, up=u, up_scales=ut, up_bias=ub)


def reference(layers, q, s, kind, out=torch.float32):
    """(h, its tolerance), float64."""
    I = q.shape[1]
    (g, g_mag), (u, u_mag) = (ref.product(q, s, w, t, b) for w, t, b in layers)
    dg, du = ref.unit(I, out) * g_mag, ref.unit(I, out) * u_mag
    h = ref.act(g, kind) * u
    off = 1.13 * dg * (u.abs() + du) + ref.act(g, kind).abs() * du
    return h, off + 2.0 ** -19 * (h.abs() + off)


def check(y, scales, h, tol, what):
    if scales is None:
        return ref.check(y, h, tol, what)
    N = h.shape[1]
    pad = ref.blocks(N) * 128 - N
    most = torch.nn.functional.pad(h.abs(), (0, pad)).reshape(h.shape[0], -1, 128).amax(2)
    off = torch.nn.functional.pad(tol, (0, pad)).reshape(h.shape[0], -1, 128).amax(2)
    assert bool(((scales.double() - most / 448.0).abs() <= off / 448.0 + most / 448.0 * 2.0 ** -22 + 2.0 ** -126).all()), what
    s = ref.spread(scales.double(), h.shape[0], N)
    got = y.double() * s
    step = torch.maximum((h.abs() + tol) * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -20)
    bad = ~((got - h).abs() <= step + tol)
    assert not bool(bad.any()), (what, int(bad.sum()))


def run(handle, x, N, out, x_scales=None, activation="silu"):
    rows = x.shape[0]
    y = torch.zeros((rows, N), device=DEV, dtype=out)
    scales = torch.full((rows, ref.blocks(N)), NAN, device=DEV) if out == ref.E4M3 else None
    runtime.fp8_gated(handle, x, y, x_scales=x_scales, y_scales=scales, activation=activation)
    torch.cuda.synchronize()
    return y, scales


def held(ctx, I, N, rows, dtype, out, activation="silu", bias=True, given=False, seed=0):
    layers = pair_of(I, N, seed, bias)
    handle = handle_of(ctx, layers)
    x = ref.rows_of(rows, I, seed + 1, dtype)
    q, s = ref.round_rows(x)
    y, scales = run(handle, q if given else x, N, out, s if given else None, activation)
    handle.destroy()
    check(y, scales, *reference(layers, q, s, activation, out), (I, N, rows, dtype, out))


@pytest.mark.parametrize("I,N", [(1, 1), (5, 33), (128, 128), (129, 31), (300, 200), (1000, 515), (5119, 70), (9000, 40)])
@pytest.mark.parametrize("rows", [1, 2, 4, 6, 16, 17, 40, 65])
@pytest.mark.parametrize("out", ["f32", "e4m3"])
def test_shapes(ctx, I, N, rows, out):
    held(ctx, I, N, rows, torch.float32, ref.TYPES.get(out, ref.E4M3), seed=I + N)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("rows,activation", [(1, "gelu"), (4, "silu"), (11, "gelu"), (90, "gelu"), (300, "silu")])
def test_types(ctx, dtype, out, rows, activation):
    held(ctx, 650, 290, rows, ref.TYPES.get(dtype, torch.float32), ref.TYPES.get(out, ref.E4M3), activation,
         bias=rows % 2 == 0, given=dtype == "e4m3")


@pytest.mark.parametrize("I,N,rows", [(2048, 1152, 260), (515, 2307, 333), (4096, 640, 700), (256, 300, 2049), (130, 96, 4500)])
@pytest.mark.parametrize("out", ["bf16", "e4m3"])
def test_many_rows(ctx, I, N, rows, out):
    held(ctx, I, N, rows, torch.bfloat16, ref.TYPES.get(out, ref.E4M3), "gelu" if N == 640 else "silu")


def test_more_rows_than_a_pass(ctx):
    held(ctx, 100, 40, 66000, torch.float16, ref.E4M3)


@pytest.mark.parametrize("rows", [2, 14, 40, 280])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_far_gates(ctx, rows, activation):
    """Gates over the whole range of the activations, up to where the exponential leaves float32."""
    I, N = 128, 160
    (w, t, _), up = pair_of(I, N, 5, bias=False)
    layers = (w, t, torch.linspace(-120, 120, N, device=DEV)), (up[0], up[1], torch.ones(N, device=DEV))
    handle = handle_of(ctx, layers)
    x = ref.rows_of(rows, I, 6) * 1e-3
    q, s = ref.round_rows(x)
    y, _ = run(handle, x, N, torch.float32, activation=activation)
    handle.destroy()
    h, tol = reference(layers, q, s, activation)
    # values below 2^-126 are off by steps of 2^-149, which u then scales
    check(y, None, h, tol + 2.0 ** -147, activation)


@pytest.mark.parametrize("rows", [3, 14, 40, 270])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_bad_values_stay_in_their_row(ctx, rows, bad):
    I, N = 300, 180
    handle = handle_of(ctx, pair_of(I, N, 7))
    x = ref.rows_of(rows, I, 8)
    for out in (torch.float32, ref.E4M3):
        clean, clean_s = run(handle, x, N, out)
        dirty = x.clone()
        dirty[1, 200] = bad
        y, scales = run(handle, dirty, N, out)
        keep = torch.arange(rows, device=DEV) != 1
        assert bool(y[1].float().isnan().all())
        assert torch.equal(y[keep].view(torch.uint8), clean[keep].view(torch.uint8))
        if scales is not None:
            assert bool(scales[1].isnan().all()) and torch.equal(scales[keep], clean_s[keep])
    handle.destroy()


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_strides(ctx, rows):
    I, N = 200, 141
    layers = pair_of(I, N, 9)
    handle = handle_of(ctx, layers)
    x = ref.rows_of(rows, I + 5, 10)[:, 3:3 + I]
    q, s = ref.round_rows(x)
    for out in (torch.bfloat16, ref.E4M3):
        h, tol = reference(layers, q, s, "silu", out)
        wide = torch.full((rows, N + 7), 1.5, device=DEV).to(out)
        scales = torch.zeros(rows, 2, device=DEV) if out == ref.E4M3 else None
        runtime.fp8_gated(handle, x, wide[:, 3:3 + N], y_scales=scales)
        torch.cuda.synchronize()
        check(wide[:, 3:3 + N], scales, h, tol, out)
        assert bool((wide[:, :3].float() == 1.5).all()) and bool((wide[:, 3 + N:].float() == 1.5).all())
    handle.destroy()


@pytest.mark.parametrize("rows", [1, 12, 50, 300])
def test_feed_forward_block(ctx, rows):
    """norm -> gated half, e4m3 -> second half, in one captured graph; each step against its definition on the values
    that the step before left."""
    D, H = 640, 900
    layers, (w2, t2, b2) = pair_of(D, H, 11, bias=False), ref.weights(H, D, 12)
    gated, down = handle_of(ctx, layers), runtime.Fp8Weights(ctx, w2, t2, bias=b2)
    stream = torch.cuda.Stream()
    residual, weight = ref.rows_of(rows, D, 13, torch.bfloat16), torch.ones(D, device=DEV)
    x = torch.zeros(rows, D, device=DEV, dtype=torch.bfloat16)
    h = torch.zeros(rows, H, device=DEV, dtype=ref.E4M3)
    hs = torch.zeros(rows, ref.blocks(H), device=DEV)
    y = torch.zeros(rows, D, device=DEV, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    steps = [runtime.BlockNormPlan(ctx, residual=residual, normed=x, pre_weight=weight, stream=stream),
             runtime.Fp8GatedPlan(gated, x, h, y_scales=hs, stream=stream),
             runtime.Fp8LinearPlan(down, h, y, x_scales=hs, stream=stream)]

    def submit():
        for p in steps:
            p.submit()

    with torch.cuda.stream(stream):
        submit()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        submit()
    for seed in range(3):
        residual.copy_(ref.rows_of(rows, D, 20 + seed, torch.bfloat16))
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        q, s = ref.round_rows(x)
        check(h, hs, *reference(layers, q, s, "silu", ref.E4M3), seed)
        z, mag = ref.product(h, hs, w2, t2, b2)
        ref.check(y, z, ref.unit(H, y.dtype) * mag, seed)
    for p in steps:
        p.destroy()
    gated.destroy()
    down.destroy()


def test_refusals(ctx):
    (w, t, b), (u, ut, ub) = pair_of(256, 64, 14)
    pair = runtime.Fp8Weights(ctx, w, t, bias=b, up=u, up_scales=ut, up_bias=ub)
    single = runtime.Fp8Weights(ctx, w, t, bias=b)
    x, y = ref.rows_of(4, 256, 15), torch.zeros(4, 64, device=DEV)
    q8, s8 = torch.zeros(4, 64, device=DEV, dtype=ref.E4M3), torch.zeros(4, 1, device=DEV)

    def refused(name, call, *args, **kw):
        with pytest.raises(abi.StrixError) as e:
            call(*args, **kw)
        assert e.value.name == name

    refused("INVALID_ARGUMENT", runtime.fp8_gated, single, x, y)
    refused("INVALID_ARGUMENT", runtime.fp8_gated, pair, x, y, y_scales=s8)
    refused("INSUFFICIENT_BUFFER", runtime.fp8_gated, pair, x, q8)
    refused("INVALID_ARGUMENT", runtime.fp8_gated, pair, x, q8, y_scales=x.view(-1)[:4])
    refused("UNSUPPORTED_FORMAT", runtime.fp8_gated, pair, x, y[:, :63])
    refused("UNSUPPORTED_FORMAT", runtime.fp8_gated, pair, x, y.to(torch.int8))
    with pytest.raises(KeyError):
        runtime.fp8_gated(pair, x, y, activation="relu")
    pair.destroy()
    single.destroy()
