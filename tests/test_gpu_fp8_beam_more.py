"""The e4m3 layers at sizes that take each of their tiles, operators that run side by side, and selection where its lists
run full or one beam holds every answer.  Definitions and tolerances as in the tests of each operator."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import fp8_ref as ref  # noqa: E402
import test_gpu_beam as beam  # noqa: E402
import test_gpu_fp8_gated as gated  # noqa: E402
import test_gpu_fp8_linear as linear  # noqa: E402
from strix_trellis import runtime  # noqa: E402

DEV = ref.DEV
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


# rows, inputs, channels (the contract test holds that such sizes take every tile)
LAYERS = [(9, 6933, 130), (9, 128, 17), (5, 4096, 4100), (33, 128, 4100), (65, 128, 4100), (33, 128, 12288),
          (2048, 130, 130), (333, 1000, 2307), (4096, 300, 300), (513, 500, 4100), (4096, 128, 300), (130, 128, 12288),
          (2048, 130, 8192)]
PAIRS = [(9, 128, 17), (5, 4096, 16), (1500, 128, 16), (2048, 130, 130), (2048, 1000, 130), (4096, 300, 130),
         (257, 128, 12288), (257, 2048, 4100), (4096, 128, 130), (65, 128, 5125), (1500, 130, 5125)]


@pytest.mark.parametrize("rows,I,N", LAYERS)
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_tiles(ctx, rows, I, N, out):
    linear.held(ctx, I, N, rows, torch.bfloat16, ref.TYPES[out], True, False)


@pytest.mark.parametrize("rows,I,N", PAIRS)
@pytest.mark.parametrize("out", ["f32", "bf16", "e4m3"])
def test_tiles_of_pairs(ctx, rows, I, N, out):
    gated.held(ctx, I, N, rows, torch.float16, ref.TYPES.get(out, ref.E4M3), "gelu" if rows % 2 else "silu")


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_bytes_stand_for_e4m3(ctx, rows):
    """uint8 tensors, as hosts without the type have them: the same bits."""
    I, N = 700, 260
    w, t, b = ref.weights(I, N, 1)
    u, ut, ub = ref.weights(I, N, 2)
    q, s = ref.round_rows(ref.rows_of(rows, I, 3))
    raw = lambda a: a.view(torch.uint8)
    plain = linear.run(ctx, w, t, b, q, torch.float32, s)
    assert torch.equal(plain, linear.run(ctx, raw(w), t, b, raw(q), torch.float32, s))
    outs = []
    for form in (lambda a: a, raw):
        handle = runtime.Fp8Weights(ctx, form(w), t, bias=b, up=form(u), up_scales=ut, up_bias=ub)
        y, ys = torch.zeros(rows, N, device=DEV, dtype=ref.E4M3), torch.zeros(rows, ref.blocks(N), device=DEV)
        runtime.fp8_gated(handle, form(q), form(y), x_scales=s, y_scales=ys)
        torch.cuda.synchronize()
        handle.destroy()
        outs.append((y.view(torch.uint8), ys))
    assert all(torch.equal(a, c) for a, c in zip(*outs))


@pytest.mark.parametrize("rows,I,N", [(3, 1152, 300), (5, 2176, 130), (9, 1024, 17), (9, 7040, 130), (9, 4096, 4100), (33, 128, 4100),
                                      (65, 128, 4100), (100, 1280, 640), (333, 1024, 2307), (700, 640, 130)])
def test_rows_of_e4m3_wherever_they_lie(ctx, rows, I, N):
    """Rows of whole blocks on 16-byte units are read in place, others are laid out first: the same bits, side by side or
    inside wider rows."""
    w, t, b = ref.weights(I, N, 30)
    q, s = ref.round_rows(ref.rows_of(rows, I, 31))
    for out in (torch.float32, torch.bfloat16):
        plain = linear.run(ctx, w, t, b, q, out, s)
        for left, right in ((16, 48), (1, 2), (0, 16)):
            wide = torch.full((rows, left + I + right), 127, device=DEV, dtype=torch.uint8).view(ref.E4M3)   # NaN
            wide[:, left:left + I] = q
            assert torch.equal(plain, linear.run(ctx, w, t, b, wide[:, left:left + I], out, s)), (out, left)
    z, mag = ref.product(q, s, w, t, b)
    ref.check(linear.run(ctx, w, t, b, q, torch.float32, s), z, ref.unit(I) * mag, (rows, I, N))


@pytest.mark.parametrize("rows", [2, 9, 40, 100, 300, 1100])
@pytest.mark.parametrize("I", [128, 1100, 1152])
def test_infinite_scales(ctx, rows, I):
    """A block's infinite scale, of a row or of weights, gives infinities of its products' signs (and NaN where a product
    is 0 or both signs meet), in every row and channel that has it."""
    N = 300
    w, t, _ = ref.weights(I, N, 40, bias=False)
    q, s = ref.round_rows(ref.rows_of(rows, I, 41))
    for last in (False, True):
        s2, t2 = s.clone(), t.clone()
        s2[0, -1 if last else 0] = INF
        t2[1, -1 if last else 0] = INF
        y = linear.run(ctx, w, t2, None, q, torch.float32, s2)
        part = slice(I - I % 128 if I % 128 else I - 128, I) if last else slice(0, 128)
        p = q[:, part].double() @ w[:, part].double().t().contiguous()
        hit = torch.zeros(rows, N, device=DEV, dtype=torch.bool)
        hit[0] = True
        hit[:, 128:256] = True
        assert bool((y[hit].double() == (p * INF)[hit]).logical_or(p[hit] == 0).all())
        assert bool(torch.isfinite(y[~hit]).all())


@pytest.mark.parametrize("rows", [2, 24, 280])
def test_two_graphs_of_one_layer(ctx, rows):
    """Two captured steps on the same weights, on streams of their own and at the same time: each has its own
    workspace."""
    I, N, V, beams = 513, 384, 4000, 2
    rows = rows // beams * beams
    layers = gated.pair_of(I, N, 4)
    handle = gated.handle_of(ctx, layers)
    w, t, _ = ref.weights(N, V, 6, bias=False)
    head = runtime.Fp8Weights(ctx, w, t)
    steps = []
    for k in range(2):
        stream = torch.cuda.Stream()
        x = ref.rows_of(rows, I, 7 + k)
        y, ys = torch.zeros(rows, N, device=DEV, dtype=ref.E4M3), torch.zeros(rows, ref.blocks(N), device=DEV)
        logits, scores = torch.zeros(rows, V, device=DEV), -torch.rand(rows, device=DEV)
        out = [torch.zeros(rows // beams, 5, device=DEV)] + [
            torch.zeros(rows // beams, 5, device=DEV, dtype=torch.int32) for _ in range(2)]
        torch.cuda.synchronize()
        plans = [runtime.Fp8GatedPlan(handle, x, y, y_scales=ys, stream=stream),
                 runtime.Fp8LinearPlan(head, y, logits, x_scales=ys, stream=stream),
                 runtime.BeamSelectPlan(ctx, logits, scores, *out, beams, stream=stream)]
        with torch.cuda.stream(stream):
            for p in plans:
                p.submit()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for p in plans:
                p.submit()
        steps.append((stream, x, y, ys, logits, scores, out, plans, graph))
    for seed in range(4):
        for k, (stream, x, *_) in enumerate(steps):
            x.copy_(ref.rows_of(rows, I, 20 + 2 * seed + k))
        torch.cuda.synchronize()
        for _ in range(5):
            for stream, *_, graph in steps:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for stream, x, y, ys, logits, scores, out, plans, graph in steps:
            h, hs = torch.zeros_like(y), torch.zeros_like(ys)
            runtime.fp8_gated(handle, x, h, y_scales=hs)
            z = torch.zeros_like(logits)
            runtime.fp8_linear(head, h, z, x_scales=hs)
            assert torch.equal(h.view(torch.uint8), y.view(torch.uint8)) and torch.equal(hs, ys) and torch.equal(z, logits)
            for a, c in zip(out, beam.select(ctx, z, scores, None, beams, 5)):
                assert torch.equal(a, c)
    for *_, plans, _ in steps:
        for p in plans:
            p.destroy()
    handle.destroy()
    head.destroy()


@pytest.mark.parametrize("rows,vocab", [(4, 129280), (2, 3000), (600, 9000)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rising_logits(ctx, rows, vocab, dtype):
    """Every token is larger than the ones before it: all of them pass the bound, and the lists run full.  (Steps of
    the type, so that BF16 has runs of equal ones, of which the lower tokens come first.)"""
    x = torch.arange(vocab, device=DEV, dtype=torch.float32).expand(rows, vocab).mul(2.0 ** -9).to(beam.TYPES[dtype])
    scores = -torch.arange(rows, device=DEV, dtype=torch.float32)
    got, _ = beam.check(ctx, x.contiguous(), scores, None, 2, 33)
    assert bool((got[1] >= 0).all())


@pytest.mark.parametrize("beams,vocab,keep", [(64, 30000, 64), (64, 500, 64), (7, 129280, 64), (2, 40000, 3)])
@pytest.mark.parametrize("at", [0, -1])
def test_one_beam_holds_every_answer(ctx, beams, vocab, keep, at):
    """The others' candidates are all lower, so the winner's lists are read to their ends."""
    x, scores, _ = beam.inputs(2, beams, vocab, torch.float32, 9)
    scores -= 1000.0
    scores.view(2, beams)[:, at] += 900.0
    # and the winner's best tokens lie side by side, in one split
    x.view(2, beams, vocab)[:, at, vocab // 2:vocab // 2 + 70] += 20.0
    (v, p, t), _ = beam.check(ctx, x, scores, None, beams, keep)
    assert bool((p == at % beams).all())


def test_falling_candidates_of_many_beams(ctx):
    """64 beams x 8 splits x 64 tokens in full order: more candidates than one round of the join takes."""
    x, scores, _ = beam.inputs(1, 64, 66000, torch.float32, 10)
    beam.check(ctx, x, scores * 0, None, 64, 64)


def test_device_arrays_without_torch_tensors(ctx):
    """A step on the library's own arrays, e4m3 as bytes, against the same step on tensors."""
    import numpy as np
    from strix_trellis import device
    rng = np.random.default_rng(6)
    rows, beams, I, N, V = 6, 3, 200, 260, 900
    gate, up, head = (rng.standard_normal(s, dtype=np.float32) * 0.1 for s in ((N, I), (N, I), (V, N)))
    x, scores = rng.standard_normal((rows, I), dtype=np.float32), -rng.random(rows, dtype=np.float32)
    cache = rng.integers(0, 255, (2, rows, 3, 50), dtype=np.uint8)

    def step(put, empty, stream):
        pair = runtime.Fp8Weights(ctx, put(gate), None, up=put(up), stream=stream)
        down = runtime.Fp8Weights(ctx, put(head), None, stream=stream)
        h, hs, y = empty((rows, N), np.uint8), empty((rows, ref.blocks(N)), np.float32), empty((rows, V), np.float32)
        out = [empty((rows // beams, beams), t) for t in (np.float32, np.int32, np.int32)]
        states = put(cache)
        runtime.fp8_gated(pair, put(x), h, y_scales=hs, stream=stream)
        runtime.fp8_linear(down, h, y, x_scales=hs, stream=stream)
        runtime.beam_select(ctx, y, put(scores), *out, beams, stream=stream)
        runtime.beam_reorder(ctx, out[1], states, stream=stream)
        (stream or torch.cuda).synchronize()
        result = [a.numpy() if isinstance(a, device.DeviceArray) else a.cpu().numpy() for a in (h, hs, y, *out, states)]
        pair.destroy()
        down.destroy()
        return result

    own = step(device.DeviceArray.from_numpy, device.DeviceArray.empty, device.Stream(0))
    tensors = step(lambda a: torch.from_numpy(a).to(DEV),
                   lambda s, t: torch.zeros(s, device=DEV, dtype=getattr(torch, np.dtype(t).name)), None)
    assert all(np.array_equal(a, b) for a, b in zip(own, tensors))
    parents = own[4]
    want = cache.reshape(2, rows // beams, beams, 3, 50)
    want = np.stack([want[:, p, parents[p]] for p in range(rows // beams)], 1).reshape(cache.shape)
    assert np.array_equal(own[6], want)
