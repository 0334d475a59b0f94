"""Selection of beams' continuations and reordering of their states (strix_amd_beam_*).

Selection is held to its definition in 64 bits.  Whole numbers are equal wherever the 64-bit values of neighbours in the
order are farther apart than what the FP32 statistics may be off by: the log sum's relative error is at most 2^-20 (an
exponential of two steps for an argument of up to 2^7 with half a step, and sums of at most 300 additions a lane), so
orders that 2e-6 decides are not asked for; the scores are within 2e-6 and half a step of the type.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from strix_trellis import abi, runtime  # noqa: E402

DEV = "cuda:0"
INF, NAN = float("inf"), float("nan")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


def reference(x, scores, finished, beams, keep, pad, scale):
    """(values float64, parents, tokens, gap): gap[p][j] is how far place j's value is from its neighbours in the order
    (0 counts as far: an exact tie, which the indices decide)."""
    x, rows, vocab = x.double() * scale, x.shape[0], x.shape[1]
    most = x.amax(1, keepdim=True)
    d = x - most
    c = scores.double()[:, None] + d - torch.log(torch.exp(d).sum(1, keepdim=True))
    valid = torch.isfinite(most[:, 0]) & ~x.isnan().any(1)
    c = torch.where(valid[:, None], c, -INF)
    if finished is not None:
        over = finished != 0
        c[over] = -INF
    c = c.reshape(rows // beams, beams * vocab)
    ids = torch.arange(beams * vocab, device=DEV).expand(c.shape)
    extra = torch.full((rows // beams, beams), -INF, device=DEV, dtype=torch.float64)
    if finished is not None:
        extra = torch.where(over, scores.double(), -INF).reshape(-1, beams)
    # a beam's pad token stands at its place in the order of indices
    at = torch.arange(beams, device=DEV).expand(extra.shape) * vocab + min(max(pad, 0), vocab - 1)
    c, ids = torch.cat([c, extra], 1), torch.cat([ids, at], 1)
    by_id = torch.sort(ids, dim=1, stable=True).indices
    c, ids, is_pad = c.gather(1, by_id), ids.gather(1, by_id), (by_id >= beams * vocab)
    alive = torch.isfinite(scores).reshape(-1, beams)
    c = torch.where(alive.gather(1, ids // vocab), c, -INF)
    c = torch.nn.functional.pad(c, (0, max(0, keep + 1 - c.shape[1])), value=-INF)
    ids = torch.nn.functional.pad(ids, (0, c.shape[1] - ids.shape[1]))
    is_pad = torch.nn.functional.pad(is_pad, (0, c.shape[1] - is_pad.shape[1]))
    v, order = torch.sort(c, dim=1, descending=True, stable=True)
    v1 = torch.nn.functional.pad(v[:, :keep + 1], (1, 0), value=INF)
    gap = torch.minimum(v1[:, :-1] - v1[:, 1:], torch.nn.functional.pad(v1[:, 1:-1] - v1[:, 2:], (0, 1), value=INF)[:, :keep + 1])
    gap = torch.where(gap == 0, INF, gap).nan_to_num(INF)[:, :keep]
    v, order = v[:, :keep], order[:, :keep]
    live = v > -INF
    ids = ids.gather(1, order)
    tokens = torch.where(is_pad.gather(1, order), pad, ids % vocab)
    return v, torch.where(live, ids // vocab, -1).int(), torch.where(live, tokens, -1).int(), gap


def select(ctx, x, scores, finished, beams, keep, pad=0, scale=1.0):
    prompts = x.shape[0] // beams
    v = torch.full((prompts, keep), NAN, device=DEV)
    p = torch.full((prompts, keep), -7, device=DEV, dtype=torch.int32)
    t = torch.full((prompts, keep), -7, device=DEV, dtype=torch.int32)
    runtime.beam_select(ctx, x, scores, v, p, t, beams, finished=finished, pad=pad, scale=scale)
    torch.cuda.synchronize()
    return v, p, t


def check(ctx, x, scores, finished, beams, keep, pad=0, scale=1.0):
    got = select(ctx, x, scores, finished, beams, keep, pad, scale)
    v, p, t, gap = reference(x, scores, finished, beams, keep, pad, scale)
    sure = gap > 2e-6 * (1 + v.abs().nan_to_num(0, 0, 0))
    off = (got[0].double() - v).abs()
    assert bool(((off <= 2e-6 * (1 + v.abs())) | (got[0].double() == v)).all()), float(off.nan_to_num(0).max())
    assert bool(((got[1] == p) | ~sure).all()) and bool(((got[2] == t) | ~sure).all())
    # what is not sure is still a set of distinct candidates
    for row in range(p.shape[0]):
        pairs = [(int(a), int(b)) for a, b in zip(got[1][row], got[2][row]) if int(a) >= 0]
        assert len(set(pairs)) == len(pairs)
    return got, float(sure.double().mean())


def inputs(prompts, beams, vocab, dtype, seed, done=0.2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = prompts * beams
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 3
    scores = -torch.rand(rows, generator=g, device=DEV) * 6
    finished = (torch.rand(rows, generator=g, device=DEV) < done).to(torch.int32)
    return x.to(dtype), scores, finished


@pytest.mark.parametrize("prompts,beams,vocab,keep", [
    (1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 1, 6), (3, 2, 7, 64), (1, 4, 129280, 8), (5, 5, 1000, 10), (16, 8, 32000, 16),
    (2, 64, 8200, 64), (1, 64, 50257, 64), (40, 16, 8192, 32), (64, 8, 16389, 16), (1, 2, 20000, 64), (300, 4, 300, 8)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_selection(ctx, prompts, beams, vocab, keep, dtype):
    x, scores, finished = inputs(prompts, beams, vocab, TYPES[dtype], vocab + keep)
    for f in (None, finished):
        _, sure = check(ctx, x, scores, f, beams, keep, pad=min(3, vocab - 1), scale=1.25)
        assert sure > 0.9


def test_first_step(ctx):
    """A prompt's first step: one beam counts, the others stand at -inf."""
    x, scores, _ = inputs(3, 4, 5000, torch.float32, 1)
    scores.view(3, 4)[:, 0] = 0.0
    scores.view(3, 4)[:, 1:] = -INF
    (v, p, t), _ = check(ctx, x, scores, None, 4, 8)
    assert bool((p == 0).all())


def test_equal_beams(ctx):
    """Beams with the same logits and scores: every candidate is tied, and the lower beam comes first."""
    x, scores, _ = inputs(2, 1, 40000, torch.bfloat16, 2)
    x, scores = x.repeat_interleave(4, 0), scores.repeat_interleave(4, 0)
    (v, p, t), _ = check(ctx, x, scores, None, 4, 16)
    assert bool((p == torch.arange(16, device=DEV) % 4).all())
    assert bool((t.view(2, 4, 4) == t.view(2, 4, 4)[:, :, :1]).all())


def test_equal_logits(ctx):
    """More equal logits than any list holds: the lowest tokens."""
    x = torch.zeros(2, 30000, device=DEV)
    scores = torch.tensor([-1.0, -1.0], device=DEV)
    v, p, t = select(ctx, x, scores, None, 2, 40)
    assert bool((p == 0).all()) and bool((t == torch.arange(40, device=DEV)).all())


def test_masks(ctx):
    """Masked tokens are no candidates; rows that leave nothing, and rows without a distribution, offer nothing."""
    x, scores, _ = inputs(4, 2, 9000, torch.float32, 3)
    x[:, 6:] = -INF
    x[2] = -INF                  # prompt 1: one beam left
    x[4, 17] = NAN
    x[5, 3] = INF                # prompt 2: none
    scores[6] = NAN              # prompt 3: nor these
    scores[7] = INF
    (v, p, t), _ = check(ctx, x, scores, None, 2, 16)
    assert bool((p[0] >= 0).sum() == 12) and bool((p[1] == 1).sum() == 6)
    assert bool((p[2:] == -1).all()) and bool((t[2:] == -1).all()) and bool((v[2:] == -INF).all())
    assert bool((v[0, 12:] == -INF).all())
    x[0] = torch.finfo(torch.float32).min   # masks of the type's lowest value
    x[0, 4] = 1.0
    (v, p, t), _ = check(ctx, x, scores, None, 2, 7)


def test_finished(ctx):
    """All finished: the beams in the order of their scores, ties by beam; their logits are not read."""
    x = torch.full((4, 3000), NAN, device=DEV)
    scores = torch.tensor([-2.0, -1.0, -2.0, -5.0], device=DEV)
    finished = torch.tensor([1, 5, -1, 1], device=DEV, dtype=torch.int32)
    v, p, t = select(ctx, x, scores, finished, 4, 6, pad=-100)
    assert p.tolist() == [[1, 0, 2, 3, -1, -1]] and t.tolist() == [[-100] * 4 + [-1, -1]]
    assert v.tolist() == [[-1.0, -2.0, -2.0, -5.0, -INF, -INF]]


@pytest.mark.parametrize("scale", [2.0 ** -16, 0.1, 1.0, 300.0, 2.0 ** 16])
def test_scales(ctx, scale):
    x, scores, finished = inputs(2, 3, 10000, torch.float32, 4)
    got = select(ctx, x, scores, finished, 3, 9, scale=scale)
    v = reference(x, scores, finished, 3, 9, 0, scale)[0]
    # the distances are held in FP32 before the exponential
    assert bool(((got[0].double() - v).abs() <= 3e-6 * (1 + v.abs())).all())


def test_stride_and_neighbours(ctx):
    """Logits inside wider rows at an odd offset; memory around the outputs stays."""
    x, scores, _ = inputs(3, 4, 1003, torch.bfloat16, 5)
    wide = torch.full((12, 1010), 99.0, device=DEV, dtype=torch.bfloat16)
    wide[:, 3:1006] = x
    out = [torch.full((5, 8), -9.0, device=DEV), torch.full((5, 8), -9, device=DEV, dtype=torch.int32),
           torch.full((5, 8), -9, device=DEV, dtype=torch.int32)]
    runtime.beam_select(ctx, wide[:, 3:1006], scores, out[0][1:4], out[1][1:4], out[2][1:4], 4)
    torch.cuda.synchronize()
    for a, b in zip(out, select(ctx, x, scores, None, 4, 8)):
        assert torch.equal(a[1:4], b) and bool((a[0] == -9).all()) and bool((a[4] == -9).all())


def test_select_refusals(ctx):
    x, scores, finished = inputs(2, 3, 50, torch.float32, 6)
    v, i = torch.zeros(2, 4, device=DEV), torch.zeros(2, 4, device=DEV, dtype=torch.int32)
    j = torch.zeros_like(i)

    def refused(name, *args, **kw):
        with pytest.raises(abi.StrixError) as e:
            runtime.beam_select(ctx, *args, **kw)
        assert e.value.name == name

    refused("UNSUPPORTED_FORMAT", x.to(torch.int8), scores, v, i, j, 3)
    refused("INSUFFICIENT_BUFFER", x, scores[:5], v, i, j, 3)
    refused("INVALID_ARGUMENT", x, scores, v, i, i, 3)
    refused("INVALID_ARGUMENT", x, scores, v, i, j, 3, scale=0.0)
    refused("INVALID_ARGUMENT", x, scores, v, i, j, 3, scale=NAN)
    big = [torch.zeros(2, 65, device=DEV), torch.zeros(2, 65, device=DEV, dtype=torch.int32), torch.zeros(2, 65, device=DEV, dtype=torch.int32)]
    refused("UNSUPPORTED_FORMAT", x, scores, *big, 3)
    one = [torch.zeros(1, 4, device=DEV), torch.zeros(1, 4, device=DEV, dtype=torch.int32), torch.zeros(1, 4, device=DEV, dtype=torch.int32)]
    refused("UNSUPPORTED_FORMAT", x, scores, *one, 4)   # six rows are no prompts of four
    with pytest.raises(ValueError):
        runtime.beam_select(ctx, x, scores, v[:1], i, j, 3)


# ---- reordering ----


def states(shape, room, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    wide = torch.randint(-128, 128, (*shape[:3], shape[3] + room), generator=g, device=DEV).to(dtype)
    return wide


def moved(x, parents):
    prompts, beams = parents.shape
    own = torch.arange(beams, device=DEV).expand(prompts, beams)
    p = torch.where((parents >= 0) & (parents < beams), parents.long(), own)
    rows = (p + beams * torch.arange(prompts, device=DEV)[:, None]).reshape(-1)
    return x[:, rows]


@pytest.mark.parametrize("prompts,beams", [(1, 1), (3, 2), (2, 4), (5, 5), (2, 8), (1, 9), (3, 16), (1, 17), (2, 32), (1, 40), (2, 64)])
@pytest.mark.parametrize("outer,inner,width,room,dtype", [
    (1, 1, 1, 0, torch.uint8), (2, 3, 15, 4, torch.uint8), (1, 2, 4096, 0, torch.uint8), (3, 1, 4099, 13, torch.uint8),
    (2, 2, 1000, 24, torch.bfloat16), (1, 1, 5000, 1, torch.float32)])
def test_reorder(ctx, prompts, beams, outer, inner, width, room, dtype):
    g = torch.Generator(device=DEV).manual_seed(width + beams)
    # any beam, their own among them, and -1 and others that are none
    parents = torch.randint(-2, beams + 2, (prompts, beams), generator=g, device=DEV).to(torch.int32)
    for offset in (0, 3):
        wide = states((outer, prompts * beams, inner, width), room + 3, dtype, beams)
        keep = wide.clone()
        x = wide[..., offset:offset + width]
        want = moved(x, parents)
        other = torch.zeros_like(wide)
        runtime.beam_reorder(ctx, parents, x, other[..., 1:1 + width])
        torch.cuda.synchronize()
        assert torch.equal(other[..., 1:1 + width], want) and torch.equal(wide, keep)
        assert not bool(other[..., :1].any()) and not bool(other[..., 1 + width:].any())
        runtime.beam_reorder(ctx, parents, x)
        torch.cuda.synchronize()
        assert torch.equal(x, want)
        assert torch.equal(wide[..., :offset], keep[..., :offset])
        assert torch.equal(wide[..., offset + width:], keep[..., offset + width:])


def test_reorder_cycles_in_place(ctx):
    """Swaps, cycles and one beam taken by all others."""
    for parents in ([[1, 0, 3, 2]], [[1, 2, 3, 0]], [[3, 3, 3, 3]], [[0, 0, 1, 2]], [[0, 1, 2, 3]]):
        parents = torch.tensor(parents, device=DEV, dtype=torch.int32)
        x = states((2, 4, 2, 777), 0, torch.int32, 1)
        want = moved(x, parents)
        runtime.beam_reorder(ctx, parents, x, x)
        torch.cuda.synchronize()
        assert torch.equal(x, want), parents


def test_reorder_other_orders(ctx):
    """Dimensions in another order in memory: rows outermost, inner ahead of outer; a source that is one state for all."""
    base = torch.randint(-99, 99, (6, 3, 2, 50), device=DEV, dtype=torch.int16)
    x = base.permute(1, 0, 2, 3)   # [outer 3, rows 6, inner 2, 50]
    parents = torch.tensor([[2, 0, 0], [1, 1, 0]], device=DEV, dtype=torch.int32)
    want = moved(x, parents)
    runtime.beam_reorder(ctx, parents, x)
    torch.cuda.synchronize()
    assert torch.equal(x, want)
    one = torch.randint(-99, 99, (3, 1, 2, 50), device=DEV, dtype=torch.int16).expand(3, 6, 2, 50)
    y = torch.zeros(3, 6, 2, 50, device=DEV, dtype=torch.int16)
    runtime.beam_reorder(ctx, parents, one, y)
    torch.cuda.synchronize()
    assert torch.equal(y, one.contiguous())


def test_reorder_far_offsets(ctx):
    """Rows and pieces past 2^32 bytes."""
    stride = (1 << 31) + 4096
    far = torch.zeros(4 * stride, device=DEV, dtype=torch.uint8)
    x = far.view(1, 4, 1, stride)[..., stride - 2000:]
    x.copy_(torch.randint(0, 256, (1, 4, 1, 2000), device=DEV, dtype=torch.uint8))
    parents = torch.tensor([[3, 0, 1, 2]], device=DEV, dtype=torch.int32)
    want = moved(x, parents)
    runtime.beam_reorder(ctx, parents, x)
    torch.cuda.synchronize()
    assert torch.equal(x, want)


def test_reorder_many_pieces(ctx):
    """More pieces, and more prompts, than a side of a launch's grid."""
    for outer, prompts, inner in ((300, 2, 250), (1, 33000, 1), (2, 40, 33000)):
        parents = torch.randint(0, 2, (prompts, 2), device=DEV).to(torch.int32)
        x = torch.randint(0, 256, (outer, prompts * 2, inner, 5), device=DEV, dtype=torch.uint8)
        want = moved(x, parents)
        runtime.beam_reorder(ctx, parents, x)
        torch.cuda.synchronize()
        assert torch.equal(x, want)


def test_reorder_refusals(ctx):
    x = torch.zeros(1, 4, 1, 64, device=DEV)
    parents = torch.zeros(1, 4, device=DEV, dtype=torch.int32)

    def refused(name, *args):
        with pytest.raises(abi.StrixError) as e:
            runtime.beam_reorder(ctx, *args)
        assert e.value.name == name

    refused("INVALID_ARGUMENT", parents, x[..., :32], x[..., 16:48])         # overlapping, not the same
    refused("UNSUPPORTED_FORMAT", parents, x, x[:, :1].expand(1, 4, 1, 64).clone()[:, :1].expand(1, 4, 1, 64))
    refused("UNSUPPORTED_FORMAT", torch.zeros(1, 65, device=DEV, dtype=torch.int32), torch.zeros(1, 65, 1, 4, device=DEV))
    with pytest.raises(ValueError):
        runtime.beam_reorder(ctx, parents, x[:, :3])
    with pytest.raises(ValueError):
        runtime.beam_reorder(ctx, parents.float(), x)
    with pytest.raises(ValueError):
        runtime.beam_reorder(ctx, parents, x.transpose(1, 3))
    runtime.beam_reorder(ctx, torch.zeros(0, 4, device=DEV, dtype=torch.int32), x[:, :0])   # nothing to move


def test_a_step_in_a_graph(ctx):
    """head (e4m3) -> selection -> reordering of a cache in place, captured and replayed; every replay against the eager
    calls on a copy."""
    import fp8_ref as ref
    prompts, beams, D, V = 3, 4, 256, 5003
    rows = prompts * beams
    w, t, _ = ref.weights(D, V, 1, bias=False)
    head = runtime.Fp8Weights(ctx, w, t)
    stream = torch.cuda.Stream()
    x, logits = ref.rows_of(rows, D, 2), torch.zeros(rows, V, device=DEV)
    scores = -torch.rand(rows, device=DEV)
    out = [torch.zeros(prompts, beams, device=DEV), torch.zeros(prompts, beams, device=DEV, dtype=torch.int32),
           torch.zeros(prompts, beams, device=DEV, dtype=torch.int32)]
    cache = states((2, rows, 2, 640), 0, torch.bfloat16, 3)
    torch.cuda.synchronize()
    steps = [runtime.Fp8LinearPlan(head, x, logits, stream=stream),
             runtime.BeamSelectPlan(ctx, logits, scores, *out, beams, stream=stream),
             runtime.BeamReorderPlan(ctx, out[1], cache, stream=stream)]
    start = cache.clone()
    with torch.cuda.stream(stream):
        for p in steps:
            p.submit()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for p in steps:
            p.submit()
    for seed in range(3):
        x.copy_(ref.rows_of(rows, D, 10 + seed))
        cache.copy_(start)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.zeros_like(logits)
        runtime.fp8_linear(head, x, eager)
        torch.cuda.synchronize()
        assert torch.equal(eager, logits)
        for a, b in zip(out, select(ctx, eager, scores, None, beams, beams)):
            assert torch.equal(a, b)
        assert torch.equal(cache, moved(start, out[1]))
    for p in steps:
        p.destroy()
    head.destroy()
