"""Selection of beams' continuations at the ends of FP32: candidates below its range, temperatures at both ends of what
they may be, and joins that read their lists deep.

Tolerance of a value, c = score + scale (x - m) - log(sum): the sum alone is held in FP32.  An exponential's argument has
three half steps (the distance, scale log2 e, their product), 3 2^-24 z for an argument z = scale (m - x), which weighs
in with e^-z: 3 2^-24 times the mean of z, at most log(vocab) <= 12.  The exponential itself has two half steps, a sum one
for each of at most 40 additions.  So the logarithm is within 2^-24 (36 + 2 + 40) = 4.7e-6, or, as fewer tokens
count, within 2^-24 42 = 2.5e-6 where it is near 0; a score of FP32 has a half step, 2^-24 of it.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_beam as beam  # noqa: E402
from strix_trellis import runtime  # noqa: E402

DEV, INF, TYPES = beam.DEV, beam.INF, beam.TYPES


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


def expected(x, scores, finished, beams, keep, pad, scale):
    """Values in 64 bits, parents and tokens in order; a candidate that is -inf in FP32 is none."""
    v, p, t, gap = beam.reference(x, scores, finished, beams, keep, pad, scale)
    none = v.float() == -INF
    return v.masked_fill(none, -INF), p.masked_fill(none, -1), t.masked_fill(none, -1), gap


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [7, 5000, 40000])
def test_masks_of_the_lowest_value_scaled_past_fp32(ctx, dtype, vocab):
    """Logits masked by the type's lowest value, at a scale above 1: their values are below FP32, -inf, and so they are no
    candidates.  Each prompt has fewer tokens than places."""
    x, scores, _ = beam.inputs(3, 2, vocab, TYPES[dtype], 3)
    low = torch.finfo(TYPES[dtype]).min
    x[:, 3:] = low
    x[0] = low
    x[0, 2] = 1.0
    x[2:4] = low                 # prompt 1: all equal, so all in range, at -log(vocab)
    x[3, 1] = 0.0                # but where one is not
    got = beam.select(ctx, x, scores, None, 2, 9, scale=1.25)
    v, p, t, _ = expected(x, scores, None, 2, 9, 0, 1.25)
    assert int((p[0] >= 0).sum()) == 4 and int((p[1] >= 0).sum()) == min(9, vocab + 1)
    assert torch.equal(got[1], p) and torch.equal(got[2], t)
    assert bool(((got[0].double() - v).abs() <= 5e-6 * (1 + v.abs())).logical_or(got[0].double() == v).all())


def test_scores_that_leave_fp32(ctx):
    """Scores near the lowest value: what leaves FP32 is no candidate, a finished beam stays at its score, and what rounds
    to the lowest value is one."""
    x = torch.full((4, 300), torch.finfo(torch.float32).min, device=DEV)
    x[:, 7] = 0.0
    scores = torch.tensor([-2e38, -1.0, -3.4e38, -1e38], device=DEV)
    finished = torch.tensor([0, 0, 1, 0], device=DEV, dtype=torch.int32)
    v, p, t = beam.select(ctx, x, scores, finished, 4, 6, pad=11)
    # beam 1's masked tokens round to the lowest value, which is finite: the first three of them
    assert p.tolist() == [[1, 3, 0, 2, 1, 1]] and t.tolist() == [[7, 7, 7, 11, 0, 1]]
    assert bool(torch.isfinite(v).all())
    v, p, t = beam.select(ctx, x[[0, 3]].contiguous(), scores[[0, 3]].contiguous(), None, 2, 6)
    assert p.tolist() == [[1, 0, -1, -1, -1, -1]] and t.tolist() == [[7, 7, -1, -1, -1, -1]]
    assert bool((v[0, 2:] == -INF).all())


@pytest.mark.parametrize("scale", [2.0 ** -16, 0.1, 1.0, 300.0, 2.0 ** 16])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_scales_with_their_tokens(ctx, scale, dtype):
    """The permitted temperatures: each place's value, and its token, which has that value.  Within a beam the tokens are its
    first ones in the order of the logits, whose distances the statistics do not touch."""
    beams, keep, vocab = 3, 9, 10000
    x, scores, finished = beam.inputs(2, beams, vocab, TYPES[dtype], 4)
    got = beam.select(ctx, x, scores, finished, beams, keep, pad=5, scale=scale)
    v = beam.reference(x, scores, finished, beams, keep, 5, scale)[0]
    tol = 5e-6 * (1 + v.abs())
    assert bool(((got[0].double() - v).abs() <= tol).logical_or(got[0].double() == v).all())
    log_p = torch.log_softmax(x.double() * scale, 1)
    order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices
    for prompt in range(2):
        taken = [0] * beams
        for j in range(keep):
            value, b, token = float(got[0][prompt, j]), int(got[1][prompt, j]), int(got[2][prompt, j])
            if b < 0:
                assert token == -1 and value == -INF
                continue
            row = prompt * beams + b
            if int(finished[row]):
                assert token == 5 and taken[b] == 0 and value == float(scores[row])
            else:
                assert token == int(order[row, taken[b]]), (prompt, j)
                assert abs(value - float(scores[row]) - float(log_p[row, token])) <= float(tol[prompt, j])
            taken[b] += 1


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lists", [1, 3])
def test_deep_lists_of_eight_splits(ctx, lists, dtype):
    """64 beams of 129280 tokens in eight splits: 512 lists of 64 keys, of which a round of the join takes two each.  The
    64 places go to a few lists, which have to be read to their ends."""
    beams, vocab, keep = 64, 129280, 64
    x, scores, _ = beam.inputs(1, beams, vocab, TYPES[dtype], 10)
    scores = torch.full_like(scores, -1000.0)
    for row, at, n in [(5, 40000, 64)] if lists == 1 else [(5, 40000, 30), (5, 80000, 30), (63, 129200, 30)]:
        x[row, at:at + n] += 30.0
        scores[row] = 0.0
    (v, p, t), _ = beam.check(ctx, x, scores, None, beams, keep)
    assert bool(((p == 5) | (p == 63)).all())


def test_falling_candidates_of_eight_splits(ctx):
    """512 lists in full order, no beam ahead of another."""
    x, scores, _ = beam.inputs(1, 64, 129280, torch.float32, 10)
    beam.check(ctx, x, scores * 0, None, 64, 64)
