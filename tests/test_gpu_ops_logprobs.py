"""Token log probabilities (strix_amd_token_logprobs) against the definition in 64 bits.

Tolerances.  With u = 2^-24 and V logits: a weight e^(c d) is off by 3 u |c d| from its exponent (the rounded d, c
and product) and 4 u from exp2f; a thread adds V / 512 of them, the joins of 64 lanes, 8 waves and up to V / 8192
splits rescale and add with under 4 roundings each.  The weights' mean |c d| is at most ln V + 2 where they matter
(farther ones weigh less than 1 / V).  So log sum is off by at most u (V / 512 + 4 (14 + V / 8192) + 2 ln V + 20)
=: e, a log probability by e + 4 u of its magnitude, and the entropy by e (2 + ln V): the third u |c d| is in the 4
per level, since the twelve levels of lanes and waves add without rescaling, one rounding each, and leave 36 u.
Whole numbers are exact.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from strix_trellis import abi, runtime  # noqa: E402

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


def outputs(rows, top):
    return {"logprobs": torch.full((rows,), 9.0, device=DEV), "ranks": torch.full((rows,), 9, dtype=torch.int32, device=DEV),
            "entropy": torch.full((rows,), 9.0, device=DEV),
            "top_ids": torch.full((rows, top), 9, dtype=torch.int32, device=DEV) if top else None,
            "top_logprobs": torch.full((rows, top), 9.0, device=DEV) if top else None}


def check(x, tokens, got, scale, what):
    """Outputs of rows that have a distribution."""
    x, tokens = x.cpu(), tokens.cpu().long()
    V = x.shape[1]
    e = U * (V / 512 + 4 * (14 + V / 8192) + 2 * math.log(V) + 20)
    l = scale * (x.double() - x.double().amax(1, keepdim=True))   # the largest first: 64 bits hold what is left
    logp = l - torch.logsumexp(l, 1, keepdim=True)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)

    def close(a, b, tol, name):
        a = a.cpu().double()
        same = (a == b) | (((a - b).abs() <= tol) & torch.isfinite(b))
        assert bool(same.all()), (what, name, a[~same][:4], b[~same][:4])

    given = logp.gather(1, tokens[:, None])[:, 0]
    close(got["logprobs"], given, e + 4 * U * given.abs(), "logprobs")
    close(got["entropy"], entropy, e * (2 + math.log(V)), "entropy")
    xt = x.gather(1, tokens[:, None])
    ranks = ((x > xt) | ((x == xt) & (torch.arange(V) < tokens[:, None]))).sum(1)
    assert torch.equal(got["ranks"].cpu().long(), ranks), (what, "ranks")
    if got["top_ids"] is not None:
        top = got["top_ids"].shape[1]
        order = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(got["top_ids"].cpu().long(), order), (what, "top_ids")
        best = logp.gather(1, order)
        close(got["top_logprobs"], best, e + 4 * U * best.abs(), "top_logprobs")


# vocabularies on and off the batch and split boundaries; few rows (split) and many
@pytest.mark.parametrize("rows,vocab", [(1, 129280), (1, 1), (2, 2), (3, 63), (1, 8191), (4, 8192), (2, 8193), (5, 16385),
                                        (1, 32000), (33, 50257), (7, 100277), (520, 9001), (600, 257), (1100, 1000)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_against_definition(ctx, rows, vocab, name):
    g = torch.Generator().manual_seed(rows * 31 + vocab)
    x = (3.0 * torch.randn(rows, vocab, generator=g)).to(TYPES[name])
    tokens = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    for top, scale in ((min(20, vocab), 1.0), (min(64, vocab), 1.7), (1, 0.3), (0, 1.0)):
        got = outputs(rows, top)
        runtime.token_logprobs(ctx, x.to(DEV), tokens=tokens.to(DEV), scale=scale, **got)
        check(x, tokens, got, scale, (rows, vocab, name, top))


def test_masked_and_tied_logits(ctx):
    inf = float("inf")
    for V, rows in ((40000, 6), (300, 6), (9000, 530)):
        g = torch.Generator().manual_seed(V)
        x = torch.randn(rows, V, generator=g)
        x[0] = 1.25                                        # all equal: ids in order
        x[1] = -inf
        x[1, [V - 1, 17, 5]] = torch.tensor([0.5, 0.5, -2.0])   # fewer tokens than asked for
        x[2] = torch.randint(0, 3, (V,), generator=g).float()   # long ties
        x[3] = torch.finfo(torch.float32).min              # a mask of the lowest value everywhere: uniform
        x[4] = torch.arange(V).float() * 1e-3              # rising: every batch beats the one before
        x[5, ::2] = -inf
        x[5, 1] = -0.0
        x[5, 3] = 0.0                                      # equal to -0
        x[5, 5:] = -x[5, 5:].abs() - 1e-3
        x[5, ::2] = -inf
        tokens = torch.randint(0, V, (rows,), generator=g, dtype=torch.int32)
        tokens[0], tokens[1], tokens[5] = V - 1, 8, 3      # a masked token: log probability -inf
        for top in (1, 20, 64):
            got = outputs(rows, top)
            runtime.token_logprobs(ctx, x.to(DEV), tokens=tokens.to(DEV), **got)
            check(x, tokens, got, 1.0, (V, top))
            assert float(got["logprobs"][1]) == -inf
    x = torch.zeros(2, 100000)                             # 16-bit ties beyond the candidate list
    x[1, ::3] = 1.0
    tokens = torch.tensor([99999, 1], dtype=torch.int32)
    for dtype in TYPES.values():
        got = outputs(2, 40)
        runtime.token_logprobs(ctx, x.to(dtype).to(DEV), tokens=tokens.to(DEV), **got)
        check(x, tokens, got, 1.0, dtype)


def test_confident_rows_keep_their_digits(ctx):
    """One token far ahead: entropy and 1 - p are tiny and have to be right in their own digits."""
    V = 20000
    x = torch.zeros(3, V)
    x[0, 777], x[1, 0], x[2, V - 1] = 25.0, 35.0, 45.0
    tokens = torch.tensor([777, 0, V - 1], dtype=torch.int32)
    got = outputs(3, 2)
    runtime.token_logprobs(ctx, x.to(DEV), tokens=tokens.to(DEV), **got)
    for r, gap in enumerate((25.0, 35.0, 45.0)):
        rest = (V - 1) * math.exp(-gap)
        logp = -math.log1p(rest)
        entropy = math.log1p(rest) + rest * gap / (1 + rest)
        assert abs(float(got["logprobs"][r]) - logp) <= 1e-5 * abs(logp)
        assert abs(float(got["entropy"][r]) - entropy) <= 1e-5 * entropy


def test_rows_without_a_distribution(ctx):
    inf, nan = float("inf"), float("nan")
    for V in (500, 40000):
        x = torch.randn(5, V)
        x[0] = -inf
        x[1, V // 2] = nan
        x[2, V - 1] = inf
        x[3, 0] = -nan
        x[3, 5] = -inf
        tokens = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32)
        got = outputs(5, 4)
        runtime.token_logprobs(ctx, x.to(DEV), tokens=tokens.to(DEV), **got)
        for k in ("logprobs", "entropy", "top_logprobs"):
            assert bool(torch.isnan(got[k][:4]).all()), k
        for k in ("ranks", "top_ids"):
            assert bool((got[k][:4] == -1).all()), k
        check(x[4:], tokens[4:], {k: v[4:] for k, v in got.items()}, 1.0, V)
        # tokens outside the vocabulary: their own outputs alone
        got = outputs(2, 3)
        runtime.token_logprobs(ctx, x[[4, 4]].to(DEV), tokens=torch.tensor([-1, V], dtype=torch.int32, device=DEV), **got)
        assert bool(torch.isnan(got["logprobs"]).all()) and bool((got["ranks"] == -1).all())
        assert bool(torch.isfinite(got["entropy"]).all()) and bool((got["top_ids"] >= 0).all())


def test_strided_rows_and_single_outputs(ctx):
    V, rows = 12345, 3
    wide = torch.randn(rows, V + 77, device=DEV).half()
    x = wide[:, 33:33 + V]
    tokens = torch.tensor([0, V - 1, 6000], dtype=torch.int32, device=DEV)
    want = outputs(rows, 6)
    runtime.token_logprobs(ctx, x, tokens=tokens, **want)
    check(x, tokens, want, 1.0, "strided")
    for key in want:
        got = torch.zeros_like(want[key])
        runtime.token_logprobs(ctx, x, tokens=tokens if key in ("logprobs", "ranks") else None, **{key: got})
        assert torch.equal(got, want[key]), key


def test_plans_streams_and_graphs(ctx):
    stream = torch.cuda.Stream()
    made = []
    for rows, V in ((1, 129280), (40, 5000), (513, 700)):
        xs = [torch.randn(rows, V, device=DEV) * (k + 1) for k in range(3)]
        tokens = torch.randint(0, V, (rows,), dtype=torch.int32, device=DEV)
        want = []
        for x in xs:
            want.append(outputs(rows, 5))
            runtime.token_logprobs(ctx, x, tokens=tokens, **want[-1])
        x, got = torch.zeros(rows, V, device=DEV), outputs(rows, 5)
        made.append((xs, want, x, got, runtime.TokenLogprobsPlan(ctx, x, tokens=tokens, stream=stream, **got)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for m in made:
            m[-1].submit()
    torch.cuda.synchronize()
    for rep in range(6):
        for xs, want, x, got, _ in made:
            x.copy_(xs[rep % 3])
            for v in got.values():
                v.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for xs, want, x, got, _ in made:
            for k in got:
                assert torch.equal(got[k], want[rep % 3][k]), (rep, k)
    for m in made:
        m[-1].destroy()


def test_refusals(ctx):
    x = torch.randn(4, 100, device=DEV)
    tokens = torch.zeros(4, dtype=torch.int32, device=DEV)

    def status(logits=x, **kw):
        with pytest.raises(abi.StrixError) as e:
            runtime.token_logprobs(ctx, logits, **kw)
        return e.value.name

    out = torch.empty(4, device=DEV)
    assert status() == "INVALID_ARGUMENT"                                       # no output
    assert status(logprobs=out) == "INVALID_ARGUMENT"                           # no tokens
    assert status(tokens=tokens[:3], logprobs=out) == "INSUFFICIENT_BUFFER"
    assert status(tokens=tokens, logprobs=out[:3]) == "INSUFFICIENT_BUFFER"
    assert status(entropy=out, scale=0.0) == "INVALID_ARGUMENT"
    assert status(entropy=out, scale=float("nan")) == "INVALID_ARGUMENT"
    assert status(entropy=out, scale=1e6) == "INVALID_ARGUMENT"
    assert status(top_logprobs=torch.empty(4, 65, device=DEV)) == "UNSUPPORTED_FORMAT"
    assert status(logits=x[:, :3], top_logprobs=torch.empty(4, 4, device=DEV)) == "UNSUPPORTED_FORMAT"
    assert status(tokens=tokens, logprobs=out, entropy=out) == "INVALID_ARGUMENT"
    assert status(logits=x.to(torch.int8), entropy=out) == "UNSUPPORTED_FORMAT"
    big = torch.randn(1, 100000, device=DEV)
    assert status(logits=big, entropy=out[:1], workspace=torch.zeros(64, dtype=torch.uint8, device=DEV)) == \
        "INSUFFICIENT_BUFFER"
    runtime.token_logprobs(ctx, x[:0], entropy=out[:0])                         # no rows
    torch.cuda.synchronize()
