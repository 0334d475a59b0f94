"""Token log probabilities of logits that are finite but farther apart than FP32 holds: small `scale`s bring their
distance back into range, so the log probability is finite.  Tolerances are those of the operator's own test."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_ops_logprobs as logprobs  # noqa: E402
from strix_trellis import runtime  # noqa: E402

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


@pytest.mark.parametrize("V", [50, 700, 40000])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_distances_past_the_range(ctx, V, name):
    g = torch.Generator().manual_seed(V)
    most = torch.finfo(logprobs.TYPES[name]).max
    x = 1e38 * torch.rand(5, V, generator=g)
    x[0, 3], x[0, 7] = 3e38, -3e38
    x[1, V - 1], x[1, 0] = most, -most                 # a mask of the lowest value below the largest one
    x[2] = -most
    x[2, 9] = most
    x[3] = torch.randn(V, generator=g)                 # an ordinary row
    x[4, 4], x[4, 11], x[4, 12] = 3e38, -2e38, -float("inf")
    x = x.to(logprobs.TYPES[name])
    tokens = torch.tensor([7, 0, 30, 5, 11], dtype=torch.int32)
    for scale in (2.0 ** -16, 0.01, 0.25):
        for top in (2, 40):
            got = logprobs.outputs(5, top)
            runtime.token_logprobs(ctx, x.to(DEV), tokens=tokens.to(DEV), scale=scale, **got)
            logprobs.check(x, tokens, got, scale, (V, name, scale))
            assert bool(torch.isfinite(got["logprobs"]).all())
    # a masked token keeps its -inf
    tokens[4] = 12
    got = logprobs.outputs(5, 0)
    runtime.token_logprobs(ctx, x.to(DEV), tokens=tokens.to(DEV), scale=0.01, **got)
    logprobs.check(x, tokens, got, 0.01, (V, name, "masked"))
    assert float(got["logprobs"][4]) == -float("inf")
