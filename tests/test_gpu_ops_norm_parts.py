"""Every instance of the block norm with every part: gates, channel scales and biases where a row takes several groups
of channels to a thread, where its last group is ragged, and where gates and weights are loaded late; in place and
not.  Tolerances are those of the operator's own test."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_ops_norm as norm  # noqa: E402
from strix_trellis import runtime  # noqa: E402

DEV = "cuda:0"

# both ends of each of the twelve instances' widths, and a width inside whose last waves hold no channel
WIDTHS = [2, 256, 257, 1024, 1025, 2048, 2049, 4096, 4097, 4099, 6144, 6145, 8192, 8193, 8195, 12288, 12289, 16384, 16385,
          20480, 20481, 24576, 24577, 28672, 28673, 28675, 32768]


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gate", ["full", "rows", "one_row"])
def test_every_part(ctx, width, name, gate):
    rows, dtype = 3, norm.TYPES[name]
    block, residual, r = norm.inputs(rows, width, dtype, width)
    shape = {"full": (rows, width), "rows": (rows, 1), "one_row": (1, width)}[gate]
    g = r(*shape).to(dtype).to(DEV)
    vec = lambda: r(width).to(DEV)  # noqa: E731
    few = {"post_weight": vec(), "pre_weight": vec()}
    every = few | {"post_bias": vec(), "pre_bias": vec(), "channel_scale": vec()}
    for kind, activation, p in (("layer", "sigmoid", every), ("rms", "linear", every), ("rms", "sigmoid", few),
                                ("layer", "linear", {"channel_scale": vec(), "pre_weight": vec()})):
        u, m, n, nm = norm.reference(block, residual, g, activation, p, kind == "layer", 1e-6, 0.5, 0.75, 1.25)
        call = {"gate": g, "gate_activation": activation, "kind": kind, "weight_offset": 0.5, "residual_scale": 0.75,
                "block_scale": 1.25, **p}
        hidden, normed = torch.full_like(block, 7.0), torch.full_like(block, 7.0)
        runtime.block_norm(ctx, block=block, residual=residual, hidden=hidden, normed=normed, **call)
        norm.check(hidden, u, m, (width, name, gate, kind, "hidden"))
        norm.check(normed, n, nm, (width, name, gate, kind, "normed"))
        b, s = block.clone(), residual.clone()
        runtime.block_norm(ctx, block=b, residual=s, hidden=s, normed=b, **call)
        assert torch.equal(s, hidden) and torch.equal(b, normed), (width, name, gate, kind, "in place")
