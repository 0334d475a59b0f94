"""The operators around the trellis layers together, as an engine runs them: a decode batch goes through norms, a
trellis layer, int8 layers, the residual sum and the head to log probabilities, in one captured graph; rows beyond
32-bit offsets; buffers without torch.

Each step of the chain is held to its own definition in 64 bits on the values that the step before left, with the
tolerances of the operators' own tests.
"""
import numpy as np
import pytest

import synth

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_ops_int8 as int8  # noqa: E402
import test_gpu_ops_logprobs as logprobs  # noqa: E402
import test_gpu_ops_norm as norm  # noqa: E402
from oracle import linear  # noqa: E402
from strix_trellis import device, runtime  # noqa: E402

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows", [1, 6, 40])
def test_block_and_head(ctx, rows):
    """x -> norm -> trellis layer -> norm, gate, residual, norm -> int8 layer -> residual, norm -> int8 head -> tokens."""
    D, H, V, K = 512, 640, 5003, 4
    g = torch.Generator().manual_seed(rows)
    r = lambda *n: torch.randn(*n, generator=g).to(DEV)  # noqa: E731
    tr, suh, svh, b = synth.layer(D, D, K, 17, bias=True)
    trellis = runtime.Weights(ctx, tr, suh, svh, b, "mul1")
    w1, t1, b1 = int8.layer(D, H, 1)
    w2, t2, b2 = int8.layer(H, D, 2)
    wh, th, bh = int8.layer(D, V, 3, bias=False)
    up, down, head = (runtime.Int8Weights(ctx, w, t, bias=bias) for w, t, bias in ((w1, t1, b1), (w2, t2, b2), (wh, th, bh)))
    p = {k: 1.0 + 0.1 * r(D) for k in ("n1", "post1", "pre2", "post2", "final")}
    x, gate = torch.zeros(rows, D, device=DEV), r(rows, 1)
    z = lambda *n, dt=torch.float32: torch.zeros(n, device=DEV, dtype=dt)  # noqa: E731
    a, o, h1, a2, u, d, h2, f, logits = (z(rows, D), z(rows, D), z(rows, D), z(rows, D), z(rows, H), z(rows, D), z(rows, D),
                                         z(rows, D), z(rows, V))
    out = logprobs.outputs(rows, 5)
    tokens = torch.randint(0, V, (rows,), generator=g, dtype=torch.int32).to(DEV)
    stream = torch.cuda.Stream()
    steps = [
        runtime.BlockNormPlan(ctx, residual=x, normed=a, pre_weight=p["n1"], stream=stream),
        runtime.LinearPlan(trellis, a, o, operation="gemv" if rows <= 8 else "gemm", stream=stream),
        runtime.BlockNormPlan(ctx, block=o, residual=x, gate=gate, gate_activation="sigmoid", hidden=h1, normed=a2,
                              post_weight=p["post1"], pre_weight=p["pre2"], block_scale=0.7, stream=stream),
        runtime.Int8LinearPlan(up, a2, u, stream=stream),
        runtime.Int8LinearPlan(down, u, d, stream=stream),
        runtime.BlockNormPlan(ctx, block=d, residual=h1, hidden=h2, normed=f, post_weight=p["post2"],
                              pre_weight=p["final"], stream=stream),
        runtime.Int8LinearPlan(head, f, logits, stream=stream),
        runtime.TokenLogprobsPlan(ctx, logits, tokens=tokens, scale=0.9, stream=stream, **out),
    ]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for s in steps:
            s.submit()
    for rep in range(3):
        x.copy_(3.0 * r(rows, D))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _, _, n, m = norm.reference(None, x, None, "linear", {"pre_weight": p["n1"]}, False, 1e-6, 0.0, 1.0, 1.0)
        norm.check(a, n, m, "first norm")
        synth.gate(o.cpu().numpy(), linear.matmul_fp32(a.cpu().numpy(), tr, suh, svh, K, "mul1", b))
        hu, hm, n, m = norm.reference(o, x, gate, "sigmoid", {"post_weight": p["post1"], "pre_weight": p["pre2"]}, False,
                                      1e-6, 0.0, 1.0, 0.7)
        norm.check(h1, hu, hm, "residual sum")
        norm.check(a2, n, m, "second norm")
        int8.check(u, *int8.reference(a2, None, w1, t1, b1, 1.0, 0.0, None), "up")
        int8.check(d, *int8.reference(u, None, w2, t2, b2, 1.0, 0.0, None), "down")
        hu, hm, n, m = norm.reference(d, h1, None, "linear", {"post_weight": p["post2"], "pre_weight": p["final"]}, False,
                                      1e-6, 0.0, 1.0, 1.0)
        norm.check(h2, hu, hm, "residual sum 2")
        norm.check(f, n, m, "final norm")
        int8.check(logits, *int8.reference(f, None, wh, th, bh, 1.0, 0.0, None), "head")
        logprobs.check(logits, tokens, out, 0.9, "tokens")
    for s in steps:
        s.destroy()
    for w in (trellis, up, down, head):
        w.destroy()


def test_rows_beyond_32_bit_offsets(ctx):
    """Three rows, 2^31 elements apart: the second and third start beyond 2 and 4 GiB of elements."""
    W, far = 1003, 2 ** 31
    base = torch.empty(2 * far + W, dtype=torch.float16, device=DEV)
    x = base.as_strided((3, W), (far, 1))
    x.copy_(torch.randn(3, W, device=DEV).half())
    base_y = torch.empty(2 * far + W, dtype=torch.float16, device=DEV)
    y = base_y.as_strided((3, W), (far, 1))
    tokens = torch.tensor([1, 2, W - 1], dtype=torch.int32, device=DEV)
    out = logprobs.outputs(3, 3)
    runtime.token_logprobs(ctx, x, tokens=tokens, **out)
    logprobs.check(x, tokens, out, 1.0, "far")
    runtime.block_norm(ctx, block=x, residual=x, hidden=y)
    u, m, _, _ = norm.reference(x, x, None, "linear", {}, False, 1e-6, 0.0, 1.0, 1.0)
    norm.check(y, u, m, "far")
    for rows in (3, 20):
        w, t, bias = int8.layer(W, W, 6)
        weights = runtime.Int8Weights(ctx, w, t, bias=bias)
        step = far if rows == 3 else 2 * far // 19
        xr, yr = base.as_strided((rows, W), (step, 1)), base_y.as_strided((rows, W), (step, 1))
        xr.copy_(torch.randn(rows, W, device=DEV).half())
        runtime.int8_linear(weights, xr, yr)
        int8.check(yr, *int8.reference(xr, None, w, t, bias, 1.0, 0.0, None), ("far", rows))
        weights.destroy()


def test_device_arrays_without_torch_tensors(ctx):
    rng = np.random.default_rng(5)
    rows, I, N = 3, 200, 90
    w = rng.integers(-127, 128, (N, I), dtype=np.int8)
    t = rng.random(N, dtype=np.float32) + 0.1
    x = rng.standard_normal((rows, I), dtype=np.float32)
    stream = device.Stream(0)
    A = device.DeviceArray
    weights = runtime.Int8Weights(ctx, A.from_numpy(w), A.from_numpy(t), stream=stream)
    y, e = A.empty((rows, N)), A.empty((rows,))
    runtime.int8_linear(weights, A.from_numpy(x), y, stream=stream)
    runtime.token_logprobs(ctx, y, entropy=e, stream=stream)
    stream.synchronize()
    ref, mag = int8.reference(torch.from_numpy(x), None, torch.from_numpy(w), torch.from_numpy(t), None, 1.0, 0.0, None)
    int8.check(torch.from_numpy(y.numpy()), ref, mag, "device arrays")
    l = torch.log_softmax(torch.from_numpy(y.numpy()).double(), 1)
    assert np.allclose(e.numpy(), -(l.exp() * l).sum(1).numpy(), rtol=1e-5, atol=1e-5)
    weights.destroy()
