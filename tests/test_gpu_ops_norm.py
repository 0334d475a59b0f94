"""Norms and residual sum between two blocks (strix_amd_block_norm) against the definition in 64 bits.

Tolerances.  With u = 2^-24: a sum of n non-negative float32 terms in the kernel's order (at most 32 of a thread,
6 levels of a wave, 16 waves) is off by at most 54 u of itself, a mean by as much of the mean magnitude; the
square root halves it; the products and sums after it are under 10 roundings, and expf and the division of a
sigmoid under 6 more.  So 80 u of the magnitudes that enter a value bounds its error: `mag` below carries them
through both norms.  16-bit results add half a step of their type.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from strix_trellis import abi, runtime  # noqa: E402

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOL = 80 * 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = runtime.Context(0)
    yield c
    torch.cuda.synchronize()


def norm64(v, err, w, b, offset, layer, eps):
    """(norm(v), magnitude of its error in units of TOL) of rows v whose own error is TOL * err."""
    mean = v.mean(1, keepdim=True) if layer else torch.zeros(v.shape[0], 1, dtype=torch.float64)
    c = v - mean
    ec = err + (v.abs().mean(1, keepdim=True) + err.mean(1, keepdim=True) if layer else 0.0) + c.abs()
    var = (c * c).mean(1, keepdim=True)
    inv = 1.0 / torch.sqrt(var + eps)
    # a relative error of the variance: its own sum, and 2 c ec / var
    rel = 1.0 + (c.abs() * ec).mean(1, keepdim=True) / (var + eps)
    scale = (offset + w).abs()
    out = c * inv * (offset + w)
    mag = ec * inv * scale + c.abs() * inv * scale * rel + c.abs() * inv * (abs(offset) + w.abs())
    if b is not None:
        out, mag = out + b, mag + b.abs() + out.abs()
    return out, mag


def reference(block, residual, gate, activation, p, layer, eps, offset, rs, bs):
    f = lambda v: None if v is None else v.cpu().double()  # noqa: E731
    block, residual, gate = f(block), f(residual), f(gate)
    p = {k: f(v) for k, v in p.items()}
    u, mag = 0.0, 0.0
    if block is not None:
        t, m = block, torch.zeros_like(block)
        if p.get("post_weight") is not None:
            t, m = norm64(block, m, p["post_weight"], p.get("post_bias"), offset, layer, eps)
        if gate is not None:
            g = torch.sigmoid(gate) if activation == "sigmoid" else gate
            t, m = t * g, m * g.abs() + (t * g).abs()
        if p.get("channel_scale") is not None:
            t, m = t * p["channel_scale"], m * p["channel_scale"].abs() + (t * p["channel_scale"]).abs()
        u, mag = bs * t, abs(bs) * (m + t.abs())
    if residual is not None:
        u, mag = u + rs * residual, mag + abs(rs) * residual.abs()
    mag = mag + u.abs()
    n = nmag = None
    if p.get("pre_weight") is not None:
        n, nmag = norm64(u, mag, p["pre_weight"], p.get("pre_bias"), offset, layer, eps)
    return u, mag, n, nmag


def check(got, ref, mag, what):
    dtype, got = got.dtype, got.cpu().double()
    tol = TOL * mag
    if dtype != torch.float32:
        info = torch.finfo(dtype)
        tol = tol * (1 + info.eps) + (ref.abs() + tol) * (info.eps / 2) + info.smallest_normal * info.eps / 2
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got - ref).abs().max()))


def inputs(rows, width, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *n: torch.randn(*n, generator=g)  # noqa: E731
    residual, block = 3.0 * r(rows, width) + 0.5, r(rows, width) * 2.0 + 1.0
    return block.to(dtype).to(DEV), residual.to(dtype).to(DEV), r


# every kernel instance, widths on and off the vector and workgroup boundaries
WIDTHS = [1, 3, 64, 255, 256, 257, 1000, 1024, 1152, 2047, 2048, 2304, 4099, 5120, 5121, 8192, 8195, 16384, 16385, 32768]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_widths(ctx, width, kind):
    for name, rows in (("f32", 5), ("bf16", 2), ("f16", 1)):
        block, residual, r = inputs(rows, width, TYPES[name], width)
        p = {"post_weight": r(width).to(DEV), "pre_weight": r(width).to(DEV)}
        if kind == "layer":
            p |= {"post_bias": r(width).to(DEV), "pre_bias": r(width).to(DEV)}
        hidden, normed = torch.full_like(block, 7.0), torch.full_like(block, 7.0)
        runtime.block_norm(ctx, block=block, residual=residual, hidden=hidden, normed=normed, kind=kind, eps=1e-5,
                           residual_scale=0.5, block_scale=-1.5, **p)
        u, m, n, nm = reference(block, residual, None, "linear", p, kind == "layer", 1e-5, 0.0, 0.5, -1.5)
        check(hidden, u, m, (name, width, "hidden"))
        check(normed, n, nm, (name, width, "normed"))


PARTS = [
    # block, residual, gate, activation, vectors, outputs
    (True, True, None, "linear", (), "h"),
    (True, False, None, "linear", ("pre_weight",), "n"),
    (False, True, None, "linear", ("pre_weight",), "n"),
    (False, True, None, "linear", ("pre_weight", "pre_bias"), "hn"),
    (True, True, "full", "sigmoid", ("post_weight", "channel_scale"), "h"),
    (True, True, "full", "linear", ("post_weight", "post_bias", "pre_weight"), "hn"),
    (True, True, "rows", "sigmoid", ("pre_weight",), "hn"),
    (True, True, "rows", "linear", ("channel_scale", "pre_weight"), "n"),
    (True, True, "one_row", "linear", ("post_weight", "pre_weight"), "hn"),
    (True, False, "one", "sigmoid", ("post_weight", "pre_weight"), "hn"),
]


@pytest.mark.parametrize("part", range(len(PARTS)))
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_parts(ctx, part, name):
    has_block, has_residual, gate, activation, vectors, outputs = PARTS[part]
    for rows, width, kind in ((7, 515, "rms"), (3, 1280, "layer")):
        block, residual, r = inputs(rows, width, TYPES[name], part)
        block, residual = block if has_block else None, residual if has_residual else None
        shape = {None: None, "full": (rows, width), "rows": (rows, 1), "one_row": (1, width), "one": (1, 1)}[gate]
        g = None if shape is None else r(*shape).to(TYPES[name]).to(DEV)
        p = {v: r(width).to(DEV) for v in vectors}
        like = block if has_block else residual
        hidden = torch.zeros_like(like) if "h" in outputs else None
        normed = torch.zeros_like(like) if "n" in outputs else None
        runtime.block_norm(ctx, block=block, residual=residual, gate=g, gate_activation=activation, hidden=hidden,
                           normed=normed, kind=kind, eps=1e-6, weight_offset=1.0, residual_scale=1.25,
                           block_scale=0.75, **p)
        u, m, n, nm = reference(block, residual, g, activation, p, kind == "layer", 1e-6, 1.0, 1.25, 0.75)
        if hidden is not None:
            check(hidden, u, m, (part, name, "hidden"))
        if normed is not None:
            check(normed, n, nm, (part, name, "normed"))


def test_in_place_and_strided(ctx):
    rows, width = 6, 1003
    block, residual, r = inputs(rows, width, torch.bfloat16, 2)
    w = r(width).to(DEV)
    hidden, normed = torch.empty_like(block), torch.empty_like(block)
    runtime.block_norm(ctx, block=block, residual=residual, hidden=hidden, normed=normed, post_weight=w, pre_weight=w)
    # rows of wider buffers, at odd offsets
    wide = [torch.full((rows + 1, width + 11), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    views = [v[:rows, 5:5 + width] for v in wide]
    views[0].copy_(block)
    views[1].copy_(residual)
    runtime.block_norm(ctx, block=views[0], residual=views[1], hidden=views[1], normed=views[0], post_weight=w,
                       pre_weight=w)
    assert torch.equal(views[1], hidden) and torch.equal(views[0], normed)
    for v in wide:
        assert bool((v[rows] == 3.0).all()) and bool((v[:, :5] == 3.0).all()) and bool((v[:, 5 + width:] == 3.0).all())
    # hidden in the block's place, normed in the residual's
    b, s = block.clone(), residual.clone()
    runtime.block_norm(ctx, block=b, residual=s, hidden=b, normed=s, post_weight=w, pre_weight=w)
    assert torch.equal(b, hidden) and torch.equal(s, normed)


def test_special_rows(ctx):
    """Zero rows, rows of one value, NaN and infinity in one row only."""
    width = 700
    block, residual, r = inputs(5, width, torch.float32, 3)
    w, b = r(width).to(DEV), r(width).to(DEV)
    block[0], residual[0] = 0.0, 0.0
    block[1], residual[1] = 4.0, 0.0
    block[2, 3] = float("nan")
    residual[3, 699] = float("inf")
    for kind in ("rms", "layer"):
        hidden, normed = torch.empty_like(block), torch.empty_like(block)
        runtime.block_norm(ctx, block=block, residual=residual, hidden=hidden, normed=normed, post_weight=w,
                           pre_weight=w, pre_bias=b, kind=kind)
        assert torch.equal(hidden[0], torch.zeros_like(hidden[0])) and torch.equal(normed[0], b)
        if kind == "layer":
            assert torch.equal(normed[1], b)        # a constant row has no spread
        assert bool(torch.isnan(hidden[2]).all()) and bool(torch.isnan(normed[2]).all())
        assert bool(torch.isfinite(hidden[3, :699]).all()) and bool(torch.isfinite(normed[4]).all())
        u, m, n, nm = reference(block[4:], residual[4:], None, "linear", {"post_weight": w, "pre_weight": w, "pre_bias": b},
                                kind == "layer", 1e-6, 0.0, 1.0, 1.0)
        check(normed[4:], n, nm, kind)


def test_plans_streams_and_graphs(ctx):
    stream = torch.cuda.Stream()
    made = []
    for rows, width, name in ((1, 5120, "f32"), (9, 600, "bf16"), (300, 2049, "f16")):
        block, residual, r = inputs(rows, width, TYPES[name], rows)
        w = r(width).to(DEV)
        kw = {"post_weight": w, "pre_weight": w, "residual_scale": 0.5}
        versions = [(block * (k + 1), residual + k) for k in range(3)]
        want = []
        for b, s in versions:
            out = torch.empty_like(b), torch.empty_like(b)
            runtime.block_norm(ctx, block=b, residual=s, hidden=out[0], normed=out[1], **kw)
            want.append(out)
        hidden, normed = torch.empty_like(block), torch.empty_like(block)
        b, s = block.clone(), residual.clone()
        made.append((versions, want, b, s, hidden, normed,
                     runtime.BlockNormPlan(ctx, block=b, residual=s, hidden=hidden, normed=normed, stream=stream, **kw)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for m in made:
            m[-1].submit()
    torch.cuda.synchronize()
    for rep in range(6):
        for versions, want, b, s, hidden, normed, _ in made:
            b.copy_(versions[rep % 3][0])
            s.copy_(versions[rep % 3][1])
            hidden.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for versions, want, b, s, hidden, normed, _ in made:
            assert torch.equal(hidden, want[rep % 3][0]) and torch.equal(normed, want[rep % 3][1])
    for m in made:
        m[-1].destroy()


def test_refusals(ctx):
    block, residual, r = inputs(4, 64, torch.float32, 1)
    w = r(64).to(DEV)

    def status(**kw):
        with pytest.raises(abi.StrixError) as e:
            runtime.block_norm(ctx, **kw)
        return e.value.name

    out = torch.empty_like(block)
    assert status(block=block, residual=residual) == "INVALID_ARGUMENT"                       # no output
    assert status(hidden=out) == "INVALID_ARGUMENT"                                           # no input
    assert status(block=block, hidden=out, normed=torch.empty_like(out)) == "INVALID_ARGUMENT"   # normed without weight
    assert status(block=block, hidden=out, pre_weight=w) == "INVALID_ARGUMENT"
    assert status(block=block, hidden=out, post_bias=w) == "INVALID_ARGUMENT"
    assert status(residual=residual, hidden=out, channel_scale=w) == "INVALID_ARGUMENT"
    assert status(block=block, residual=residual[:3], hidden=out) == "UNSUPPORTED_FORMAT"
    assert status(block=block, residual=residual.half(), hidden=out) == "UNSUPPORTED_FORMAT"
    assert status(block=block, hidden=out, gate=r(2, 64).to(DEV)) == "UNSUPPORTED_FORMAT"
    assert status(block=block, hidden=out, post_weight=w[:63]) == "INSUFFICIENT_BUFFER"
    assert status(block=block, hidden=out, eps=0.0) == "INVALID_ARGUMENT"
    assert status(block=block, hidden=out, residual_scale=float("nan")) == "INVALID_ARGUMENT"
    assert status(block=block, hidden=out, normed=out, pre_weight=w) == "INVALID_ARGUMENT"
    assert status(block=block, hidden=out, gate=out) == "INVALID_ARGUMENT"
    wide = torch.zeros(5, 64, device=DEV)
    assert status(block=wide[:4], hidden=wide[1:]) == "INVALID_ARGUMENT"                      # overlap, not the same
    big = torch.zeros(1, 32769, device=DEV)
    assert status(block=big, hidden=torch.empty_like(big)) == "UNSUPPORTED_FORMAT"
    runtime.block_norm(ctx, block=block[:0], hidden=out[:0])                                  # no rows
    torch.cuda.synchronize()
