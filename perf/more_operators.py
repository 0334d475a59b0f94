"""Operators of checkpoints in 8-bit floating point and of decoding with several beams, on one GPU.

Four operators, each one pass through a public entry point:

* fp8: the linear layer in e4m3 with a scale for each 128 x 128 block of the weights.  Activations are float rows,
  rounded in the call with a scale per token and block of 128 inputs, or e4m3 rows with their scales.
* gated: the first half of a dense feed-forward block on such weights: both projections, the activation and the
  product; the hidden rows leave as floats, or in e4m3 with a scale per token and 128 channels, as the second half
  takes them.
* select: the best continuations of each batch entry's beams, from the logits and the beams' scores.
* reorder: the beams' states (a cache) take the contents of the beams that they continue.

`run` computes them in elementary torch operations, or, with `own`, through this repository's plans.  `exact`
restates the definitions in 64 bits.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda:0"
_E4M3 = torch.float8_e4m3fn
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": _E4M3}

# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # One token through a square layer: the smallest product, where the launch and the round trips count.
        {"name": "fp8_r1", "op": "fp8", "I": 4096, "N": 4096, "rows": 1, "input": "f32", "output": "f32",
         "bias": False},
        # Four sequences through the output head, the largest layer of a model.
        {"name": "fp8_head_r4", "op": "fp8", "I": 5120, "N": 129280, "rows": 4, "input": "bf16", "output": "f32",
         "bias": False},
        # A serving batch whose rows arrive in e4m3, from the feed-forward block's first half.
        {"name": "fp8_m48", "op": "fp8", "I": 12288, "N": 4096, "rows": 48, "input": "e4m3", "output": "bf16",
         "bias": False},
        # A short prompt through a layer whose sizes divide by nothing.
        {"name": "fp8_m333", "op": "fp8", "I": 5119, "N": 2307, "rows": 333, "input": "f16", "output": "f16",
         "bias": True},
        # A prefill chunk through the widest dense layer.
        {"name": "fp8_m2048", "op": "fp8", "I": 4096, "N": 12288, "rows": 2048, "input": "bf16", "output": "bf16",
         "bias": False},
        # One token through the feed-forward block's first half.
        {"name": "gated_r1", "op": "gated", "I": 5120, "N": 2304, "rows": 1, "input": "f32", "output": "f32",
         "bias": False, "activation": "silu"},
        # A ragged batch with biases through sizes that divide by nothing.
        {"name": "gated_m150", "op": "gated", "I": 4091, "N": 5125, "rows": 150, "input": "f16", "output": "f16",
         "bias": True, "activation": "gelu"},
        # A prefill chunk whose hidden rows stay in 8 bits for the second half.
        {"name": "gated_m2048", "op": "gated", "I": 4096, "N": 12288, "rows": 2048, "input": "bf16",
         "output": "e4m3", "bias": False, "activation": "silu"},
        # One prompt with four beams.
        {"name": "select_b1", "op": "select", "batch": 1, "beams": 4, "vocab": 129280, "type": "f32", "keep": 8,
         "done": 0.0},
        # A batch of prompts with eight beams each, some of them finished.
        {"name": "select_b64", "op": "select", "batch": 64, "beams": 8, "vocab": 129280, "type": "bf16", "keep": 16,
         "done": 0.1},
        # The cache of one layer for one prompt of an odd length, into a second buffer.
        {"name": "reorder_b1", "op": "reorder", "outer": 1, "batch": 1, "beams": 4, "inner": 8, "tokens": 301,
         "dim": 128, "moved": 2, "in_place": False},
        # The cache of four layers for sixteen prompts, in place: half of the beams move.
        {"name": "reorder_b16", "op": "reorder", "outer": 4, "batch": 16, "beams": 4, "inner": 8, "tokens": 1000,
         "dim": 128, "moved": 2, "in_place": True},
    ]


# Dense layers of the benchmark and of the tensor-parallel sites (whole and per rank).
_DENSE = [(4096, 4096), (5120, 5120), (4096, 12288), (1280, 32768), (1280, 16384), (8192, 5120), (4096, 5120),
          (5120, 2304), (5120, 1152), (2304, 5120), (1152, 5120), (5120, 1280), (5120, 512), (2048, 2048),
          (12288, 4096)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["fp8", "fp8", "gated", "gated", "select", "reorder"])
    types = ["f32", "f16", "bf16", "bf16"]
    if op in ("fp8", "gated"):
        I, N = rng.choice(_DENSE)
        if rng.random() < 0.4:   # layers off the grid
            I, N = I - rng.randint(1, 255), N - rng.randint(1, 255)
        rows = rng.randint(1, 16) if rng.random() < 0.4 else _log_int(rng, 2, min(4096, 2048 * 4096 * 12288 // (I * N)))
        case = {"op": op, "I": I, "N": N, "rows": rows, "input": rng.choice(types + ["e4m3"]),
                "output": rng.choice(types), "bias": rng.random() < 0.4}
        if op == "gated":
            case["activation"] = rng.choice(["silu", "silu", "gelu"])
            case["output"] = rng.choice(types + ["e4m3", "e4m3"])
        return case
    if op == "select":
        vocab = rng.choice([129280, 100277, 32000, 50257, _log_int(rng, 200, 160000)])
        beams = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 16])
        batch = _log_int(rng, 1, max(1, min(256, 512 * 129280 // (vocab * beams))))
        return {"op": op, "batch": batch, "beams": beams, "vocab": vocab, "type": rng.choice(types),
                "keep": beams * rng.choice([1, 2, 2]), "done": rng.choice([0.0, 0.1, 0.4])}
    beams = rng.choice([2, 3, 4, 4, 5, 8, 8, 16])
    outer, inner, dim = rng.choice([1, 2, 4]), rng.choice([1, 2, 8]), rng.choice([64, 80, 128])
    most = 4 * 32 * 8 * 1000 * 128 // (outer * beams * inner * dim)   # tokens of all prompts
    batch = _log_int(rng, 1, 32)
    return {"op": op, "outer": outer, "batch": batch, "beams": beams, "inner": inner,
            "tokens": _log_int(rng, 1, max(2, min(16384, most // batch))), "dim": dim,
            "moved": rng.randint(1, beams), "in_place": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


class _State:
    """Buffers of one case, with the library's plan and weights under `own`."""

    def __init__(self):
        self.plan, self.weights = None, None

    def __del__(self):
        try:
            if self.plan is not None:
                torch.cuda.synchronize()
                self.plan.destroy()
            if self.weights is not None:
                self.weights.destroy()
        except Exception:
            pass


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _blocks(n):
    return (n + 127) // 128


def _fp8_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    I, N, rows = case["I"], case["N"], case["rows"]
    layers = []
    for _ in range(2 if case["op"] == "gated" else 1):
        # normal weights whose largest of a block stands near the type's largest, 448
        w = (110.0 * _normal(g, N, I)).clamp(-448.0, 448.0).to(_E4M3)
        # scales that keep the outputs of order one
        scales = (0.5 + torch.rand(_blocks(N), _blocks(I), generator=g, device=DEV)) / (110.0 * math.sqrt(I))
        layers.append((w, scales, _normal(g, N) if case["bias"] else None))
    # normalised hidden states: a spread of channel scales
    x = _normal(g, rows, I) * torch.exp(0.5 * _normal(g, I))
    x_scales = None
    if case["input"] == "e4m3":
        x_scales = torch.rand(rows, _blocks(I), generator=g, device=DEV) * 0.01 + 0.005
        x = x / x_scales.repeat_interleave(128, dim=1)[:, :I]
        x = x.clamp(-448.0, 448.0)
    return layers, x.to(_TYPES[case["input"]]), x_scales


def _select_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
    rows = batch * beams
    # a broad spread with a confident head of some tokens in each row
    x = 2.5 * _normal(g, rows, vocab)
    at = torch.randint(0, vocab, (rows, 1), generator=g, device=DEV) + torch.arange(16, device=DEV) * (vocab // 16)
    x.scatter_(1, at % vocab, 8.0 + 4.0 * _normal(g, rows, 16))
    # beams in the order of their scores
    scores = -torch.cumsum(torch.rand(batch, beams, generator=g, device=DEV), 1) * 2.0 - 3.0
    finished = (torch.rand(rows, generator=g, device=DEV) < case["done"]).to(torch.int32)
    return x.to(_TYPES[case["type"]]), scores.reshape(rows).contiguous(), finished


def _reorder_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    batch, beams, moved = case["batch"], case["beams"], case["moved"]
    width = case["tokens"] * case["dim"]
    # room for longer sequences behind the tokens that are there
    room = (case["tokens"] + 63) // 64 * 64 * case["dim"]
    cache = torch.randint(-2 ** 15, 2 ** 15, (case["outer"], batch * beams, case["inner"], room), generator=g, device=DEV,
                          dtype=torch.int16)
    # `moved` beams of each prompt continue another one; the others continue themselves
    order = torch.rand(batch, beams, generator=g, device=DEV).argsort(1)
    places = torch.arange(beams, device=DEV).expand(batch, beams)
    away = torch.randint(1, beams, (batch, beams), generator=g, device=DEV)
    parents = torch.where(order < moved, (places + away) % beams, places)
    return cache[..., :width], parents.to(torch.int32).contiguous()


_SCALE = 1.0 / 0.8   # sampling temperature 0.8
_PAD = 3             # what a finished beam continues with

_CONTEXT = []


def _runtime():
    at = str(Path(__file__).resolve().parent.parent / "strix-trellis_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from strix_trellis import runtime
    if not _CONTEXT:
        _CONTEXT.append(runtime.Context(0))
    return runtime, _CONTEXT[0]


def prepare(case, seed):
    s = _State()
    s.op = case["op"]
    if s.op in ("fp8", "gated"):
        s.layers, s.x, s.x_scales = _fp8_inputs(case, seed)
        s.out, s.activation = _TYPES[case["output"]], case.get("activation")
        if own:
            runtime, ctx = _runtime()
            rows, N = case["rows"], case["N"]
            s.y = torch.zeros((rows, N), device=DEV, dtype=s.out)
            w, scales, bias = s.layers[0]
            if s.op == "fp8":
                s.weights = runtime.Fp8Weights(ctx, w, scales, bias=bias)
                s.plan = runtime.Fp8LinearPlan(s.weights, s.x, s.y, x_scales=s.x_scales)
            else:
                up, up_scales, up_bias = s.layers[1]
                s.weights = runtime.Fp8Weights(ctx, w, scales, bias=bias, up=up, up_scales=up_scales, up_bias=up_bias)
                s.y_scales = torch.zeros((rows, _blocks(N)), device=DEV) if s.out == _E4M3 else None
                s.plan = runtime.Fp8GatedPlan(s.weights, s.x, s.y, x_scales=s.x_scales, y_scales=s.y_scales,
                                              activation=s.activation)
            s.layers = None   # preparation has laid them out
    elif s.op == "select":
        s.logits, s.scores, s.finished = _select_inputs(case, seed)
        s.beams, s.keep = case["beams"], case["keep"]
        if own:
            runtime, ctx = _runtime()
            n = (case["batch"], s.keep)
            s.answer = {"scores": torch.zeros(n, device=DEV),
                        "parents": torch.zeros(n, device=DEV, dtype=torch.int32),
                        "tokens": torch.zeros(n, device=DEV, dtype=torch.int32)}
            s.plan = runtime.BeamSelectPlan(ctx, s.logits, s.scores, s.answer["scores"], s.answer["parents"],
                                            s.answer["tokens"], beams=s.beams, finished=s.finished, pad=_PAD,
                                            scale=_SCALE)
    else:
        s.cache, s.parents = _reorder_inputs(case, seed)
        s.in_place = case["in_place"]
        if own:
            runtime, ctx = _runtime()
            s.target = s.cache if s.in_place else torch.zeros_like(s.cache)
            s.plan = runtime.BeamReorderPlan(ctx, s.parents, s.cache, s.target)
    return s


# ---------------------------------------------------------------------------
# The operators
# ---------------------------------------------------------------------------


def run(state):
    s = state
    if own:
        s.plan.submit()
        if s.op == "fp8":
            return s.y
        if s.op == "gated":
            return {"hidden": s.y} if s.y_scales is None else {"hidden": s.y, "scales": s.y_scales}
        return s.answer if s.op == "select" else s.target
    return {"fp8": _fp8, "gated": _gated, "select": _select, "reorder": _reorder}[s.op](s)


# The smallest scale: the least normal float32.
_TINY = 2.0 ** -126


def _rounded(x):
    """e4m3 values of float32 rows and their scales: per row and block of 128, s = max / 448 in 32 bits, and
    x * (1 / s), in 32 bits, to the nearest e4m3 (ties to even)."""
    rows, width = x.shape
    pad = _blocks(width) * 128 - width
    v = torch.nn.functional.pad(x, (0, pad)).reshape(rows, -1, 128)
    # quotients in 64 bits, as each is rounded once
    s = (v.abs().amax(dim=2).double() / 448.0).float().clamp(min=_TINY)
    q = (v * (1.0 / s.double()).float()[:, :, None]).to(_E4M3)
    return q.reshape(rows, -1)[:, :width], s


def _product(x, x_scales, w, scales, bias):
    """sum over blocks of x_scale * scale * (the block's sum of products), plus the bias, in 32 bits."""
    N, I = w.shape
    a = x.float() * x_scales.repeat_interleave(128, dim=1)[:, :I]
    b = w.float() * scales.repeat_interleave(128, dim=0)[:N].repeat_interleave(128, dim=1)[:, :I]
    y = a @ b.t()
    return y if bias is None else y + bias


def _rows(s):
    return (s.x, s.x_scales) if s.x_scales is not None else _rounded(s.x.float())


def _fp8(s):
    return _product(*_rows(s), *s.layers[0]).to(s.out)


def _gated(s):
    """act(gate) * up, with silu(g) = g sigmoid(g) or gelu(g) = g / 2 (1 + tanh(sqrt(2 / pi) (g + 0.044715 g^3)))."""
    x, x_scales = _rows(s)
    g, u = _product(x, x_scales, *s.layers[0]), _product(x, x_scales, *s.layers[1])
    if s.activation == "silu":
        h = g * torch.sigmoid(g) * u
    else:
        h = 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g))) * u
    if s.out != _E4M3:
        return {"hidden": h.to(s.out)}
    q, scales = _rounded(h)
    return {"hidden": q, "scales": scales}


def _select(s):
    """The `keep` largest of score + log softmax(scale * logits) over a prompt's beams and tokens, ties to the lower
    beam, then token.  A finished beam has one continuation, the pad token at its own score."""
    rows, vocab = s.logits.shape
    # in 64 bits: long sums, and candidates of different beams next to each other
    x = s.logits.double() * _SCALE
    x = x - x.amax(dim=1, keepdim=True)
    c = s.scores.double()[:, None] + (x - torch.log(torch.exp(x).sum(dim=1, keepdim=True)))
    at_pad = torch.arange(vocab, device=c.device) == _PAD
    only = torch.where(at_pad, s.scores.double()[:, None], -math.inf)
    c = torch.where((s.finished != 0)[:, None], only, c).reshape(rows // s.beams, -1)
    best, order = torch.sort(c, dim=1, descending=True, stable=True)
    best, order = best[:, :s.keep], order[:, :s.keep]
    live = best > -math.inf
    return {"scores": best.float(), "parents": torch.where(live, order // vocab, -1).to(torch.int32),
            "tokens": torch.where(live, order % vocab, -1).to(torch.int32)}


def _reorder(s):
    """Row b of prompt p becomes row parents[p][b] of that prompt."""
    batch, beams = s.parents.shape
    rows = (s.parents + beams * torch.arange(batch, device=s.parents.device, dtype=torch.int32)[:, None]).reshape(-1)
    moved = s.cache[:, rows]
    return s.cache.copy_(moved) if s.in_place else moved


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
    if case["op"] in ("fp8", "gated"):
        I, N, rows, layers = case["I"], case["N"], case["rows"], 2 if case["op"] == "gated" else 1
        bytes_ = layers * (I * N + 4 * _blocks(I) * _blocks(N) + (4 * N if case["bias"] else 0))
        bytes_ += rows * I * size[case["input"]] + (4 * rows * _blocks(I) if case["input"] == "e4m3" else 0)
        bytes_ += rows * N * size[case["output"]] + (4 * rows * _blocks(N) if case["output"] == "e4m3" else 0)
        return {"bytes": bytes_, "flops": 2 * layers * rows * I * N}
    if case["op"] == "select":
        rows, vocab = case["batch"] * case["beams"], case["vocab"]
        live = rows * (1.0 - case["done"])   # a finished beam's logits are not looked at
        return {"bytes": live * vocab * size[case["type"]] + 8 * rows + 12 * case["batch"] * case["keep"],
                "flops": 4 * live * vocab}
    # rows that others take, each read once, and the rows written: in place those that move
    row, beams = case["outer"] * case["inner"] * case["tokens"] * case["dim"] * 2, case["beams"]
    moved = case["moved"]
    taken = beams * (1.0 - (1.0 - 1.0 / beams) ** moved)
    rows = taken + moved if case["in_place"] else min(beams, taken + beams - moved) + beams
    return {"bytes": case["batch"] * rows * row + 4 * case["batch"] * beams, "flops": 0}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "reorder":
        return None   # nothing is computed
    if case["op"] == "select":
        return _exact_select(case, seed)
    layers, x, x_scales = _fp8_inputs(case, seed)
    q, s = (x, x_scales) if x_scales is not None else _exact_rounding(x)
    y = [_exact_product(q.to(torch.float64), s.double(), *layer) for layer in layers]
    if case["op"] == "fp8":
        return y[0]
    g, u = y
    if case["activation"] == "silu":
        h = g / (1.0 + torch.exp(-g)) * u
    else:   # (1 + tanh z) / 2 = 1 / (1 + e^-2z)
        h = g / (1.0 + torch.exp(-2.0 * (2.0 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3))) * u
    if case["output"] != "e4m3":
        return {"hidden": h}
    # before their rounding to 8 bits
    width = h.shape[1]
    most = torch.stack([part.abs().max(dim=1).values for part in h.split(128, dim=1)], dim=1)
    scales = most / 448.0
    return {"hidden": h / scales.repeat_interleave(128, dim=1)[:, :width], "scales": scales}


def _exact_rounding(x):
    """Each block's scale and its inverse are held in 32 bits, and so is the product that is rounded to e4m3: four
    significant bits, steps of 2^-9 at least."""
    x = x.double()
    q, scales = torch.empty_like(x), []
    for b in range(_blocks(x.shape[1])):
        part = x[:, 128 * b:128 * (b + 1)]
        s = torch.maximum(part.max(dim=1).values, -part.min(dim=1).values).div(448).to(torch.float32)
        s = torch.where(s < _TINY, torch.full_like(s, _TINY), s)
        inverse = s.double().reciprocal().to(torch.float32).double()
        v = (part * inverse.unsqueeze(1)).to(torch.float32).double()
        exponent = torch.frexp(v).exponent - 1
        step = torch.ldexp(torch.ones_like(v), exponent.clamp(min=-6) - 3)
        q[:, 128 * b:128 * (b + 1)] = torch.round(v / step) * step
        scales.append(s)
    return q, torch.stack(scales, dim=1)


def _exact_product(q, s, w, scales, bias):
    (rows, I), N = q.shape, w.shape[0]
    q = torch.cat([q[:, 128 * b:128 * (b + 1)] * s[:, b:b + 1] for b in range(_blocks(I))], dim=1)
    y = torch.empty((rows, N), dtype=torch.float64, device=DEV)
    step = max(1, (1 << 28) // I // 128) * 128
    for n in range(0, N, step):   # channels at a time: the weights in 64 bits are large
        part = w[n:n + step].double()
        t = scales[n // 128:_blocks(n + part.shape[0])].double()
        part *= torch.kron(t, torch.ones(128, 128, dtype=torch.float64, device=DEV))[:part.shape[0], :I]
        y[:, n:n + step] = torch.matmul(q, part.t().contiguous())
    return y if bias is None else y.add_(bias.double())


def _exact_select(case, seed):
    x, scores, finished = _select_inputs(case, seed)
    best = []
    for p in range(case["batch"]):   # a prompt at a time: 64 bits of all would be large
        part = slice(p * case["beams"], (p + 1) * case["beams"])
        l = x[part].double() * _SCALE
        c = l - torch.logsumexp(l, dim=1, keepdim=True) + scores[part].double().unsqueeze(1)
        over = finished[part].bool()
        c[over] = -math.inf
        c[over, _PAD] = scores[part][over].double()
        best.append(torch.topk(c.flatten(), case["keep"]).values)
    return {"scores": torch.stack(best), "parents": None, "tokens": None}
