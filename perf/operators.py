"""Operators that stand around the trellis linear layers in a model, on one GPU.

Three operators, each one pass through a public entry point:

* int8: the linear layer in 8-bit integers, for the layers of a model that are
  not trellis-quantized.  Weights are int8 [N][I] with a scale per output
  channel; activations are float rows, rounded to int8 with a scale per token
  inside the call, or int8 rows with their scales.
* norm: everything between two blocks in one pass: the norm of a block's
  output, its gate, the residual sum with its scales, and the norm that feeds
  the next block.
* logprobs: the log probability and rank of a given token per row of logits,
  the row's entropy and its most likely tokens.

`run` computes them in elementary torch operations, or, with `own`, through
this repository's plans.  `exact` restates the definitions in 64 bits.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda:0"
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # One token through a square layer: the smallest product, where the
        # launch and the memory round trips count.
        {"name": "int8_r1", "op": "int8", "I": 4096, "N": 4096, "rows": 1, "input": "f32", "output": "f32",
         "bias": False},
        # Eight sequences decoding through the hidden-size projection of an
        # engine that keeps its activations in bf16.
        {"name": "int8_r8", "op": "int8", "I": 5120, "N": 5120, "rows": 8, "input": "bf16", "output": "bf16",
         "bias": True},
        # Four sequences through the output head, the largest layer of a model.
        {"name": "int8_head_r4", "op": "int8", "I": 5120, "N": 129280, "rows": 4, "input": "f32", "output": "f32",
         "bias": False},
        # A serving batch whose activations arrive in int8 from a static
        # calibration.
        {"name": "int8_m48", "op": "int8", "I": 4096, "N": 12288, "rows": 48, "input": "i8", "output": "f32",
         "bias": False},
        # A short prompt through a layer whose sizes divide by nothing.
        {"name": "int8_m333", "op": "int8", "I": 5119, "N": 2307, "rows": 333, "input": "f16", "output": "f16",
         "bias": True},
        # A prefill chunk through the widest dense layer.
        {"name": "int8_m2048", "op": "int8", "I": 4096, "N": 12288, "rows": 2048, "input": "f32", "output": "f32",
         "bias": False},
        # One token between two blocks, with every part in use.
        {"name": "norm_r1", "op": "norm", "rows": 1, "width": 5120, "type": "f32", "kind": "rms", "post": True,
         "gate": "row", "pre": True, "channel": False},
        # A ragged batch of a layer-norm model with a gate per element.
        {"name": "norm_m333", "op": "norm", "rows": 333, "width": 4099, "type": "f16", "kind": "layer", "post": True,
         "gate": "full", "pre": True, "channel": True},
        # A prefill chunk on the float32 residual stream of the trellis layers.
        {"name": "norm_m4096", "op": "norm", "rows": 4096, "width": 5120, "type": "f32", "kind": "rms", "post": True,
         "gate": "none", "pre": True, "channel": False},
        # One sampled token: its log probability beside the twenty most likely.
        {"name": "logprobs_r1", "op": "logprobs", "rows": 1, "vocab": 129280, "type": "f32", "top": 20,
         "masked": 0.0},
        # A decode batch under a grammar that masks half of an odd vocabulary.
        {"name": "logprobs_r33", "op": "logprobs", "rows": 33, "vocab": 100277, "type": "bf16", "top": 5,
         "masked": 0.5},
        # Scoring the tokens of a prompt.
        {"name": "logprobs_m512", "op": "logprobs", "rows": 512, "vocab": 129280, "type": "f32", "top": 8,
         "masked": 0.0},
    ]


# Dense layers of the benchmark and of the tensor-parallel sites (whole and per rank).
_DENSE = [(4096, 4096), (5120, 5120), (4096, 12288), (1280, 32768), (1280, 16384), (8192, 5120), (4096, 5120),
          (5120, 2304), (5120, 1152), (2304, 5120), (1152, 5120), (5120, 1280), (5120, 512), (2048, 2048)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["int8", "int8", "int8", "norm", "logprobs", "logprobs"])
    types = ["f32", "f32", "f16", "bf16"]
    if op == "int8":
        I, N = rng.choice(_DENSE)
        if rng.random() < 0.4:   # layers off the grid
            I, N = I - rng.randint(1, 255), N - rng.randint(1, 255)
        rows = rng.randint(1, 16) if rng.random() < 0.4 else _log_int(rng, 2, min(4096, 2048 * 4096 * 12288 // (I * N)))
        return {"op": op, "I": I, "N": N, "rows": rows, "input": rng.choice(types + ["i8"]),
                "output": rng.choice(types), "bias": rng.random() < 0.4}
    if op == "norm":
        width = _log_int(rng, 96, 16384)
        rows = _log_int(rng, 1, 4096 * 5120 // width if width > 5120 else 4096)
        post, pre = rng.choice([(True, True), (True, True), (False, True), (True, False)])
        return {"op": op, "rows": rows, "width": width, "type": rng.choice(types),
                "kind": rng.choice(["rms", "rms", "layer"]), "post": post, "gate": rng.choice(["none", "row", "full"]),
                "pre": pre, "channel": rng.random() < 0.3}
    vocab = rng.choice([129280, 100277, 32000, 50257, _log_int(rng, 200, 160000)])
    rows = _log_int(rng, 1, min(4096, 512 * 129280 // vocab))
    return {"op": op, "rows": rows, "vocab": vocab, "type": rng.choice(types), "top": rng.choice([1, 5, 8, 20, 40]),
            "masked": rng.choice([0.0, 0.0, 0.5, 0.98])}


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


def _int8_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    I, N, rows = case["I"], case["N"], case["rows"]
    weights = torch.randint(-127, 128, (N, I), generator=g, device=DEV, dtype=torch.int8)
    # scales that keep the outputs of order one: uniform weights have a deviation of 73
    scales = (0.5 + torch.rand(N, generator=g, device=DEV)) / (73.0 * math.sqrt(I))
    bias = _normal(g, N) if case["bias"] else None
    # normalised hidden states: a spread of channel scales
    x = _normal(g, rows, I) * torch.exp(0.5 * _normal(g, I))
    x_scales = None
    if case["input"] == "i8":
        x_scales = torch.rand(rows, generator=g, device=DEV) * 0.02 + 0.01
        x = (x / x_scales[:, None]).round().clamp(-127, 127).to(torch.int8)
    else:
        x = x.to(_TYPES[case["input"]])
    return weights, scales, bias, x, x_scales


def _norm_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, width, dtype = case["rows"], case["width"], _TYPES[case["type"]]
    # a residual stream that has grown over the layers, and a block's output
    residual = (4.0 * _normal(g, rows, width) * torch.exp(0.3 * _normal(g, width))).to(dtype)
    block = (_normal(g, rows, width) * torch.exp(0.3 * _normal(g, rows, 1)) + 0.1).to(dtype)
    gate = {"none": None, "row": _normal(g, rows, 1), "full": _normal(g, rows, width)}[case["gate"]]
    gate = gate if gate is None else gate.to(dtype)
    weight = lambda: 1.0 + 0.2 * _normal(g, width)  # noqa: E731
    layer = case["kind"] == "layer"
    p = {"post_weight": weight() if case["post"] else None, "pre_weight": weight() if case["pre"] else None,
         "post_bias": 0.1 * _normal(g, width) if case["post"] and layer else None,
         "pre_bias": 0.1 * _normal(g, width) if case["pre"] and layer else None,
         "channel_scale": weight() if case["channel"] else None}
    return block, residual, gate, p


# scales of the residual sum and the norms' epsilon
_RESIDUAL_SCALE, _BLOCK_SCALE, _EPS = 0.75, 1.5, 1e-6


def _logprobs_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    # a broad spread with a confident head of some tokens in each row
    x = 2.5 * _normal(g, rows, vocab)
    at = torch.randint(0, vocab, (rows, 16), generator=g, device=DEV)
    x.scatter_(1, at, 8.0 + 4.0 * _normal(g, rows, 16))
    if case["masked"]:
        x[torch.rand(rows, vocab, generator=g, device=DEV) < case["masked"]] = -math.inf
        x[:, 7] = 1.0   # the grammar allows some token
    # a sampled token: one of the head, or any
    tokens = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.7, at[:, 0],
                         torch.randint(0, vocab, (rows,), generator=g, device=DEV)).to(torch.int32)
    return x.to(_TYPES[case["type"]]), tokens


_SCALE = 1.0 / 0.8   # sampling temperature 0.8

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
    if s.op == "int8":
        s.w, s.w_scales, s.bias, s.x, s.x_scales = _int8_inputs(case, seed)
        s.out = _TYPES[case["output"]]
        if own:
            runtime, ctx = _runtime()
            s.weights = runtime.Int8Weights(ctx, s.w, s.w_scales, bias=s.bias)
            s.w = s.w_scales = s.bias = None   # preparation has laid them out
            s.y = torch.zeros((case["rows"], case["N"]), device=DEV, dtype=s.out)
            s.plan = runtime.Int8LinearPlan(s.weights, s.x, s.y, x_scales=s.x_scales)
    elif s.op == "norm":
        s.block, s.residual, s.gate, s.p = _norm_inputs(case, seed)
        s.layer = case["kind"] == "layer"
        if own:
            runtime, ctx = _runtime()
            s.hidden = torch.zeros_like(s.residual)
            s.normed = torch.zeros_like(s.residual) if case["pre"] else None
            s.plan = runtime.BlockNormPlan(ctx, block=s.block, residual=s.residual, gate=s.gate,
                                           gate_activation="sigmoid", hidden=s.hidden, normed=s.normed,
                                           kind=case["kind"], eps=_EPS, residual_scale=_RESIDUAL_SCALE,
                                           block_scale=_BLOCK_SCALE, **s.p)
    else:
        s.logits, s.tokens = _logprobs_inputs(case, seed)
        s.top = case["top"]
        if own:
            runtime, ctx = _runtime()
            rows = case["rows"]
            f32 = lambda *n: torch.zeros(n, device=DEV)  # noqa: E731
            i32 = lambda *n: torch.zeros(n, device=DEV, dtype=torch.int32)  # noqa: E731
            s.answer = {"logprobs": f32(rows), "ranks": i32(rows), "entropy": f32(rows),
                        "top_ids": i32(rows, s.top), "top_logprobs": f32(rows, s.top)}
            s.plan = runtime.TokenLogprobsPlan(ctx, s.logits, tokens=s.tokens, scale=_SCALE, **s.answer)
    return s


# ---------------------------------------------------------------------------
# The operators
# ---------------------------------------------------------------------------


def run(state):
    s = state
    if own:
        s.plan.submit()
        if s.op == "int8":
            return s.y
        if s.op == "norm":
            return {"hidden": s.hidden} if s.normed is None else {"hidden": s.hidden, "normed": s.normed}
        return s.answer
    return {"int8": _int8, "norm": _norm, "logprobs": _logprobs}[s.op](s)


# The smallest scale of a token: the least normal float32.
_TINY = 2.0 ** -126


def _int8(s):
    """y = (sum_i q[m][i] w[n][i]) x_scale[m] w_scale[n] + bias[n] with q the nearest integers of x / x_scale
    (ties to even) and x_scale the row's largest magnitude over 127, held in 32 bits."""
    if s.x_scales is None:
        x = s.x.float()
        # in 64 bits: the scale's own rounding, and quotients next to a tie
        scale = (x.abs().amax(dim=1).double() / 127.0).float().clamp(min=_TINY)
        q = (x.double() / scale.double()[:, None]).round().float()
    else:
        q, scale = s.x.float(), s.x_scales
    y = (q @ s.w.float().t()) * scale[:, None] * s.w_scales
    return (y if s.bias is None else y + s.bias).to(s.out)


def _normalised(x, weight, bias, layer):
    if layer:
        x = x - x.mean(dim=1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + _EPS) * weight
    return x if bias is None else x + bias


def _norm(s):
    """hidden = residual_scale residual + block_scale channel_scale sigmoid(gate) norm(block), normed = norm(hidden)."""
    t, p = s.block.float(), s.p
    if p["post_weight"] is not None:
        t = _normalised(t, p["post_weight"], p["post_bias"], s.layer)
    if s.gate is not None:
        t = t * torch.sigmoid(s.gate.float())
    if p["channel_scale"] is not None:
        t = t * p["channel_scale"]
    u = _RESIDUAL_SCALE * s.residual.float() + _BLOCK_SCALE * t
    out = {"hidden": u.to(s.block.dtype)}
    if p["pre_weight"] is not None:
        out["normed"] = _normalised(u, p["pre_weight"], p["pre_bias"], s.layer).to(s.block.dtype)
    return out


def _logprobs(s):
    """log softmax of scale * logits at the given token and at the `top` most likely ones (ties to the lowest id),
    the tokens ahead of the given one, and the entropy in nats."""
    x = s.logits.float()
    most = x.amax(dim=1, keepdim=True)
    d = (x - most) * _SCALE
    e = torch.exp(d)
    total = e.sum(dim=1, dtype=torch.float64)   # long sums
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, e * d, 0.0).sum(dim=1, dtype=torch.float64) / total
    at = s.tokens.long()[:, None]
    given = x.gather(1, at)
    ids = torch.arange(x.shape[1], device=x.device)
    ranks = ((x > given) | ((x == given) & (ids < at))).sum(dim=1)
    best, order = torch.sort(x, dim=1, descending=True, stable=True)
    log_p = lambda v: (((v - most) * _SCALE).double() - log_total[:, None]).float()  # noqa: E731
    return {"logprobs": log_p(given)[:, 0], "ranks": ranks.to(torch.int32), "entropy": entropy.float(),
            "top_ids": order[:, :s.top].to(torch.int32), "top_logprobs": log_p(best[:, :s.top])}


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
    if case["op"] == "int8":
        I, N, rows = case["I"], case["N"], case["rows"]
        bytes_ = I * N + 4 * N * (2 if case["bias"] else 1)
        bytes_ += rows * (I * size[case["input"]] + (4 if case["input"] == "i8" else 0) + N * size[case["output"]])
        return {"bytes": bytes_, "flops": 2 * rows * I * N}
    if case["op"] == "norm":
        n, width = case["rows"] * case["width"], case["width"]
        gate = {"none": 0, "row": case["rows"], "full": n}[case["gate"]]
        vectors = case["post"] + case["pre"] + case["channel"]
        vectors += (case["post"] + case["pre"]) if case["kind"] == "layer" else 0
        elements = (3 + case["pre"]) * n + gate
        return {"bytes": elements * size[case["type"]] + 4 * vectors * width, "flops": 12 * n}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * (vocab * size[case["type"]] + 16 + 8 * case["top"]), "flops": 6 * rows * vocab}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    return {"int8": _exact_int8, "norm": _exact_norm, "logprobs": _exact_logprobs}[case["op"]](case, seed)


def _exact_int8(case, seed):
    w, w_scales, bias, x, x_scales = _int8_inputs(case, seed)
    x = x.to(torch.float64)
    if x_scales is None:
        # the scale is held in 32 bits: the quotient rounded to float32
        x_scales = torch.maximum(x.max(dim=1).values, -x.min(dim=1).values).div(127).to(torch.float32)
        x_scales = torch.where(x_scales < _TINY, torch.full_like(x_scales, _TINY), x_scales)
        v = x / x_scales.double().unsqueeze(1)
        low = torch.floor(v)
        up = (v - low > 0.5) | ((v - low == 0.5) & (torch.remainder(low, 2) == 1))
        x = low + up.double()
    y = torch.empty((case["rows"], case["N"]), dtype=torch.float64, device=DEV)
    step = max(1, (1 << 28) // case["I"])
    for n in range(0, case["N"], step):   # columns at a time: the weights in 64 bits are large
        part = slice(n, n + step)
        y[:, part] = torch.matmul(x, w[part].double().t().contiguous())
        y[:, part] *= torch.outer(x_scales.double(), w_scales[part].double())
        if bias is not None:
            y[:, part] += bias[part].double()
    return y


def _exact_norm(case, seed):
    block, residual, gate, p = _norm_inputs(case, seed)
    p = {k: v if v is None else v.double() for k, v in p.items()}

    def norm(v, weight, bias):
        centre = v.mean(1) if case["kind"] == "layer" else v.new_zeros(v.shape[0])
        spread = torch.sqrt(((v - centre[:, None]) ** 2).sum(1) / v.shape[1] + _EPS)
        v = weight[None] * ((v - centre[:, None]) / spread[:, None])
        return v if bias is None else v + bias[None]

    t = block.double()
    if case["post"]:
        t = norm(t, p["post_weight"], p["post_bias"])
    if gate is not None:
        t = t / (1.0 + torch.exp(-gate.double()))
    if case["channel"]:
        t = t * p["channel_scale"][None]
    out = {"hidden": residual.double() * _RESIDUAL_SCALE + t * _BLOCK_SCALE}
    if case["pre"]:
        out["normed"] = norm(out["hidden"], p["pre_weight"], p["pre_bias"])
    return out


def _exact_logprobs(case, seed):
    x, tokens = _logprobs_inputs(case, seed)
    y = {"logprobs": [], "ranks": None, "entropy": [], "top_ids": None, "top_logprobs": []}
    for a in range(0, case["rows"], 64):   # rows at a time: 64 bits of all would be large
        l = _SCALE * x[a:a + 64].double()
        l = l - torch.logsumexp(l, dim=1, keepdim=True)
        p = torch.exp(l)
        y["entropy"].append(-torch.where(p > 0, p * l, torch.zeros_like(p)).sum(1))
        y["logprobs"].append(l[torch.arange(l.shape[0], device=DEV), tokens[a:a + 64].long()])
        y["top_logprobs"].append(torch.topk(l, case["top"], dim=1).values)
    return {k: torch.cat(v) if v else None for k, v in y.items()}
