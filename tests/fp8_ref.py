"""Definitions of the e4m3 layers in 64 bits, on the GPU that the tests have (plain tensor operations of float64, or
float32 where a step is held in 32 bits), with the magnitudes that the tests' tolerances count.

Rounding: s = max(RN32(max |x| / 448), 2^-126) per row and block of 128, r = RN32(1 / s), q = e4m3(RN32(x r)).  Quotients
and products are taken in 64 bits and rounded once to 32: a product of two float32 values is exact in float64, and a
quotient of them is far enough from every tie of float32 for its float64 value to fall on the same side.

Tolerance of a product.  Each output is a sum of I exact products (8 bits times 8 bits), in FP32: in any order, with
any association, at most min(I, 128) additions within a block, one per block and the fold of the waves (8) lie
between a product and the end; the scales s t, their product and the fma add three roundings, and the bias, alpha, beta and
the last addition four more.  With a step of 2^-23 per operation, which covers truncation as well as rounding,
|y - exact| <= 2^-23 (min(I, 128) + blocks + 16) A, where A is the sum of the terms' magnitudes.

Outputs of 16 and 8 bits may come from the 8-bit matrix instructions, which bring the products of eight inputs to the
exponent of the largest of them and drop what lies below 2^-13 of that exponent's power of two.  The power is at most
the largest product's magnitude, so eight products lose at most 8 2^-13 of one of them, and a sum at most 2^-10 A.  (A
random sum loses far less; `typical` is held in the 2-norm over all outputs, 16 times what random blocks have.)
Outputs in 16 bits are half a step (eps / 2 of the value, or half the least subnormal) further off.
"""
import math

import torch

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn


def blocks(n):
    return (n + 127) // 128


def spread(s, rows, width):
    """Scales per block [.., blocks] over `width` columns (and per 128 rows where there are fewer than `rows`)."""
    s = s.repeat_interleave(128, dim=1)[:, :width]
    return s if s.shape[0] == rows else s.repeat_interleave(128, dim=0)[:rows]


def scale_of(most):
    s = (most.double() / 448.0).float().clamp(min=2.0 ** -126)
    return s, (1.0 / s.double()).float()


def round_rows(x):
    """(q e4m3, s [rows, blocks]) of rows of any type."""
    rows, width = x.shape
    x = x.float()
    v = torch.nn.functional.pad(x, (0, blocks(width) * 128 - width)).reshape(rows, -1, 128)
    s, r = scale_of(v.abs().amax(2))
    return (v.double() * r.double()[:, :, None]).float().to(E4M3).reshape(rows, -1)[:, :width].contiguous(), s


def round_weights(w):
    """(q e4m3, t [row blocks, blocks]) of weights of any type."""
    n, width = w.shape
    w = w.float()
    v = torch.nn.functional.pad(w, (0, blocks(width) * 128 - width, 0, blocks(n) * 128 - n))
    v = v.reshape(blocks(n), 128, -1, 128)
    t, r = scale_of(v.abs().amax((1, 3)))
    q = (v.double() * r.double()[:, None, :, None]).float().to(E4M3)
    return q.reshape(blocks(n) * 128, -1)[:n, :width].contiguous(), t


def product(q, s, w, t, bias=None):
    """(sum with the bias, magnitude of its terms), float64."""
    a = q.double() * spread(s.double(), q.shape[0], q.shape[1])
    b = w.double() * spread(t.double(), w.shape[0], w.shape[1])
    z, mag = a @ b.t().contiguous(), a.abs() @ b.abs().t().contiguous()
    return (z, mag) if bias is None else (z + bias.double(), mag + bias.double().abs())


def unit(I, out=torch.float32):
    return 2.0 ** -23 * (min(I, 128) + blocks(I) + 16) + (0.0 if out == torch.float32 else 2.0 ** -10)


TYPICAL = 2e-4


def typical(y, ref, what):
    """16-bit outputs in the 2-norm: the type's rounding (at most eps / 2 of each value) and TYPICAL of the whole."""
    off, all_ = float((y.double() - ref).norm()), float(ref.norm())
    assert off <= (torch.finfo(y.dtype).eps / 2 + TYPICAL) * all_ + torch.finfo(y.dtype).tiny * y.numel(), (what, off / all_)


def half_step(dtype, value):
    """Half a step of `dtype` at float64 values (0 for float32, whose step `unit` counts)."""
    if dtype == torch.float32:
        return torch.zeros_like(value)
    info = torch.finfo(dtype)
    return torch.maximum(value.abs() * (info.eps / 2), torch.full_like(value, info.smallest_normal * info.eps / 2))


def check(y, ref, tol, what):
    got = y.double()
    tol = tol + half_step(y.dtype, ref.abs() + tol)
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got - ref).abs().nan_to_num(math.inf).max()), float(tol.max()))


def weights(I, N, seed, bias=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(N, I, generator=g, device=DEV) * 110).clamp(-448, 448).to(E4M3)
    t = (torch.rand(blocks(N), blocks(I), generator=g, device=DEV) + 0.25) / (110 * math.sqrt(I))
    return w, t, torch.randn(N, generator=g, device=DEV) if bias else None


def rows_of(rows, I, seed, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, I, generator=g, device=DEV) * torch.exp(torch.randn(I, generator=g, device=DEV) * 0.5)
    return x.to(dtype)


def act(g, kind):
    if kind == "silu":
        return g * torch.sigmoid(g)
    return g * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))
