"""Shared by the tests of the products with epilogues and the grouped products: the operators in
64 bits from their formulas, and how far a 32-bit kernel may be off them.

Tolerances, from the arithmetic (u = 2^-24, the half step of f32):
* a sum of K products held in f32, in any order and with each addition rounded or truncated, is
  off by at most (K + 8) * 2u * sum |a||b|;
* bias and residual additions: 2u each, relative to the largest magnitude that takes part;
* an activation is off by its argument's error times its largest slope (1.13 for gelu) plus its own
  evaluation error: e^-s carries |s| * 2u from its scaled argument, the exponential, division
  and erf a few u each - EVAL(x) = 2^-20 * (1 + |s|) covers them, relative to |x| for the
  value and to 1 + |x| for the slope (s the sigmoid's argument, x itself for erf);
* the one rounding to the output type: half a step, eps / 2 relative, plus half the smallest
  subnormal of f16 (2^-25).
"""
import math

import torch

U = 2.0 ** -24
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
PAIRS = [("f16", "f16"), ("f32", "f16"), ("bf16", "bf16"), ("f32", "bf16")]
ACTS = ["none", "relu", "silu", "gelu_tanh", "gelu"]
G = math.sqrt(2 / math.pi)


def value(x, act):
    if act == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(G * (x + 0.044715 * x ** 3)))
    if act == "gelu":
        return 0.5 * x * torch.special.erfc(-x * math.sqrt(0.5))
    return x


def slope(x, act):
    if act == "relu":
        return (x > 0).to(x.dtype)
    if act == "silu":
        s = torch.sigmoid(x)
        return s * (1 + x * (1 - s))
    if act == "gelu_tanh":
        t = torch.tanh(G * (x + 0.044715 * x ** 3))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * G * (1 + 3 * 0.044715 * x * x)
    if act == "gelu":
        return 0.5 * torch.special.erfc(-x * math.sqrt(0.5)) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    return torch.ones_like(x)


def eval_error(x, act):
    """Relative evaluation error of an activation or slope at x."""
    if act in ("none", "relu"):
        return torch.zeros_like(x)
    s = x if act != "gelu_tanh" else 2 * G * (x + 0.044715 * x ** 3)
    return 2.0 ** -20 * (1 + s.abs().clamp(max=100))


def rounding(y, dtype):
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return torch.finfo(dtype).eps / 2 * y.abs() + sub


def product(a, b):
    """(a b, bound of the f32 error) in 64 bits; a [..., M, K], b [..., K, N]."""
    a, b = a.double(), b.double()
    return a @ b, (a.shape[-1] + 8) * 2 * U * (a.abs() @ b.abs())


def forward(a, b, act, bias=None, residual=None):
    """(C, tolerance of C before rounding, Z, tolerance of Z) of the forward epilogue; bias broadcasts."""
    z, ez = product(a, b)
    if bias is not None:
        ez = ez + 2 * U * (z.abs() + bias.double().abs())
        z = z + bias.double()
    y = value(z, act)
    ey = 1.13 * ez + z.abs() * eval_error(z, act)
    if residual is not None:
        ey = ey + 2 * U * (y.abs() + residual.double().abs())
        y = y + residual.double()
    return y, ey, z, ez


def gradient(x, ex, z, act):
    """(x act'(z), tolerance before rounding)"""
    if act == "none":
        return x, ex
    z = z.double()
    s = slope(z, act)
    return x * s, ex * s.abs() + x.abs() * (1 + z.abs()) * eval_error(z, act) + 2 * U * (x * s).abs()


def check(got, want, tol, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got.double()).all(), f"{what}: unwritten, NaN or infinite elements"
    over = (got.double() - want).abs() - tol - rounding(want, got.dtype)
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{what}: off by {worst:.3g} more than the arithmetic allows ({int((over > 0).sum())} of {over.numel()} elements)"


def check_sum(got, d, ed, dim, what=""):
    """A bias gradient: f32 sums of d over `dim`, each element of d off by ed."""
    n = 1
    for i in (dim if isinstance(dim, tuple) else (dim,)):
        n *= d.shape[i]
    want = d.sum(dim) if n else torch.zeros_like(got, dtype=torch.float64)
    tol = ed.sum(dim) + (n + 8) * 2 * U * (d.abs() + ed).sum(dim) if n else torch.zeros_like(want)
    check(got, want, tol, what)


class Guarded:
    """A buffer of n elements with poisoned guard elements either side; itself poisoned."""

    def __init__(self, shape, dtype, pad=64, offset=0):
        n = math.prod(shape)
        self.pad = pad + offset
        self.raw = torch.full((n + 2 * pad + offset,), float("nan"), dtype=dtype, device="cuda")
        self.t = self.raw[self.pad:self.pad + n].view(shape)

    def intact(self):
        n = self.t.numel()
        return bool(torch.isnan(self.raw[:self.pad]).all() and torch.isnan(self.raw[self.pad + n:]).all())


def randn(gen, *shape, dtype, scale=1.0, offset=0):
    """A contiguous tensor that starts `offset` elements behind a 256-byte boundary."""
    n = math.prod(shape)
    raw = torch.empty(n + offset, device="cuda", dtype=dtype)
    raw[offset:] = (torch.randn(n, device="cuda", generator=gen) * scale).to(dtype)
    return raw[offset:].view(shape)


def store(x, layout):
    """x [..., R, C] laid out row-major (0) or column-major (1), as a contiguous buffer."""
    return x.transpose(-1, -2).contiguous() if layout else x.contiguous()


def view(buf, rows, cols, layout, lead=()):
    """The [..., rows, cols] matrix that a buffer in `layout` holds."""
    return buf.view(*lead, cols, rows).transpose(-1, -2) if layout else buf.view(*lead, rows, cols)
