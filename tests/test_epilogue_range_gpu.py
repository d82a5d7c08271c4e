"""Activations and slopes over the whole range of the types, on the GPU: where x^2 or x^3 leaves f32's
range, at the types' largest values, at the infinities (the limits) and at NaN, through every epilogue
that evaluates them; and the exact gelu's tail.

Z is given exactly: forward, A is zero and the bias holds the values; gradient, the product is 2.
From |z| = 1e4 on, relu, silu and both gelus are z or 0 and their slopes 1 or 0 to well below a
half step of f32, so the results there have to be equal.  (gelu'(x) - 1 = x phi(x) < e^-(5e7); the
sigmoids differ from 0 and 1 by e^-1e4.)  At the infinities: act(inf) = inf, act(-inf) = 0, slopes 1
and 0; "none" passes everything on.
"""
import pytest
import torch

import rocm_wmma_gemm_b200 as g
from epilogue_util import ACTS, DTYPES, U, eval_error, rounding, slope, store, value, view

pytestmark = pytest.mark.gpu

FAR = [1e4, 3e4, 1e10, 1e15, 1.8e19, 2e19, 1e30, 3e38, float("inf")]
NEAR = [0.0, 0.25, 0.5, 1.0, 3.0, 5.0, 9.0, 20.0, 60.0, 87.0, 89.0, 104.0, 1000.0]


@pytest.fixture(scope="module")
def L():
    return g.loader()


@pytest.fixture(autouse=True)
def _device_ok():
    yield
    g.device_status()


def values(dtype, nan=False):
    """Every value the type holds of FAR, NEAR and its largest, with both signs, and NaN on request."""
    top = torch.finfo(dtype).max
    v = [x for x in FAR if x <= top or x == float("inf")] + NEAR + [float(top)]
    v += [-x for x in v] + ([float("nan")] if nan else [])
    return torch.tensor(v, dtype=torch.float64, device="cuda").to(dtype)


def filled(v, *shape):
    """v over and over, in the given shape."""
    n = torch.Size(shape).numel()
    return v.repeat(n // v.numel() + 1)[:n].view(shape)


def limits(z, act, f):
    """f (value or slope) of z in 64 bits, with its limits at the infinities."""
    z = z.double()
    if act == "none":
        return z if f is value else torch.ones_like(z)
    y = f(z.clamp(-1e300, 1e300) if act != "gelu_tanh" else z.clamp(-1e100, 1e100), act)
    return torch.where(z == float("inf"), z if f is value else torch.ones_like(z),
                       torch.where(z == float("-inf"), torch.zeros_like(z), y))


def same(got, want, tol, z, what):
    """Equal where |z| >= 1e4 (as the result's type holds it), within tol elsewhere, NaN where z is."""
    nan = torch.isnan(z)
    assert torch.isnan(got[nan]).all(), f"{what}: a NaN was lost"
    far = z.abs() >= 1e4
    w = want.to(got.dtype)
    bad = far & ~nan & (got != w)
    assert not bad.any(), f"{what}: {got[bad][:4].tolist()}, not {w[bad][:4].tolist()}, at {z[bad][:4].tolist()}"
    near = ~far & ~nan
    over = (got.double() - want).abs()[near] - tol[near] - rounding(want, got.dtype)[near]
    assert not (over > 0).any() and torch.isfinite(got[near].double()).all(), f"{what}: off by {over.max().item():.3g} more than allowed"


def check_values(got, z, act, what):
    """got = act(z); z holds the unrounded values."""
    same(got, limits(z, act, value), z.double().abs() * eval_error(z.double(), act), z, what)


def check_slopes(got, z, act, what, factor=2.0):
    tol = factor * ((1 + z.double().abs()) * eval_error(z.double(), act) + 2 * U)
    same(got, factor * limits(z, act, slope), tol, z, what)


# (M, N, K, layouts) of tiles, pairs, swapped slabs, K partitions in clusters and in the workspace, sizes TMA cannot address
DENSE = [(300, 264, 136, (0, 0, 1)), (2048, 1024, 64, (0, 0, 1)), (16, 256, 128, (0, 0, 1)), (16, 512, 2048, (0, 0, 1)),
         (192, 8192, 4096, (0, 0, 0)), (128, 1024, 8192, (0, 0, 1)), (264, 300, 136, (1, 0, 0)), (256, 16, 128, (1, 0, 0)), (67, 131, 75, (0, 0, 0))]
TYPES = [("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16")]
ids = lambda t: "_".join(map(str, t[:3]))  # noqa: E731


@pytest.mark.parametrize("M,N,K,layouts", DENSE, ids=lambda v: str(v))
@pytest.mark.parametrize("pair", TYPES, ids=ids)
def test_forward(L, M, N, K, layouts, pair):
    out, dt = DTYPES[pair[0]], DTYPES[pair[1]]
    bias = filled(values(out, nan=True), N)
    a, b = torch.zeros(M, K, device="cuda", dtype=dt), torch.ones(N, K, device="cuda", dtype=dt)
    for act in ACTS:
        c = torch.full((M * N,), 7.0, device="cuda", dtype=out)
        L.gemm_fused(c, a, b, M, N, K, *layouts, activation=act, bias=bias)
        check_values(view(c, M, N, layouts[0]), bias.expand(M, N), act, act)


@pytest.mark.parametrize("M,N,K,layouts", DENSE, ids=lambda v: str(v))
@pytest.mark.parametrize("pair", TYPES, ids=ids)
def test_gradient(L, M, N, K, layouts, pair):
    out, dt = DTYPES[pair[0]], DTYPES[pair[1]]
    z = filled(values(out), M, N)
    a, b = torch.zeros(M, K, device="cuda", dtype=dt), torch.zeros(N, K, device="cuda", dtype=dt)
    (a.view(K, M)[0] if layouts[1] else a[:, 0]).fill_(1.0)  # the product is 2 everywhere, exactly
    (b[:, 0] if layouts[2] else b.view(K, N)[0]).fill_(2.0)
    bg = torch.empty(N, device="cuda")
    for act in ACTS:
        c = torch.full((M * N,), 7.0, device="cuda", dtype=out)
        L.gemm_fused(c, a, b, M, N, K, *layouts, activation=act, preact=store(z, layouts[0]), gradient=True, bias_grad=bg)
        check_slopes(view(c, M, N, layouts[0]), z, act, act)
        d = 2 * limits(z, act, slope)
        tol = 2 * ((1 + z.double().abs().clamp(max=1e4)) * eval_error(z.double(), act) * (z.abs() < 1e4) + 2 * U) + (M + 8) * 2 * U * d.abs()
        assert ((bg - d.sum(0)).abs() <= tol.sum(0)).all(), act


# few rows per group (swapped one-CTA tiles), one-CTA tiles, pairs with the rows as N, with the rows as M
@pytest.mark.parametrize("counts,N", [([4, 0, 7, 2], 1024), ([100, 0, 60], 256), ([1000, 0, 1500, 1500], 1024), ([1000, 0, 1500, 1500], 1025)], ids=str)
@pytest.mark.parametrize("pair", TYPES, ids=ids)
def test_grouped(L, counts, N, pair):
    out, dt = DTYPES[pair[0]], DTYPES[pair[1]]
    E, T, K = len(counts), sum(counts), 64
    offs = torch.tensor([sum(counts[:e]) for e in range(E + 1)], dtype=torch.int32, device="cuda")
    owner = torch.repeat_interleave(torch.arange(E), torch.tensor(counts)).cuda()
    bias, z = filled(values(out, nan=True), E, N), filled(values(out), T, N)
    a, b = torch.zeros(T, K, device="cuda", dtype=dt), torch.zeros(E, N, K, device="cuda", dtype=dt)
    b[:, :, 0] = 2
    for act in ACTS:
        c = torch.full((T, N), 7.0, device="cuda", dtype=out)
        a[:, 0] = 0
        L.gemm_grouped(c, a, b, offs, T, N, K, E, layout_b=1, activation=act, bias=bias)
        check_values(c, bias[owner], act, act)
        a[:, 0] = 1
        bg = torch.empty(E, N, device="cuda")
        L.gemm_grouped(c, a, b, offs, T, N, K, E, layout_b=1, activation=act, preact=z, gradient=True, bias_grad=bg)
        check_slopes(c, z, act, act)
        assert torch.isfinite(bg).all()


@pytest.mark.parametrize("M,N", [(40, 264), (1000, 131), (3000, 72)])
@pytest.mark.parametrize("layout", (0, 1))
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
def test_activation_backward(L, M, N, layout, out):
    dt = DTYPES[out]
    z = filled(values(dt, nan=True), M, N)
    dy = torch.full((M, N), 2.0, device="cuda", dtype=dt)
    for act in ACTS:
        dz = torch.empty(M * N, device="cuda", dtype=dt)
        L.activation_backward(dz, store(dy, layout), store(z, layout), M, N, layout=layout, activation=act)
        got = view(dz, M, N, layout)
        if act == "none":
            assert (got == 2).all()
        else:
            check_slopes(got, z, act, act)


def test_exact_gelu_tail(L):
    """The exact gelu's value and slope between -9 and 9 in f32.  The tail 1 - Phi(|x|) = t q(t) e^(-x^2/2) is
    off by 0.75e-7 (half of Abramowitz and Stegun's 1.5e-7 for erf) and by its evaluation: t's 1.8e-7
    (a rounding, a reciprocal of one unit) times t d(tq)/dt <= 1.72, the five steps of the polynomial
    1e-7, the exponential 1.7e-7 of at most 1/2 and its argument's rounding 2^-23 x^2/2: below
    (5.5e-7 + 2^-23 x^2/2) e^(-x^2/2) together.  An absolute error: relative to the value it grows on
    the left.  The density x phi(x) shares the exponential."""
    n = 1 << 16
    x = torch.linspace(-9, 9, n, device="cuda")
    xd = x.double()
    e = torch.exp(-xd * xd / 2)
    tail = 0.75e-7 + (5.5e-7 + 2.0 ** -23 * xd * xd / 2) * e
    a, b, c = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(n, 64, device="cuda", dtype=torch.bfloat16), torch.empty(8, n, device="cuda")
    L.gemm_fused(c, a, b, 8, n, 64, layout_b=1, activation="gelu", bias=x)
    want = value(xd, "gelu")
    over = (c - want).abs() - xd.abs() * tail - 4 * U * want.abs()
    assert (over <= 0).all(), over.max().item()
    dz, one = torch.empty(8, n, device="cuda"), torch.ones(8, n, device="cuda")
    L.activation_backward(dz, one, x.expand(8, n).contiguous(), 8, n, activation="gelu")
    want = slope(xd, "gelu")
    over = (dz - want).abs() - tail - xd.abs() * e * 0.4 * (1.7e-7 + 2.0 ** -23 * xd * xd / 2 + 4 * U) - 4 * U * want.abs()
    assert (over <= 0).all(), over.max().item()
