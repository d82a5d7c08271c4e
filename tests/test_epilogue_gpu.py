"""GPU tests of the products with epilogues, the grouped products and their gradients against the
operators in 64 bits (tests/epilogue_util.py derives the tolerances)."""
import itertools
import zlib

import pytest
import torch

import rocm_wmma_gemm_b200 as g
from epilogue_util import (ACTS, DTYPES, PAIRS, Guarded, check, check_sum, forward, gradient, product, randn, slope, store,
                           value, view)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    return g.loader()


@pytest.fixture(autouse=True)
def _device_ok():
    yield
    assert g.device_status() == 0


def make_gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def fused(L, M, N, K, pair=("bf16", "bf16"), layouts=(0, 0, 1), batch=1, act="gelu_tanh", bias=True, residual=True, preact=True,
          grad=False, bias_grad=True, own_bias=False, in_place=False, offset=0, seed=0):
    """One call of gemm_fused, every output checked."""
    lc, la, lb = layouts
    out, dt = DTYPES[pair[0]], DTYPES[pair[1]]
    gen = torch.Generator(device="cuda").manual_seed(1000 + seed + 7 * M + 11 * N + 13 * K)
    lead = (batch,)
    a = randn(gen, batch, *((K, M) if la else (M, K)), dtype=dt, offset=offset)
    b = randn(gen, batch, *((N, K) if lb else (K, N)), dtype=dt, scale=max(K, 1) ** -0.5, offset=offset)
    A, B = view(a, M, K, la, lead), view(b, K, N, lb, lead)
    shape = (batch, N, M) if lc else (batch, M, N)
    c = Guarded(shape, out, offset=offset)
    stride = N if own_bias else 0
    nb = batch if own_bias else 1
    kw = dict(layout_c=lc, layout_a=la, layout_b=lb, batch_count=batch, activation=act, bias_stride=stride)
    if grad:
        zs = randn(gen, *shape, dtype=out, offset=offset)
        Z = view(zs, M, N, lc, lead).clone()
        if in_place and act != "none":
            c.t.copy_(zs)
            zs = c.t
        bg = Guarded((nb, N), torch.float32) if bias_grad else None
        L.gemm_fused(c.t, a, b, M, N, K, preact=zs if act != "none" else None, gradient=True, bias_grad=bg.t if bg else None, **kw)
        x, ex = product(A, B)
        d, ed = gradient(x, ex, Z, act)
        check(view(c.t, M, N, lc, lead), d, ed, "C")
        if bg:
            assert bg.intact()
            check_sum(bg.t if own_bias else bg.t[0], d, ed, 1 if own_bias else (0, 1), "bias_grad")
    else:
        bv = randn(gen, nb, N, dtype=out, offset=offset) if bias else None
        rs = randn(gen, *shape, dtype=out, offset=offset) if residual else None
        R = view(rs, M, N, lc, lead).clone() if residual else None
        if in_place and residual:
            c.t.copy_(rs)
            rs = c.t
        z = Guarded(shape, out, offset=offset) if preact else None
        L.gemm_fused(c.t, a, b, M, N, K, bias=bv, residual=rs, preact=z.t if z else None, **kw)
        y, ey, Z, ez = forward(A, B, act, bv[:, None, :] if bias else None, R)
        check(view(c.t, M, N, lc, lead), y, ey, "C")
        if z:
            assert z.intact(), "wrote outside preact"
            check(view(z.t, M, N, lc, lead), Z, ez, "preact")
    assert c.intact(), "wrote outside C"


SMALL = [(1, 1, 1), (1, 8, 8), (5, 7, 9), (16, 520, 200), (33, 65, 17), (64, 128, 64), (129, 264, 72), (300, 96, 1032), (200, 40, 0)]


@pytest.mark.parametrize("M,N,K", SMALL)
@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: "_".join(p))
def test_fused_small(L, M, N, K, pair):
    for i, act in enumerate(ACTS):
        fused(L, M, N, K, pair, act=act, residual=i % 2 == 0, preact=i % 3 != 0, bias=i != 3, seed=i)
        fused(L, M, N, K, pair, act=act, grad=True, bias_grad=i != 1, seed=i)


@pytest.mark.parametrize("layouts", list(itertools.product((0, 1), repeat=3)), ids=lambda t: "c%da%db%d" % t)
@pytest.mark.parametrize("M,N,K", [(24, 200, 136), (136, 24, 328), (200, 264, 520), (67, 131, 75)])
def test_fused_layouts(L, M, N, K, layouts):
    fused(L, M, N, K, layouts=layouts)
    fused(L, M, N, K, ("f32", "f16"), layouts=layouts, act="silu")
    fused(L, M, N, K, ("f16", "f16"), layouts=layouts, act="gelu", grad=True)


@pytest.mark.parametrize("layout_c", (0, 1))
@pytest.mark.parametrize("own_bias", (False, True), ids=("shared", "own"))
@pytest.mark.parametrize("M,N,K", [(16, 136, 64), (160, 72, 136), (9, 21, 13)])
def test_fused_batched(L, M, N, K, own_bias, layout_c):
    for batch in (2, 5):
        fused(L, M, N, K, batch=batch, layouts=(layout_c, 0, 0), own_bias=own_bias)
        fused(L, M, N, K, ("f32", "bf16"), batch=batch, layouts=(layout_c, 0, 1), own_bias=own_bias, grad=True)


@pytest.mark.parametrize("M,N,K,pair,layouts", [
    (2048, 2048, 512, ("bf16", "bf16"), (0, 0, 1)), (2048, 5120, 1024, ("f32", "bf16"), (0, 0, 1)),
    (1111, 1544, 264, ("f16", "f16"), (1, 0, 0)), (4096, 4096, 512, ("bf16", "bf16"), (0, 0, 0)),
    (16, 8192, 1024, ("bf16", "bf16"), (0, 0, 1)), (48, 2048, 4096, ("f16", "f16"), (0, 0, 0)),
    (128, 2048, 4096, ("bf16", "bf16"), (0, 0, 1)), (128, 1024, 8192, ("f32", "f16"), (0, 0, 1)),
    (8192, 64, 512, ("bf16", "bf16"), (0, 0, 1)), (16, 4096, 1024, ("bf16", "bf16"), (1, 0, 1)),
    (256, 512, 4096, ("bf16", "bf16"), (0, 0, 0)), (2304, 2560, 576, ("bf16", "bf16"), (0, 0, 1)),
    (1000, 1000, 1000, ("bf16", "bf16"), (0, 0, 1)), (999, 1001, 1003, ("bf16", "bf16"), (0, 0, 1)),
])
def test_fused_tiles(L, M, N, K, pair, layouts):
    """Sizes that take the different tiles, slabs and K partitions of the plan."""
    fused(L, M, N, K, pair, layouts)
    fused(L, M, N, K, pair, layouts, act="none", preact=False)
    fused(L, M, N, K, pair, layouts, act="relu", bias=False, residual=False)
    fused(L, M, N, K, pair, layouts, act="silu", grad=True)
    fused(L, M, N, K, pair, layouts, act="none", grad=True)


@pytest.mark.parametrize("M,N,K,layouts,pair", [
    (16, 64, 64, (1, 0, 0), "bf16"), (16, 64, 2048, (1, 0, 0), "bf16"), (32, 64, 2048, (1, 0, 0), "f16"),      # narrow tiles, K partitions in the workspace
    (16, 64, 2048, (0, 0, 0), "bf16"), (192, 512, 8192, (0, 0, 0), "bf16"), (192, 1024, 8192, (0, 0, 0), "f16"),
    (192, 8192, 64, (0, 0, 0), "bf16"), (512, 8192, 64, (0, 0, 0), "bf16"),                                     # 128 x 128 and 128 x 256 tiles
    (100, 4096, 4096, (1, 0, 0), "f32"), (192, 8192, 4096, (0, 0, 0), "bf16"),                                  # K partitions in clusters
    (192, 8192, 2048, (0, 0, 1), "f32"), (192, 4096, 4096, (0, 0, 1), "bf16"), (512, 8192, 2048, (0, 0, 1), "f32"),  # CTA pairs, widths 160 to 224
    (512, 8192, 1024, (0, 0, 1), "bf16"), (1024, 8192, 1024, (0, 0, 0), "bf16"), (1024, 8192, 1024, (0, 0, 0), "f32"),  # 256 and 512 wide
    (16, 128, 64, (0, 0, 0), "bf16"), (16, 128, 2048, (0, 0, 0), "bf16"), (48, 128, 2048, (0, 0, 0), "f32"),    # operands swapped
    (16, 512, 2048, (0, 0, 1), "bf16"), (32, 512, 2048, (0, 0, 1), "f32"), (256, 64, 2048, (1, 0, 0), "bf16"),  # and K partitions in clusters
    (16, 256, 0, (0, 0, 1), "bf16"), (300, 256, 0, (1, 0, 0), "f32"), (2048, 1024, 0, (0, 0, 0), "bf16"),
])
def test_fused_every_kernel(L, M, N, K, layouts, pair):
    """Every kernel the plan can choose, each mode of the epilogue."""
    p = (pair, "bf16" if pair != "f16" else "f16")
    for i, act in enumerate(("gelu", "none", "silu")):
        fused(L, M, N, K, p, layouts, act=act, residual=i != 1, preact=i != 2, seed=i)
        fused(L, M, N, K, p, layouts, act=act, residual=False, bias=i != 0, preact=False, seed=i)
        fused(L, M, N, K, p, layouts, act=act, grad=True, bias_grad=i != 1, seed=i)
    fused(L, M, N, K, p, layouts, act="relu", in_place=True, offset=1)  # C, residual and Z between 16-byte boundaries
    fused(L, M, N, K, p, layouts, act="relu", in_place=True, grad=True, offset=1)


def test_past_32_bits(L):
    """Matrices of more than 2^31 elements: rows from both ends and the middle."""
    M, N, K = 66000, 32776, 64
    gen = make_gen("large")
    bf = torch.bfloat16
    a, b = randn(gen, M, K, dtype=bf), randn(gen, N, K, dtype=bf, scale=K ** -0.5)
    c = torch.randn(M * N // 8, device="cuda", generator=gen).to(bf).repeat(8).view(M, N)
    rows = torch.tensor([0, 1, 127, 128, M // 2, 65535, 65536, M - 130, M - 1], device="cuda")
    res, bias = c[rows].clone(), randn(gen, N, dtype=bf)
    L.gemm_fused(c, a, b, M, N, K, layout_b=1, activation="silu", bias=bias, residual=c)
    y, ey, _, _ = forward(a[rows], b.t(), "silu", bias, res)
    check(c[rows], y, ey, "fused")
    # the same rows as four groups (weights shared by copying), gradient in place with bias sums
    offs, T, spans = ragged([1000, 64000, 0, 1000])
    w = b.repeat(4, 1, 1)
    z, bg = c[rows].clone(), torch.empty(4, N, device="cuda")
    L.gemm_grouped(c, a, w, offs, T, N, K, 4, layout_b=1, activation="silu", preact=c, gradient=True, bias_grad=bg)
    d, ed = gradient(*product(a[rows], b.t()), z, "silu")
    check(c[rows], d, ed, "grouped")
    dz, s = c[rows].clone(), torch.empty(N, device="cuda")
    L.activation_backward(c, c, c, M, N, activation="relu", bias_grad=s)
    check(c[rows], *gradient(dz.double(), torch.zeros(len(rows), N, device="cuda", dtype=torch.float64), dz, "relu"), "backward")


def test_fused_in_place(L):
    for M, N, K in [(16, 512, 256), (300, 520, 264), (7, 9, 11)]:
        for pair in PAIRS:
            fused(L, M, N, K, pair, in_place=True)
            fused(L, M, N, K, pair, in_place=True, grad=True)


@pytest.mark.parametrize("offset", (1, 4, 8))
def test_fused_unaligned(L, offset):
    """Buffers that start between 16-byte boundaries."""
    for M, N, K in [(16, 512, 256), (130, 264, 136)]:
        fused(L, M, N, K, offset=offset)
        fused(L, M, N, K, ("f32", "f16"), offset=offset, grad=True, layouts=(1, 0, 0))


def test_fused_is_the_product(L):
    """Without an epilogue the call computes what gemm computes."""
    gen = make_gen("plain")
    a, b = randn(gen, 192, 320, dtype=torch.bfloat16), randn(gen, 448, 320, dtype=torch.bfloat16)
    c, d = (torch.empty(192, 448, device="cuda") for _ in range(2))
    L.gemm_fused(c, a, b, 192, 448, 320, layout_b=1)
    L.gemm(d, a, b, 192, 448, 320, layout_b=1)
    x, ex = product(a, b.t())
    check(c, x, ex)
    check(d, x, ex)


def test_fused_empty(L):
    bg = torch.full((40,), 7.0, device="cuda")
    a = torch.ones(8, 8, dtype=torch.float16, device="cuda")
    L.gemm_fused(a, a, torch.ones(8, 40, dtype=torch.float16, device="cuda"), 0, 40, 8, gradient=True, bias_grad=bg)
    assert (bg == 0).all(), "a bias gradient over no rows is zero"
    c = torch.full((4, 6), 5.0, device="cuda", dtype=torch.float16)
    L.gemm_fused(c, a, a, 4, 0, 8)
    assert (c == 5).all()


def test_infinities_stay_in_their_rows(L):
    """A NaN or infinity in one row of A reaches that row of C only."""
    for M, N, K in [(16, 256, 128), (300, 264, 136), (9, 11, 13)]:
        gen = make_gen(M)
        a, b = randn(gen, M, K, dtype=torch.bfloat16), randn(gen, N, K, dtype=torch.bfloat16, scale=K ** -0.5)
        a[M // 2, 3], a[M // 2, 5] = float("nan"), float("inf")
        c = torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
        for act in ACTS:
            L.gemm_fused(c, a, b, M, N, K, layout_b=1, activation=act)
            rows = torch.arange(M, device="cuda") != M // 2
            assert torch.isnan(c[~rows]).all()
            y, ey, _, _ = forward(a[rows], b.t(), act)
            check(c[rows], y, ey)


# ------------------------------------------------------------------------------ grouped products
def ragged(counts, head=0, tail=0):
    """(offsets tensor, rows, spans) of groups of the given sizes behind `head` unowned rows."""
    offs = [head]
    for c in counts:
        offs.append(offs[-1] + c)
    return torch.tensor(offs, dtype=torch.int32, device="cuda"), offs[-1] + tail, list(zip(offs[:-1], offs[1:]))


COUNTS = {
    "one row": [1],
    "ones": [1] * 9,
    "empty ends": [0, 5, 0, 0, 130, 0],
    "all empty": [0, 0, 0],
    "around a tile": [127, 128, 129, 0, 255, 257],
    "ragged": [3, 64, 0, 17, 300, 1, 31, 33, 96],
    "many": [i % 7 for i in range(70)],
    "one big": [0, 900],
}


def grouped(L, counts, N, K, pair=("bf16", "bf16"), lb=0, act="silu", bias=True, residual=True, preact=True, grad=False,
            bias_grad=True, head=0, tail=0, in_place=False, offset=0, seed=0):
    out, dt = DTYPES[pair[0]], DTYPES[pair[1]]
    offs, T, spans = ragged(counts, head, tail)
    E = len(counts)
    gen = torch.Generator(device="cuda").manual_seed(2000 + seed + 7 * T + 11 * N + 13 * K)
    a = randn(gen, T, K, dtype=dt, offset=offset)
    b = randn(gen, E, *((N, K) if lb else (K, N)), dtype=dt, scale=max(K, 1) ** -0.5, offset=offset)
    B = view(b, K, N, lb, (E,))
    owned = torch.zeros(T, dtype=torch.bool, device="cuda")
    owned[head:T - tail] = True
    a[~owned] = float("nan")  # unowned rows reach no result
    c = Guarded((T, N), out, offset=offset)
    if grad:
        zs = randn(gen, T, N, dtype=out, offset=offset)
        Z = zs.clone()
        if in_place:
            c.t.copy_(zs)
            zs = c.t
        bg = Guarded((E, N), torch.float32) if bias_grad else None
        before = c.t.clone()
        L.gemm_grouped(c.t, a, b, offs, T, N, K, E, layout_b=lb, activation=act, preact=zs, gradient=True, bias_grad=bg.t if bg else None)
        for e, (p, q) in enumerate(spans):
            x, ex = product(a[p:q], B[e])
            d, ed = gradient(x, ex, Z[p:q], act)
            check(c.t[p:q], d, ed, f"C of group {e}")
            if bg:
                check_sum(bg.t[e], d, ed, 0, f"bias_grad of group {e}")
        assert bg is None or bg.intact()
    else:
        bv = randn(gen, E, N, dtype=out, offset=offset) if bias else None
        rs = randn(gen, T, N, dtype=out, offset=offset) if residual else None
        R = rs.clone() if residual else None
        if in_place and residual:
            c.t.copy_(rs)
            rs = c.t
        z = Guarded((T, N), out, offset=offset) if preact else None
        before = c.t.clone()
        L.gemm_grouped(c.t, a, b, offs, T, N, K, E, layout_b=lb, activation=act, bias=bv, residual=rs, preact=z.t if z else None)
        for e, (p, q) in enumerate(spans):
            y, ey, Z, ez = forward(a[p:q], B[e], act, bv[e] if bias else None, R[p:q] if residual else None)
            check(c.t[p:q], y, ey, f"C of group {e}")
            if z:
                check(z.t[p:q], Z, ez, f"preact of group {e}")
        if z:
            assert z.intact()
            assert torch.isnan(z.t[~owned]).all(), "wrote preact rows that belong to no group"
    assert c.intact()
    assert torch.equal(c.t[~owned].view(torch.uint8), before[~owned].view(torch.uint8)), "wrote rows that belong to no group"


@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("lb", (0, 1))
def test_grouped_counts(L, name, lb):
    for N, K in [(136, 72), (264, 328), (40, 8), (13, 21)]:
        grouped(L, COUNTS[name], N, K, lb=lb, head=3, tail=5)
        grouped(L, COUNTS[name], N, K, lb=lb, grad=True, act="gelu_tanh", head=2, tail=1)


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: "_".join(p))
def test_grouped_types(L, pair):
    for i, act in enumerate(ACTS):
        for lb in (0, 1):
            grouped(L, COUNTS["ragged"], 200, 136, pair, lb, act=act, residual=i % 2 == 0, preact=i % 3 != 0, bias=i != 2, seed=i)
            grouped(L, COUNTS["ragged"], 200, 136, pair, lb, act=act, grad=True, bias_grad=i != 1, seed=i)
            grouped(L, COUNTS["ragged"], 200, 136, pair, lb, act=act, in_place=True, grad=i % 2 == 0 and act != "none", seed=i)


@pytest.mark.parametrize("counts,N,K,lb", [
    ([4, 0, 7, 2, 3, 1, 8, 5], 2048, 1024, 1), ([4, 0, 7, 2, 3, 1, 8, 5], 2048, 1024, 0),
    ([40, 0, 70, 20, 33, 10, 80, 50], 1024, 512, 1), ([90, 200, 0, 77, 300], 1032, 520, 0),
    ([1000, 0, 513, 300], 768, 512, 1), ([2000, 0, 1513, 2300], 1536, 256, 0), ([0, 0, 0, 64], 4096, 64, 1),
])
def test_grouped_sizes(L, counts, N, K, lb):
    for pair in (("bf16", "bf16"), ("f32", "f16")):
        grouped(L, counts, N, K, pair, lb, head=1, tail=3)
        grouped(L, counts, N, K, pair, lb, head=1, tail=3, grad=True)
        grouped(L, counts, N, K, pair, lb, act="none", bias=False, residual=False, preact=False)


def test_grouped_many_groups(L):
    grouped(L, [(i * 7) % 5 for i in range(g.MAX_GROUPS)], 64, 64, head=1)
    grouped(L, [(i * 7) % 5 for i in range(g.MAX_GROUPS)], 64, 64, head=1, grad=True)


@pytest.mark.parametrize("offset", (1, 4))
def test_grouped_unaligned(L, offset):
    grouped(L, COUNTS["ragged"], 136, 72, offset=offset)
    grouped(L, COUNTS["ragged"], 136, 72, offset=offset, grad=True)


def running_offsets(offs, rows):
    out, top = [], 0
    for o in offs:
        top = max(top, min(max(o, 0), rows))
        out.append(top)
    return out


BAD_OFFSETS = [[0, 50, 20, 90], [-5, 30, 10 ** 9, 40], [90, 10, 0, 0], [2 ** 31 - 1] * 4, [-2 ** 31] * 4]


@pytest.mark.parametrize("offs", BAD_OFFSETS)
def test_grouped_offsets_outside_the_rule(L, offs):
    """Taken as their running maximum, clamped to the rows: nothing outside is touched."""
    T, N, K, E = 90, 136, 72, len(offs) - 1
    gen = make_gen("offsets")
    a = randn(gen, T, K, dtype=torch.bfloat16)
    b = randn(gen, E, K, N, dtype=torch.bfloat16, scale=K ** -0.5)
    o = torch.tensor(offs, dtype=torch.int64).to(torch.int32).cuda()
    real = running_offsets(offs, T)
    c, bg = Guarded((T, N), torch.bfloat16), Guarded((E, N), torch.float32)
    zs = randn(gen, T, N, dtype=torch.bfloat16)
    L.gemm_grouped(c.t, a, b, o, T, N, K, E, activation="silu", preact=zs, gradient=True, bias_grad=bg.t)
    w = Guarded((E, K, N), torch.float32)
    L.gemm_grouped_wgrad(w.t, a, zs, o, T, K, N, E)
    dz = Guarded((T, N), torch.bfloat16)
    s = Guarded((E, N), torch.float32)
    L.activation_backward(dz.t, zs, zs, T, N, activation="silu", bias_grad=s.t, offsets=o, groups=E)
    for e, (p, q) in enumerate(zip(real[:-1], real[1:])):
        x, ex = product(a[p:q], b[e])
        d, ed = gradient(x, ex, zs[p:q], "silu")
        check(c.t[p:q], d, ed)
        check_sum(bg.t[e], d, ed, 0)
        check(w.t[e], *product(a[p:q].t(), zs[p:q]))
        d, ed = gradient(zs[p:q].double(), torch.zeros(q - p, N, device="cuda", dtype=torch.float64), zs[p:q], "silu")
        check(dz.t[p:q], d, ed)
        check_sum(s.t[e], d, ed, 0)
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[real[0]:real[-1]] = False
    assert torch.isnan(c.t[rest]).all() and torch.isnan(dz.t[rest]).all()
    assert c.intact() and bg.intact() and w.intact() and dz.intact() and s.intact()


# ------------------------------------------------------------------------------ weight gradient
def wgrad(L, counts, M, N, pair=("bf16", "bf16"), lc=0, accumulate=False, head=0, tail=0, offset=0):
    out, dt = DTYPES[pair[0]], DTYPES[pair[1]]
    offs, T, spans = ragged(counts, head, tail)
    E = len(counts)
    gen = torch.Generator(device="cuda").manual_seed(3000 + 7 * T + 11 * N + 13 * M)
    a, b = randn(gen, T, M, dtype=dt, offset=offset), randn(gen, T, N, dtype=dt, offset=offset)
    for x in (a, b):  # rows that belong to no group reach no result
        x[:head] = float("nan")
        x[T - tail:] = float("inf")
    c = Guarded((E, N, M) if lc else (E, M, N), out, offset=offset)
    if accumulate:
        c.t.copy_(torch.randn(c.t.shape, device="cuda", generator=gen))
    before = view(c.t, M, N, lc, (E,)).clone()
    L.gemm_grouped_wgrad(c.t, a, b, offs, T, M, N, E, layout_c=lc, accumulate=accumulate)
    got = view(c.t, M, N, lc, (E,))
    for e, (p, q) in enumerate(spans):
        y, ey, _, _ = forward(a[p:q].t(), b[p:q], "none", None, before[e] if accumulate else None)
        check(got[e], y, ey, f"group {e}")
    assert c.intact()


@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("lc", (0, 1))
def test_wgrad_counts(L, name, lc):
    for M, N in [(72, 136), (264, 328), (8, 40), (13, 21)]:
        wgrad(L, COUNTS[name], M, N, lc=lc, head=3, tail=5)
        wgrad(L, COUNTS[name], M, N, lc=lc, accumulate=True, head=1)


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: "_".join(p))
@pytest.mark.parametrize("lc", (0, 1))
def test_wgrad_types(L, pair, lc):
    for counts, M, N in [(COUNTS["ragged"], 200, 136), ([700, 0, 300], 512, 768), ([64, 128, 0, 65], 1032, 520)]:
        wgrad(L, counts, M, N, pair, lc, head=2, tail=2)
        wgrad(L, counts, M, N, pair, lc, accumulate=True, tail=7)


def test_wgrad_neighbours_with_infinities(L):
    """A NaN in one group's rows stays in that group's gradient."""
    counts = [37, 70, 5]
    offs, T, spans = ragged(counts)
    gen = make_gen("wnan")
    a, b = randn(gen, T, 136, dtype=torch.bfloat16), randn(gen, T, 264, dtype=torch.bfloat16)
    a[spans[1][0]], b[spans[1][1] - 1] = float("nan"), float("inf")
    c = torch.empty(3, 136, 264, device="cuda")
    L.gemm_grouped_wgrad(c, a, b, offs, T, 136, 264, 3)
    for e in (0, 2):
        p, q = spans[e]
        check(c[e], *product(a[p:q].t(), b[p:q]))
    assert torch.isnan(c[1]).any()


def test_wgrad_without_rows(L):
    offs = torch.zeros(4, dtype=torch.int32, device="cuda")
    a = torch.empty(0, 72, device="cuda", dtype=torch.bfloat16)
    for lc in (0, 1):
        c = Guarded((3, 72, 136), torch.float32)
        L.gemm_grouped_wgrad(c.t, a, a, offs, 0, 72, 136, 3, layout_c=lc)
        assert (c.t == 0).all() and c.intact()
        c.t.fill_(5)
        L.gemm_grouped_wgrad(c.t, a, a, offs, 0, 72, 136, 3, layout_c=lc, accumulate=True)
        assert (c.t == 5).all()


def test_wgrad_unaligned(L):
    wgrad(L, COUNTS["ragged"], 72, 136, offset=1)
    wgrad(L, COUNTS["ragged"], 72, 136, ("f32", "f16"), lc=1, offset=4, accumulate=True)


# ------------------------------------------------------------------------------ activation backward
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout", (0, 1))
@pytest.mark.parametrize("M,N", [(1, 1), (7, 9), (64, 264), (333, 1000), (2000, 136), (5, 5000), (257, 4100)])
def test_activation_backward(L, M, N, layout, out):
    dt = DTYPES[out]
    for i, act in enumerate(ACTS):
        for batch, own in [(1, False), (3, True), (3, False)]:
            for offset in (0, 1):
                gen = make_gen(M, N, i)
                shape = (batch, N, M) if layout else (batch, M, N)
                dy, z = randn(gen, *shape, dtype=dt, offset=offset), randn(gen, *shape, dtype=dt, offset=offset)
                dz, bg = Guarded(shape, dt, offset=offset), Guarded((batch if own else 1, N), torch.float32)
                L.activation_backward(dz.t, dy, z, M, N, layout=layout, batch_count=batch, activation=act, bias_grad=bg.t, bias_stride=N if own else 0)
                Y, Z = view(dy, M, N, layout, (batch,)).double(), view(z, M, N, layout, (batch,))
                d, ed = gradient(Y, torch.zeros_like(Y), Z, act)
                check(view(dz.t, M, N, layout, (batch,)), d, ed, "dZ")
                check_sum(bg.t if own else bg.t[0], d, ed, 1 if own else (0, 1), "bias_grad")
                assert dz.intact() and bg.intact()
                if offset:
                    # in place and sums only
                    only = torch.empty_like(bg.t)
                    L.activation_backward(None, dy, z, M, N, layout=layout, batch_count=batch, activation=act, bias_grad=only, bias_stride=N if own else 0)
                    assert torch.equal(only, bg.t)
                    target = dy if i % 2 else z
                    L.activation_backward(target, dy, z, M, N, layout=layout, batch_count=batch, activation=act)
                    assert torch.equal(target, dz.t)


@pytest.mark.parametrize("name", COUNTS)
def test_activation_backward_grouped(L, name):
    for N in (136, 21, 1000):
        offs, T, spans = ragged(COUNTS[name], 2, 3)
        gen = make_gen(name, N)
        dy, z = randn(gen, T, N, dtype=torch.bfloat16), randn(gen, T, N, dtype=torch.bfloat16)
        dz, bg = Guarded((T, N), torch.bfloat16), Guarded((len(spans), N), torch.float32)
        L.activation_backward(dz.t, dy, z, T, N, activation="gelu", bias_grad=bg.t, offsets=offs, groups=len(spans))
        for e, (p, q) in enumerate(spans):
            Y = dy[p:q].double()
            d, ed = gradient(Y, torch.zeros_like(Y), z[p:q], "gelu")
            check(dz.t[p:q], d, ed)
            check_sum(bg.t[e], d, ed, 0)
        assert torch.isnan(dz.t[:2]).all() and torch.isnan(dz.t[T - 3:]).all() and dz.intact() and bg.intact()


# ------------------------------------------------------------------------------ the slopes by differences
@pytest.mark.parametrize("act", ACTS)
def test_slope_is_the_difference_quotient(L, act):
    """The gradient the library computes against differences of the value it computes.

    Central differences with step h of values off by e: |quotient - slope| <= h^2/6 max|act'''| + e/h.
    |act'''| <= 3.2 for the smooth activations, e = |x| EVAL(x) + u|x| <= 8 (2^-20 (1 + 42) + u) (the
    sigmoid argument of the tanh form is 42 at |x| = 8), h = 2^-4: 0.0021 + 0.0053.  relu is
    exact away from 0; its values are exact.  The product is with the identity: exact."""
    x = torch.linspace(-8, 8, 2048, device="cuda").to(torch.float16).float()
    x = x[x.abs() > 0.1] if act == "relu" else x
    x = x[: x.numel() // 64 * 64].view(-1, 64)
    h = 2.0 ** -4
    eye = torch.eye(64, device="cuda", dtype=torch.float16)

    def val(t):
        c, b = torch.empty_like(t), torch.zeros(64, device="cuda")
        M = t.shape[0]
        # x enters as the residual-free bias path cannot take a matrix: pass it as the pre-activation's product
        L.gemm_fused(c, t.to(torch.float16), eye, M, 64, 64, bias=b, activation=act)
        return c

    xp, xm = (x + h).to(torch.float16).float(), (x - h).to(torch.float16).float()
    quotient = (val(xp).double() - val(xm).double()) / (xp - xm).double()
    ones = torch.empty_like(x)
    L.activation_backward(ones, torch.ones_like(x), x, x.shape[0], 64, activation=act)
    assert (quotient - ones.double()).abs().max().item() <= 0.0075
    # and the gradient epilogue has the same slope
    c = torch.empty_like(x)
    L.gemm_fused(c, torch.ones_like(x).to(torch.float16), eye, x.shape[0], 64, 64, activation=act, preact=x, gradient=True)
    assert (c - ones).abs().max().item() <= 2.0 ** -22


# ------------------------------------------------------------------------------ a layer, forward and backward
def test_two_layer_block_and_its_gradients(L):
    """y = gelu(x W1 + b1) W2 + b2 + x and every gradient of <y, dy>, as a training step runs them,
    against the formulas in 64 bits with the intermediate roundings the calls make, and the
    gradients against differences of the 64-bit loss."""
    M, D, H = 200, 264, 520
    gen = make_gen("mlp")
    bf = torch.bfloat16
    x, dy = randn(gen, M, D, dtype=bf), randn(gen, M, D, dtype=bf)
    w1, w2 = randn(gen, D, H, dtype=bf, scale=D ** -0.5), randn(gen, H, D, dtype=bf, scale=H ** -0.5)
    b1, b2 = randn(gen, H, dtype=bf, scale=0.1), randn(gen, D, dtype=bf, scale=0.1)
    z, h, dz = (torch.empty(M, H, device="cuda", dtype=bf) for _ in range(3))
    y, dx = (torch.empty(M, D, device="cuda", dtype=bf) for _ in range(2))
    dw1, dw2 = torch.empty(D, H, device="cuda"), torch.empty(H, D, device="cuda")
    db1, db2 = torch.empty(H, device="cuda"), torch.empty(D, device="cuda")
    L.gemm_fused(h, x, w1, M, H, D, activation="gelu", bias=b1, preact=z)
    L.gemm_fused(y, h, w2, M, D, H, bias=b2, residual=x)
    L.activation_backward(None, dy, None, M, D, bias_grad=db2)
    L.gemm(dw2, h, dy, H, D, M, layout_a=1)                       # h^T dy
    L.gemm_fused(dz, dy, w2, M, H, D, layout_b=1, activation="gelu", preact=z, gradient=True, bias_grad=db1)
    L.gemm(dw1, x, dz, D, H, M, layout_a=1)                       # x^T dz
    L.gemm_fused(dx, dz, w1, M, D, H, layout_b=1, residual=dy)
    hh, eh, zz, ez = forward(x, w1, "gelu", b1)
    check(h, hh, eh)
    check(z, zz, ez)
    yy, ey, _, _ = forward(h, w2, "none", b2, x)
    check(y, yy, ey)
    check_sum(db2, dy.double(), torch.zeros_like(dy, dtype=torch.float64), 0)
    check(dw2, *product(h.t(), dy))
    d, ed = gradient(*product(dy, w2.t()), z, "gelu")
    check(dz, d, ed)
    check_sum(db1, d, ed, 0)
    check(dw1, *product(x.t(), dz))
    check(dx, *forward(dz, w1.t(), "none", None, dy)[:2])

    # directional differences of the loss in 64 bits: the stored gradients carry bf16 roundings of z, h
    # and dz (2^-8 relative each, independent over thousands of elements): 2 % of the norms' product
    p = {"x": x, "w1": w1, "w2": w2, "b1": b1, "b2": b2}
    p = {k: v.double() for k, v in p.items()}
    grads = {"x": dx, "w1": dw1, "w2": dw2, "b1": db1, "b2": db2}

    def loss(q):
        return ((value(q["x"] @ q["w1"] + q["b1"], "gelu") @ q["w2"] + q["b2"] + q["x"]) * dy.double()).sum().item()

    for k, gr in grads.items():
        v = gr.double() / gr.double().norm()  # along the gradient: the quotient is its norm
        step = 1e-4
        hi, lo = ({**p, k: p[k] + s * step * v} for s in (1, -1))
        quotient = (loss(hi) - loss(lo)) / (2 * step)
        assert abs(quotient - gr.double().norm().item()) <= 0.02 * gr.double().norm().item(), k


def test_expert_block_and_its_gradients(L):
    """The same over experts with ragged rows: grouped products, grouped gradients, weight gradients."""
    counts, D, H = [70, 0, 33, 129, 1], 136, 264
    offs, T, spans = ragged(counts)
    E = len(counts)
    gen = make_gen("moe")
    bf = torch.bfloat16
    x, dy = randn(gen, T, D, dtype=bf), randn(gen, T, D, dtype=bf)
    w1, w2 = randn(gen, E, H, D, dtype=bf, scale=D ** -0.5), randn(gen, E, D, H, dtype=bf, scale=H ** -0.5)
    b1, b2 = randn(gen, E, H, dtype=bf, scale=0.1), randn(gen, E, D, dtype=bf, scale=0.1)
    z, h, dz = (torch.empty(T, H, device="cuda", dtype=bf) for _ in range(3))
    y, dx = (torch.empty(T, D, device="cuda", dtype=bf) for _ in range(2))
    dw1, dw2 = torch.empty(E, H, D, device="cuda"), torch.empty(E, D, H, device="cuda")
    db1, db2 = torch.empty(E, H, device="cuda"), torch.empty(E, D, device="cuda")
    L.gemm_grouped(h, x, w1, offs, T, H, D, E, layout_b=1, activation="silu", bias=b1, preact=z)
    L.gemm_grouped(y, h, w2, offs, T, D, H, E, layout_b=1, bias=b2, residual=x)
    L.activation_backward(None, dy, None, T, D, bias_grad=db2, offsets=offs, groups=E)
    L.gemm_grouped_wgrad(dw2, h, dy, offs, T, H, D, E, layout_c=1)
    L.gemm_grouped(dz, dy, w2, offs, T, H, D, E, layout_b=0, activation="silu", preact=z, gradient=True, bias_grad=db1)
    L.gemm_grouped_wgrad(dw1, x, dz, offs, T, D, H, E, layout_c=1)
    L.gemm_grouped(dx, dz, w1, offs, T, D, H, E, layout_b=0, residual=dy)
    total = {k: 0.0 for k in ("x", "w1", "w2", "b1", "b2")}
    for e, (p, q) in enumerate(spans):
        hh, eh, zz, ez = forward(x[p:q], w1[e].t(), "silu", b1[e])
        check(h[p:q], hh, eh)
        check(z[p:q], zz, ez)
        yy, ey, _, _ = forward(h[p:q], w2[e].t(), "none", b2[e], x[p:q])
        check(y[p:q], yy, ey)
        check_sum(db2[e], dy[p:q].double(), torch.zeros(q - p, D, device="cuda", dtype=torch.float64), 0)
        check(dw2[e], *product(dy[p:q].t(), h[p:q]))
        d, ed = gradient(*product(dy[p:q], w2[e]), z[p:q], "silu")
        check(dz[p:q], d, ed)
        check_sum(db1[e], d, ed, 0)
        check(dw1[e], *product(dz[p:q].t(), x[p:q]))
        check(dx[p:q], *forward(dz[p:q], w1[e], "none", None, dy[p:q])[:2])

    def loss(q_):
        s = 0.0
        for e, (p, q) in enumerate(spans):
            u = value(q_["x"][p:q] @ q_["w1"][e].t() + q_["b1"][e], "silu")
            s = s + ((u @ q_["w2"][e].t() + q_["b2"][e] + q_["x"][p:q]) * dy[p:q].double()).sum()
        return float(s)

    par = {k: v.double() for k, v in {"x": x, "w1": w1, "w2": w2, "b1": b1, "b2": b2}.items()}
    for k, gr in {"x": dx, "w1": dw1, "w2": dw2, "b1": db1, "b2": db2}.items():
        v = gr.double() / gr.double().norm()
        quotient = (loss({**par, k: par[k] + 1e-4 * v}) - loss({**par, k: par[k] - 1e-4 * v})) / 2e-4
        assert abs(quotient - gr.double().norm().item()) <= 0.02 * gr.double().norm().item(), k


# ------------------------------------------------------------------------------ streams, graphs, repeats
def _work_set(gen, M=130, N=264, K=200):
    bf = torch.bfloat16
    return dict(a=randn(gen, M, K, dtype=bf), b=randn(gen, N, K, dtype=bf, scale=K ** -0.5), z=randn(gen, M, N, dtype=bf),
                c=torch.empty(M, N, device="cuda", dtype=bf), bg=torch.empty(N, device="cuda"), M=M, N=N, K=K)


def _grad_call(L, s, **kw):
    L.gemm_fused(s["c"], s["a"], s["b"], s["M"], s["N"], s["K"], layout_b=1, activation="silu", preact=s["z"], gradient=True, bias_grad=s["bg"], **kw)


def _grad_check(s):
    d, ed = gradient(*product(s["a"], s["b"].t()), s["z"], "silu")
    check(s["c"], d, ed)
    check_sum(s["bg"], d, ed, 0)


def test_streams_do_not_share_scratch(L):
    gen = make_gen("streams")
    sets = [_work_set(gen, M=900 + 30 * i) for i in range(4)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, st in zip(sets, streams):
            if _ % 2:
                _grad_call(L, s, stream=st)
            else:
                with torch.cuda.stream(st):
                    _grad_call(L, s)
    torch.cuda.synchronize()
    for s in sets:
        _grad_check(s)


def test_graphs_replay_and_do_not_share_scratch(L):
    gen = make_gen("graphs")
    sets = [_work_set(gen, M=700), _work_set(gen, M=1300)]
    offs, T, spans = ragged([100, 0, 333, 40])
    ga, gb = randn(gen, T, 136, dtype=torch.bfloat16), randn(gen, T, 264, dtype=torch.bfloat16)
    gc = torch.empty(4, 136, 264, device="cuda")
    for s in sets:
        _grad_call(L, s)  # first calls outside the capture
    L.gemm_grouped_wgrad(gc, ga, gb, offs, T, 136, 264, 4)
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            _grad_call(L, s)
            L.gemm_grouped_wgrad(gc, ga, gb, offs, T, 136, 264, 4)
        graphs.append(gr)
    for round_ in range(3):
        for s in sets:
            s["a"].copy_(torch.randn(s["a"].shape, device="cuda", generator=gen))
            s["c"].fill_(float("nan"))
            s["bg"].fill_(float("nan"))
        # other routing than at capture: the offsets are read when the kernel runs
        offs2, _, spans = ragged([[50, 373, 0, 50], [0, 0, 473, 0], [473, 0, 0, 0]][round_])
        offs.copy_(offs2)
        gc.fill_(float("nan"))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            graphs[0].replay()
        side.synchronize()
        graphs[1].replay()
        _grad_call(L, sets[0])  # an ordinary call between replays
        torch.cuda.synchronize()
        for s in sets:
            _grad_check(s)
        for e, (p, q) in enumerate(spans):
            check(gc[e], *product(ga[p:q].t(), gb[p:q]))


def test_two_host_threads(L):
    """Calls from two threads, each on its own stream."""
    import threading
    gen = make_gen("threads")
    sets = [_work_set(gen, M=500 + 100 * i, N=1032, K=2056) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    errors = []

    def work(s, st):
        try:
            with torch.cuda.stream(st):
                for _ in range(40):
                    _grad_call(L, s)
        except Exception as e:  # noqa: BLE001 (reported below)
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(sets, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for s in sets:
        _grad_check(s)


def test_two_host_threads_on_one_stream(L):
    """Scratch of different sizes, growing, with K partitions and without: the calls' launches do not mix."""
    import threading
    gen = make_gen("one stream")
    sets = [[_work_set(gen, M=m, N=n, K=k) for m, n, k in sizes] for sizes in
            ([(700, 1032, 264), (300, 1000, 2056), (3001, 2056, 136)], [(1100, 520, 136), (333, 1000, 2056), (2500, 4104, 72)])]
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    errors = []

    def work(mine):
        try:
            with torch.cuda.stream(st):
                for i in range(60):
                    for s in mine[:1 + i // 20]:
                        _grad_call(L, s)
                        L.gemm(s["p"], s["a"], s["b"], s["M"], s["N"], s["K"], layout_b=1)
        except Exception as e:  # noqa: BLE001 (reported below)
            errors.append(e)

    for s in sets[0] + sets[1]:
        s["p"] = torch.empty(s["M"], s["N"], device="cuda", dtype=torch.bfloat16)
    threads = [threading.Thread(target=work, args=(m,)) for m in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for s in sets[0] + sets[1]:
        _grad_check(s)
        check(s["p"], *product(s["a"], s["b"].t()))


def test_results_repeat_bit_for_bit(L):
    gen = make_gen("repeat")
    s = _work_set(gen, M=2000, N=520, K=1032)
    first = None
    for _ in range(4):
        s["c"].fill_(0), s["bg"].fill_(0)
        _grad_call(L, s)
        got = (s["c"].clone(), s["bg"].clone())
        assert first is None or (torch.equal(got[0], first[0]) and torch.equal(got[1], first[1]))
        first = got


def test_python_refusals(L):
    a = torch.zeros(64, 64, device="cuda", dtype=torch.bfloat16)
    c = torch.zeros(64, 64, device="cuda", dtype=torch.bfloat16)
    offs = torch.tensor([0, 64], device="cuda", dtype=torch.int32)
    bad = [
        lambda: L.gemm_fused(c, a, a, 64, 64, 65),                                    # A too short
        lambda: L.gemm_fused(c.t()[:, :32], a, a, 64, 32, 64),                        # not contiguous
        lambda: L.gemm_fused(c, a, a, 64, 64, 64, bias=torch.zeros(64, device="cuda")),   # bias is f32, C bf16
        lambda: L.gemm_fused(c, a, a, 64, 64, 64, bias=torch.zeros(63, device="cuda", dtype=torch.bfloat16)),
        lambda: L.gemm_fused(c, a, a.cpu(), 64, 64, 64),
        lambda: L.gemm_fused(c, a, a.half(), 64, 64, 64),
        lambda: L.gemm_fused(c, a, a, 64, 64, 64, activation="tanh"),
        lambda: L.gemm_fused(c, a, a, 64, 64, 64, gradient=True, bias_grad=torch.zeros(64, device="cuda", dtype=torch.bfloat16)),
        lambda: L.gemm_grouped(c, a, a, offs.long(), 64, 64, 64, 1),
        lambda: L.gemm_grouped(c, a, a, offs, 64, 64, 64, 2),                         # B and offsets too short
        lambda: L.gemm_grouped_wgrad(c, a, a, offs.cpu(), 64, 64, 64, 1),
        lambda: L.activation_backward(c, a, a[:32], 64, 64, activation="relu"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(g.GemmError):
        L.gemm_fused(c, a, a, 64, 64, 64, bias_grad=torch.zeros(64, device="cuda"))
    with pytest.raises(g.GemmError):
        L.gemm_fused(a, a, c, 64, 64, 64)  # C is A
    assert (c == 0).all() and (a == 0).all()


def test_same_sizes_in_turn(L):
    """One size in all its modes, alignments, layouts and types, in changing order: no call runs by another's plan."""
    cases = [dict(pair=p, layouts=l, offset=o, grad=gr, residual=r, preact=z, act="silu", batch=n)
             for p in PAIRS for l in ((0, 0, 1), (1, 1, 0)) for o in (0, 1, 4) for gr, r, z in
             ((False, True, True), (False, False, False), (False, True, False), (True, True, True)) for n in (1, 2)]
    for step in (1, 59, 101):  # (each without a common factor with the number of cases)
        for i in range(len(cases)):
            fused(L, 128, 256, 1024, **cases[i * step % len(cases)])


# ------------------------------------------------------------------------------ corners of what the documentation allows
def strided_bias(L, M, N, K, batch, stride, pair=("bf16", "bf16"), layouts=(0, 0, 1), act="silu"):
    """Bias and bias gradient vectors further apart than they are long; what lies between is left as it is."""
    out, dt = DTYPES[pair[0]], DTYPES[pair[1]]
    lc, la, lb = layouts
    gen = make_gen("stride", M, N, K, batch, stride)
    a = randn(gen, batch, *((K, M) if la else (M, K)), dtype=dt)
    b = randn(gen, batch, *((N, K) if lb else (K, N)), dtype=dt, scale=max(K, 1) ** -0.5)
    A, B = view(a, M, K, la, (batch,)), view(b, K, N, lb, (batch,))
    shape = (batch, N, M) if lc else (batch, M, N)
    length = (batch - 1) * stride + N
    where = (torch.arange(batch, device="cuda")[:, None] * stride + torch.arange(N, device="cuda")).flatten()
    flat = torch.full((length,), float("nan"), dtype=out, device="cuda")
    bias = randn(gen, batch, N, dtype=out)
    flat[where] = bias.flatten()
    c, z = Guarded(shape, out), Guarded(shape, out)
    kw = dict(layout_c=lc, layout_a=la, layout_b=lb, batch_count=batch, activation=act, bias_stride=stride)
    L.gemm_fused(c.t, a, b, M, N, K, bias=flat, preact=z.t, **kw)
    y, ey, Z, ez = forward(A, B, act, bias[:, None, :])
    check(view(c.t, M, N, lc, (batch,)), y, ey, "C")
    check(view(z.t, M, N, lc, (batch,)), Z, ez, "preact")
    sums = [Guarded((length,), torch.float32) for _ in range(2)]
    for s in sums:
        s.t.fill_(7.0)
    Z = view(z.t, M, N, lc, (batch,)).clone()
    L.gemm_fused(c.t, a, b, M, N, K, preact=z.t, gradient=True, bias_grad=sums[0].t, **kw)
    d, ed = gradient(*product(A, B), Z, act)
    check(view(c.t, M, N, lc, (batch,)), d, ed, "gradient")
    dy = c.t.clone()
    L.activation_backward(c.t, dy, z.t, M, N, layout=lc, batch_count=batch, activation=act, bias_grad=sums[1].t, bias_stride=stride)
    d2, ed2 = gradient(view(dy, M, N, lc, (batch,)).double(), torch.zeros_like(d), Z, act)
    check(view(c.t, M, N, lc, (batch,)), d2, ed2, "backward")
    for s, (v, e) in zip(sums, ((d, ed), (d2, ed2))):
        check_sum(s.t[where].view(batch, N), v, e, 1, "bias_grad")
        s.t[where] = 7.0
        assert (s.t == 7.0).all() and s.intact(), "wrote between the vectors"
    assert c.intact() and z.intact()


@pytest.mark.parametrize("layouts", [(0, 0, 1), (1, 0, 0)], ids=("rows", "columns"))
@pytest.mark.parametrize("M,N,K,batch,stride", [(16, 136, 64, 3, 139), (160, 72, 136, 4, 1000), (192, 512, 8192, 2, 515), (16, 64, 2048, 5, 64), (9, 21, 13, 2, 22)])
def test_fused_bias_stride(L, M, N, K, batch, stride, layouts):
    strided_bias(L, M, N, K, batch, stride, layouts=layouts)
    strided_bias(L, M, N, K, batch, stride, ("f32", "f16"), layouts, act="gelu")


@pytest.mark.parametrize("layout_c", (0, 1))
def test_many_items(L, layout_c):
    """More batch items than a grid's second and third extent."""
    for M, N, K, batch in [(3, 8, 8, 66000), (8, 5, 3, 70001)]:
        fused(L, M, N, K, batch=batch, layouts=(layout_c, 0, 0), own_bias=True)
        fused(L, M, N, K, batch=batch, layouts=(layout_c, 0, 0), own_bias=True, grad=True)
        fused(L, M, N, K, batch=batch, layouts=(layout_c, 0, 0), grad=True)
    strided_bias(L, 2, 8, 8, 66001, 9, layouts=(layout_c, 0, 0))


@pytest.mark.parametrize("lb", (0, 1))
def test_grouped_without_k_and_narrow(L, lb):
    for N, K in [(136, 0), (1, 64), (8, 1), (1, 1), (5, 0)]:
        for counts in (COUNTS["ragged"], COUNTS["all empty"], [700, 0, 500]):
            grouped(L, counts, N, K, lb=lb, head=2, tail=3)
            grouped(L, counts, N, K, ("f32", "f16"), lb=lb, grad=True, act="gelu_tanh", head=1)
    for M, N in [(1, 1), (1, 264), (264, 1)]:
        wgrad(L, COUNTS["ragged"], M, N, lc=lb)
        wgrad(L, COUNTS["all empty"], M, N, lc=lb, accumulate=True)


def test_no_rows_at_all(L):
    """Every group empty and no rows: sums and weight gradients are zero, everything else is left alone."""
    E, N, K = g.MAX_GROUPS, 24, 16
    offs = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    bf = torch.bfloat16
    none, w = torch.empty(0, K, device="cuda", dtype=bf), torch.ones(E, K, N, device="cuda", dtype=bf)
    for call in ("product", "backward"):
        bg = Guarded((E, N), torch.float32)
        empty = torch.empty(0, N, device="cuda", dtype=bf)
        if call == "product":
            L.gemm_grouped(empty, none, w, offs, 0, N, K, E, activation="relu", preact=empty, gradient=True, bias_grad=bg.t)
        else:
            L.activation_backward(empty, empty, empty, 0, N, activation="relu", bias_grad=bg.t, offsets=offs, groups=E)
        assert (bg.t == 0).all() and bg.intact()
    dw = Guarded((E, K, N), torch.float32)
    empty = torch.empty(0, N, device="cuda", dtype=bf)
    L.gemm_grouped_wgrad(dw.t, none, empty, offs, 0, K, N, E)
    assert (dw.t == 0).all()
    dw.t.fill_(3.0)
    L.gemm_grouped_wgrad(dw.t, none, empty, offs, 0, K, N, E, accumulate=True)
    assert (dw.t == 3).all() and dw.intact()
