"""CPU tests of the products with epilogues and the grouped products: what the entry points
refuse before anything could run, and how the Python view names them."""
import ctypes
import os
import shutil
import subprocess

import pytest

BAD_LAYOUT, NULL, BAD_SIZE, MISALIGNED, NO_DEVICE, BAD_CONFIG = 1, 2, 3, 4, 5, 7
P = [0x10000000 * (i + 1) for i in range(8)]  # stand-in addresses, far apart, never dereferenced
C, A, B, BIAS, RES, PRE, BG, OFF = P


@pytest.fixture(scope="module")
def gl(gemm_lib):
    return gemm_lib, gemm_lib.lib()


def ran(status):
    """Accepted: all that stops the call here is the missing device."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("stand-in addresses: only for processes without a GPU")
    return status == NO_DEVICE


def fused(gl, types=2, c=C, a=A, b=B, M=64, N=64, K=64, batch=1, lc=0, la=0, lb=0, **epi):
    g, lib = gl
    e = g.Epilogue(**epi)
    return lib.b200_gemm_fused(types, c, a, b, M, N, K, batch, lc, la, lb, None, ctypes.byref(e))


@pytest.mark.parametrize("want,kw", [
    (BAD_LAYOUT, dict(lc=2)), (BAD_LAYOUT, dict(lb=-1)),
    (BAD_CONFIG, dict(types=4)),
    (BAD_SIZE, dict(M=2 ** 31)), (BAD_SIZE, dict(batch=0)),
    (NULL, dict(c=None)), (NULL, dict(a=None)),
    (MISALIGNED, dict(a=A + 1)), (MISALIGNED, dict(bias=BIAS + 1)), (MISALIGNED, dict(types=3, residual=RES + 2)),
    (MISALIGNED, dict(preact=PRE + 1)), (MISALIGNED, dict(gradient=1, bias_grad=BG + 2)),
    (BAD_CONFIG, dict(activation=5)), (BAD_CONFIG, dict(activation=-1)), (BAD_CONFIG, dict(gradient=2)),
    (BAD_CONFIG, dict(gradient=1, bias=BIAS)), (BAD_CONFIG, dict(gradient=1, residual=RES)),
    (BAD_CONFIG, dict(bias_grad=BG)),
    (NULL, dict(gradient=1, activation=2)),
    (BAD_SIZE, dict(batch=2, bias=BIAS, bias_stride=63)),
    (BAD_CONFIG, dict(c=A)), (BAD_CONFIG, dict(c=B + 64)), (BAD_CONFIG, dict(residual=C + 64)),
    (BAD_CONFIG, dict(preact=C)), (BAD_CONFIG, dict(preact=A)), (BAD_CONFIG, dict(preact=RES, residual=RES)),
    (BAD_CONFIG, dict(bias=C + 128)),
    (BAD_CONFIG, dict(gradient=1, activation=2, preact=C + 2)),
    (BAD_CONFIG, dict(gradient=1, bias_grad=C)), (BAD_CONFIG, dict(gradient=1, activation=1, preact=PRE, bias_grad=PRE + 64)),
])
def test_fused_refusals(gl, want, kw):
    g, lib = gl
    assert fused(gl, **kw) == want
    assert lib.b200_gemm_last_status() == want and lib.b200_gemm_last_error()


def test_fused_accepts(gl):
    for kw in [dict(), dict(bias=BIAS, residual=RES, preact=PRE, activation=4), dict(residual=C), dict(K=0, a=None, b=None),
               dict(gradient=1), dict(gradient=1, activation=3, preact=C, bias_grad=BG), dict(batch=3, bias=BIAS, bias_stride=64),
               dict(types=3, lc=1, la=1, lb=1, M=5, N=7, K=9)]:
        assert ran(fused(gl, **kw)), kw
    g, lib = gl
    assert ran(lib.b200_gemm_fused(2, C, A, B, 8, 8, 8, 1, 0, 0, 0, None, None))  # no epilogue: the product


def test_fused_empty_runs_nothing(gl):
    assert fused(gl, c=None, a=None, b=None, M=0) == 0
    assert fused(gl, c=None, a=None, b=None, N=0, gradient=1, bias_grad=BG) == 0


def grouped(gl, types=2, c=C, a=A, b=B, off=OFF, rows=64, N=64, K=64, groups=4, lb=0, **epi):
    g, lib = gl
    e = g.Epilogue(**epi)
    return lib.b200_gemm_grouped(types, c, a, b, off, rows, N, K, groups, lb, None, ctypes.byref(e))


@pytest.mark.parametrize("want,kw", [
    (BAD_SIZE, dict(groups=0)), (BAD_SIZE, dict(groups=1025)), (NULL, dict(off=None)), (MISALIGNED, dict(off=OFF + 2)),
    (BAD_LAYOUT, dict(lb=2)), (BAD_SIZE, dict(rows=2 ** 31)), (NULL, dict(b=None)), (BAD_CONFIG, dict(c=OFF - 128)),
    (BAD_CONFIG, dict(activation=9)), (BAD_CONFIG, dict(gradient=1, bias=BIAS)), (NULL, dict(gradient=1, activation=1)),
    (BAD_CONFIG, dict(gradient=1, bias_grad=OFF)), (BAD_CONFIG, dict(c=B + 3 * 64 * 64 * 2)),
    (BAD_CONFIG, dict(bias=C - 128)),
])
def test_grouped_refusals(gl, want, kw):
    assert grouped(gl, **kw) == want


def test_grouped_accepts(gl):
    for kw in [dict(), dict(groups=1024, N=8), dict(bias=BIAS, residual=C, preact=PRE, activation=2), dict(gradient=1, activation=2, preact=PRE, bias_grad=BG),
               dict(rows=0, gradient=1, bias_grad=BG), dict(N=7, K=5)]:
        assert ran(grouped(gl, **kw)), kw
    assert grouped(gl, rows=0) == 0


def wgrad(gl, types=3, c=C, a=A, b=B, off=OFF, rows=64, M=64, N=64, groups=4, lc=0, acc=0):
    return gl[1].b200_gemm_grouped_wgrad(types, c, a, b, off, rows, M, N, groups, lc, acc, None)


@pytest.mark.parametrize("want,kw", [
    (BAD_SIZE, dict(groups=0)), (NULL, dict(off=None)), (BAD_LAYOUT, dict(lc=2)), (BAD_CONFIG, dict(acc=2)), (BAD_CONFIG, dict(types=-1)),
    (NULL, dict(c=None)), (NULL, dict(a=None)), (MISALIGNED, dict(c=C + 2)), (BAD_CONFIG, dict(c=A - 64)), (BAD_SIZE, dict(M=2 ** 31)),
])
def test_wgrad_refusals(gl, want, kw):
    assert wgrad(gl, **kw) == want


def test_wgrad_accepts(gl):
    for kw in [dict(), dict(acc=1, lc=1), dict(rows=0, a=None, b=None), dict(M=3, N=5, types=0)]:
        assert ran(wgrad(gl, **kw)), kw
    assert wgrad(gl, M=0) == 0


def backward(gl, types=2, dz=C, dy=A, z=PRE, M=64, N=64, batch=1, layout=0, act=2, bg=BG, stride=0, off=None, groups=0):
    return gl[1].b200_gemm_activation_backward(types, dz, dy, z, M, N, batch, layout, act, bg, stride, off, groups, None)


@pytest.mark.parametrize("want,kw", [
    (BAD_CONFIG, dict(types=4)), (BAD_LAYOUT, dict(layout=2)), (BAD_CONFIG, dict(act=5)), (BAD_SIZE, dict(batch=0)), (BAD_SIZE, dict(N=2 ** 31)),
    (NULL, dict(dy=None)), (NULL, dict(z=None)), (MISALIGNED, dict(dy=A + 1)), (MISALIGNED, dict(bg=BG + 1)), (BAD_CONFIG, dict(dz=A + 2)),
    (BAD_CONFIG, dict(bg=A)), (BAD_SIZE, dict(batch=2, stride=3)), (BAD_SIZE, dict(off=OFF)), (NULL, dict(groups=2)),
    (BAD_CONFIG, dict(groups=2, off=OFF, layout=1)), (BAD_CONFIG, dict(groups=2, off=OFF, batch=2)), (BAD_SIZE, dict(groups=2000, off=OFF)),
])
def test_backward_refusals(gl, want, kw):
    assert backward(gl, **kw) == want


def test_backward_accepts(gl):
    for kw in [dict(), dict(dz=A), dict(dz=PRE), dict(dz=None), dict(act=0, z=None), dict(groups=3, off=OFF), dict(M=0, dy=None, z=None), dict(layout=1, batch=3, stride=64)]:
        assert ran(backward(gl, **kw)), kw
    assert backward(gl, dz=None, bg=None) == 0  # nothing is wanted


def test_python_names(gl):
    g, _ = gl
    assert g.ACTIVATIONS == {"none": 0, "relu": 1, "silu": 2, "gelu_tanh": 3, "gelu": 4}
    L = g.loader()
    with pytest.raises(ValueError, match="unknown activation"):
        L.gemm_fused(C, A, B, 8, 8, 8, activation="swish", types=2)
    with pytest.raises(g.GemmError):
        L.gemm_fused(C, A, B, 8, 8, 8, activation="gelu", gradient=True, types=2)


@pytest.mark.parametrize("stride", (2 ** 64 - 64, 2 ** 63, 2 ** 48))
def test_bias_strides_past_every_address(gl, stride):
    """Refused: a stride that wraps (a negative one, say) must not pass for a vector inside the tensor."""
    assert fused(gl, batch=3, bias=BIAS, bias_stride=stride) == BAD_SIZE
    assert fused(gl, batch=3, gradient=1, bias_grad=BG, bias_stride=stride) == BAD_SIZE
    assert backward(gl, batch=3, stride=stride) == BAD_SIZE


def test_python_types(gl):
    """Given types that are not the tensors', and pairs without a kernel."""
    import torch
    L = gl[0].loader()
    t = {n: torch.zeros(64, dtype=getattr(torch, n)) for n in ("float16", "bfloat16", "float32", "float64")}
    bf, f16, f32, f64 = t["bfloat16"], t["float16"], t["float32"], t["float64"]
    for c, a, types in [(bf, bf, 3), (bf, bf, ("f32", "bf16")), (f32, bf, ("f32", "f16")), (C, bf, 1), (f32, B, 2), (bf, bf, 4),
                        (bf, bf, ("bf16", "f16")), (bf, f16, None), (f64, f64, None), (f32, f32, None), (C, bf, None), (C, A, None)]:
        for call in (lambda: L.gemm_fused(c, a, a, 8, 8, 8, types=types), lambda: L.gemm_grouped(c, a, a, OFF, 8, 8, 8, 1, types=types),
                     lambda: L.gemm_grouped_wgrad(c, a, a, OFF, 8, 8, 8, 1, types=types)):
            with pytest.raises(ValueError, match="types|product"):
                call()
    for dy, types in [(f64, None), (A, None), (bf, 3), (f32, ("f16", "f16")), (bf, 9)]:
        with pytest.raises(ValueError, match="types"):
            L.activation_backward(None, dy, PRE, 8, 8, activation="relu", types=types)


CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


@pytest.fixture(scope="session")
def frontend(gemm_lib):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    return subprocess.run(["sh", os.path.join(CPP, "build_epilogue_test.sh")], check=True, capture_output=True, text=True).stdout.strip()


def test_cpp_front_end_compiles(frontend):
    assert os.path.exists(frontend)


@pytest.mark.gpu
def test_cpp_front_end(frontend):
    r = subprocess.run([frontend], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
