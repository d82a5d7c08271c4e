"""Scratch of the products with epilogues under streams that come and go, and beside captures of other
threads, on the GPU."""
import ctypes
import threading

import pytest
import torch

import rocm_wmma_gemm_b200 as g
from epilogue_util import check, check_sum, gradient, product, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    return g.loader()


@pytest.fixture(autouse=True)
def _device_ok():
    yield
    g.device_status()


class Work:
    """A gradient call with bias sums whose operands need padded copies (odd K): partial sums and copies
    in scratch; and the weight gradient of ragged rows, whose tensor maps lie there."""

    def __init__(self, seed, M, N, K):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        bf = torch.bfloat16
        self.M, self.N, self.K = M, N, K
        self.a, self.b, self.z = randn(gen, M, K, dtype=bf), randn(gen, N, K, dtype=bf, scale=K ** -0.5), randn(gen, M, N, dtype=bf)
        self.c, self.bg = torch.empty(M, N, device="cuda", dtype=bf), torch.empty(N, device="cuda")
        self.offs = torch.tensor([0, M // 3, M // 3, M], dtype=torch.int32, device="cuda")
        self.w = torch.empty(3, K, N, device="cuda")

    def call(self, L, stream=None):
        L.gemm_fused(self.c, self.a, self.b, self.M, self.N, self.K, layout_b=1, activation="silu", preact=self.z, gradient=True,
                     bias_grad=self.bg, stream=stream)
        L.gemm_grouped_wgrad(self.w, self.a, self.z, self.offs, self.M, self.K, self.N, 3, stream=stream)

    def check(self):
        d, ed = gradient(*product(self.a, self.b.t()), self.z, "silu")
        check(self.c, d, ed)
        check_sum(self.bg, d, ed, 0)
        for e, (p, q) in enumerate(((0, self.M // 3), (0, 0), (self.M // 3, self.M))):
            check(self.w[e], *product(self.a[p:q].t(), self.z[p:q]))


@pytest.fixture(scope="module")
def delay():
    """Queues about a millisecond of work on the current stream."""
    big = torch.randn(8192, 8192, device="cuda").bfloat16()
    out = torch.empty_like(big)
    torch.mm(big, big, out=out)
    torch.cuda.synchronize()
    return lambda: torch.mm(big, big, out=out)


def works(n):
    w = [Work(i, 300 + 40 * (i % 3), 264 + 8 * (i % 4), 333 + 2 * (i % 5)) for i in range(n)]
    torch.cuda.synchronize()
    return w


def test_streams_destroyed_with_calls_pending(L, delay):
    """Each stream is destroyed while its calls are still queued behind other work, and a new one is made at once."""
    rt = torch.cuda.cudart()
    todo = works(12)
    for w in todo:
        box = ctypes.c_uint64(0)
        assert int(rt.cudaStreamCreate(ctypes.addressof(box))) == 0
        with torch.cuda.stream(torch.cuda.ExternalStream(box.value)):
            delay()
            w.call(L)
        assert int(rt.cudaStreamDestroy(box.value)) == 0
    torch.cuda.synchronize()
    for w in todo:
        w.check()


def test_threads_that_end_with_calls_pending(L, delay):
    """On the per-thread default stream: one handle, another stream in every thread, and the next thread
    may find itself at the address of the last one."""
    per_thread = 2  # cudaStreamPerThread
    todo, errors = works(12), []

    def call(w):
        try:
            with torch.cuda.stream(torch.cuda.ExternalStream(per_thread)):
                delay()
                w.call(L)
        except Exception as e:  # noqa: BLE001 (reported below)
            errors.append(e)

    for w in todo:
        t = threading.Thread(target=call, args=(w,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for w in todo:
        w.check()


def test_first_call_of_a_stream_beside_a_capture(L):
    """Scratch is allocated while another thread captures (in the mode that forbids other threads'
    allocations): neither the call nor the capture fails."""
    mine, other = Work(1, 320, 264, 333), Work(2, 900, 520, 777)
    mine.call(L)
    torch.cuda.synchronize()
    stream, errors = torch.cuda.Stream(), []

    def call():
        try:
            with torch.cuda.stream(stream):
                other.call(L)
        except Exception as e:  # noqa: BLE001 (reported below)
            errors.append(e)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="global"):
        mine.call(L)
        t = threading.Thread(target=call)
        t.start()
        t.join()
        mine.call(L)
    assert not errors, errors
    mine.c.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    mine.check()
    other.check()


FIRST = """
import sys; sys.path.insert(0, {root!r}); sys.path.insert(0, {tests!r})
import torch, rocm_wmma_gemm_b200 as g
from test_epilogue_streams_gpu import Work
L, w = g.loader(), Work(3, 320, 264, 333)
x = torch.ones(64, 64, device="cuda", dtype=torch.bfloat16)
L.gemm(torch.empty_like(x), x, x, 64, 64, 64)  # the plain product only
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, capture_error_mode="global"):
    w.call(L)
    L.activation_backward(w.c, w.z, w.z, w.M, w.N, activation="gelu")
    w.call(L)
graph.replay()
torch.cuda.synchronize()
w.check()
g.device_status()
print("fine")
"""


def test_first_call_is_captured(L):
    """A process that has made plain products only captures its first calls with an epilogue."""
    import os
    import subprocess
    import sys
    tests = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST.format(root=os.path.dirname(tests), tests=tests)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
