"""CPU tests of the Python view of the products with epilogues: first calls of several threads, and
which tensors it takes.  Tensors are stand-ins (a shape, a type, a device; no memory behind them)."""
import threading

import pytest


class Tensor:
    """What the Python view looks at of a CUDA tensor."""

    def __init__(self, dtype, n=1 << 20, device=0, address=0x10000000):
        self.dtype, self.n, self.device, self.address = dtype, n, device, address
        self.is_cuda = True

    def get_device(self):
        return self.device

    def numel(self):
        return self.n

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.address


@pytest.mark.parametrize("at", ("_cuda_getCurrentRawStream", "_cuda_getDevice"))
def test_first_calls_of_two_threads(gemm_lib, monkeypatch, at):
    """A thread whose first call falls into another's set-up finds all of it or does it itself."""
    import torch
    L = gemm_lib.loader()
    spec = (("A", Tensor(torch.float32), 16, None),)
    errors, results, inside = [], [], []

    def call():
        try:
            results.append(L._arguments(None, spec)[0])
        except Exception as e:  # noqa: BLE001 (reported below)
            errors.append(e)

    class Calls:
        """torch._C that lets the other thread make its call when the name `at` is looked up."""

        def __getattr__(self, name):
            if name == at and not inside:
                inside.append(name)
                t = threading.Thread(target=call)
                t.start()
                t.join()
            return {"_cuda_getCurrentRawStream": lambda index: 0, "_cuda_getDevice": lambda: 0}[name]

    for name in [n for n in vars(gemm_lib.loader) if n in ("_raw_stream", "_raw_device", "_torch_cuda", "_cuda")]:
        monkeypatch.setattr(gemm_lib.loader, name, None)  # as before any call
    monkeypatch.setattr(torch, "_C", Calls())
    call()
    assert not errors and len(results) == 2 and set(results) == {None}, errors


C, A, B, SIDE, OFF = [0x10000000 * (i + 1) for i in range(5)]  # addresses, never dereferenced


@pytest.mark.parametrize("types,out,inp", [(("f32", "bf16"), "float32", "bfloat16"), (0, "float16", "float16")])
def test_tensors_beside_addresses(gemm_lib, monkeypatch, types, out, inp):
    """With some arguments given as addresses, the tensors among the others still have the types that
    the call takes: a narrower one would end before the kernels do."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("stand-in addresses: only for processes without a GPU")
    L = gemm_lib.loader()
    monkeypatch.setattr(gemm_lib.loader, "_cuda", (lambda index: 0, lambda: 0, torch.cuda))
    other = {torch.float32: torch.bfloat16, torch.float16: torch.float32, torch.bfloat16: torch.uint8}
    co, io = getattr(torch, out), getattr(torch, inp)
    bad_c, bad_i = Tensor(other[co]), Tensor(other[io])
    calls = [
        lambda: L.gemm_fused(C, A, bad_i, 8, 8, 8, types=types),
        lambda: L.gemm_fused(C, A, B, 8, 8, 8, bias=bad_c, types=types),
        lambda: L.gemm_fused(C, A, B, 8, 8, 8, residual=bad_c, types=types),
        lambda: L.gemm_fused(C, A, B, 8, 8, 8, preact=bad_c, types=types),
        lambda: L.gemm_fused(C, Tensor(io), B, 8, 8, 8, residual=bad_c, types=types),
        lambda: L.gemm_grouped(C, A, bad_i, OFF, 8, 8, 8, 1, types=types),
        lambda: L.gemm_grouped(C, A, B, OFF, 8, 8, 8, 1, bias=bad_c, types=types),
        lambda: L.gemm_grouped(C, A, B, OFF, 8, 8, 8, 1, preact=bad_c, gradient=True, activation="relu", types=types),
        lambda: L.gemm_grouped_wgrad(C, A, bad_i, OFF, 8, 8, 8, 1, types=types),
        lambda: L.activation_backward(bad_c, A, B, 8, 8, activation="relu", types=types),
        lambda: L.activation_backward(C, A, bad_c, 8, 8, activation="relu", types=types),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="is torch"):
            call()
            pytest.fail(f"call {i} was taken")
    ok = [lambda: L.gemm_fused(C, A, Tensor(io, address=B), 8, 8, 8, bias=Tensor(co, address=SIDE), types=types),
          lambda: L.gemm_grouped_wgrad(C, A, Tensor(io, address=B), OFF, 8, 8, 8, 1, types=types),
          lambda: L.activation_backward(C, A, Tensor(co, address=SIDE), 8, 8, activation="relu", types=types)]
    for call in ok:  # accepted: all that stops these is the missing device
        with pytest.raises(gemm_lib.GemmError, match="no CUDA device"):
            call()
