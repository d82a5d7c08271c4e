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
