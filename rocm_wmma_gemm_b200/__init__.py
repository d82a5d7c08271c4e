"""B200-native half-precision GEMM behind the C ABI of adelj88/rocm_wmma_gemm.

This package is a thin ctypes view of `librocm_wmma_gemm_sm100a.so` (hand-written sm_100a
kernels + the C ABI of include/b200_gemm.h).  It mirrors the reference's host interface:

* `m_layout`                       rocm_wmma_gemm/include/rocm_wmma_gemm/kernel/common.hpp:38-42
* `loader().gemm(...)`             rocm_wmma_gemm/include/rocm_wmma_gemm/kernel_loader.hpp:132-154
* `get_gemm_params(...)`           generated by rocm_wmma_gemm/config/generate_config.py:286-303

There is no CPU path: importing works anywhere (so the symbols can be checked), but every
compute call needs a B200 and raises if the library or the device is missing.
"""
from __future__ import annotations

import ctypes
import enum
import os
from typing import Optional

from . import build as _build

__all__ = [
    "m_layout", "loader", "GemmConfig", "GemmError", "lib", "get_gemm_params", "slab",
    "Epilogue", "ACTIVATIONS", "MAX_GROUPS", "TYPE_PAIRS", "ABI_SYMBOLS", "device_status", "static_status", "launch_count", "plan", "PlanInfo", "RASTER_SNAKE",
]


class m_layout(enum.IntEnum):
    """Matrix storage order; the integer values are part of the C ABI."""
    row_major = 0
    col_major = 1


class GemmError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"b200_gemm status {status}: {message}")
        self.status = status


class GemmConfig(ctypes.Structure):
    """Mirror of `b200_gemm_config` (include/b200_gemm.h)."""
    _fields_ = [("tile_m", ctypes.c_int), ("tile_n", ctypes.c_int), ("stages", ctypes.c_int),
                ("cluster", ctypes.c_int), ("split_k", ctypes.c_int), ("raster", ctypes.c_int)]

    def as_dict(self) -> dict:
        return {k: getattr(self, k) for k, _ in self._fields_}

    def __repr__(self) -> str:
        return "GemmConfig(" + ", ".join(f"{k}={v}" for k, v in self.as_dict().items()) + ")"


class Epilogue(ctypes.Structure):
    """Mirror of `b200_gemm_epilogue` (include/b200_gemm.h)."""
    _fields_ = [("activation", ctypes.c_int), ("gradient", ctypes.c_int), ("bias", ctypes.c_void_p),
                ("residual", ctypes.c_void_p), ("preact", ctypes.c_void_p), ("bias_grad", ctypes.c_void_p),
                ("bias_stride", ctypes.c_size_t)]


# Activation names -> b200_gemm_activation
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu_tanh": 3, "gelu": 4}
MAX_GROUPS = 1024  # B200_GEMM_MAX_GROUPS


class PlanInfo(ctypes.Structure):
    """Mirror of `b200_gemm_plan_info` (include/b200_gemm.h)."""
    KERNELS = {0: "none", 1: "generic", 2: "staged", 3: "transposed"}
    _fields_ = [("kernel", ctypes.c_int), ("tile_m", ctypes.c_int), ("tile_n", ctypes.c_int),
                ("cluster", ctypes.c_int), ("split_k", ctypes.c_int), ("slots", ctypes.c_int),
                ("k_blocks_per_slot", ctypes.c_int), ("raster", ctypes.c_int), ("ctas", ctypes.c_int),
                ("work_units", ctypes.c_longlong), ("cluster_k", ctypes.c_int)]

    def as_dict(self) -> dict:
        d = {k: getattr(self, k) for k, _ in self._fields_}
        d["kernel"] = self.KERNELS.get(self.kernel, str(self.kernel))
        return d

    def short(self) -> str:
        """One-line description, e.g. `transposed 56x16 k1 4kb/slot x5 147 CTAs`."""
        if self.kernel <= 1:
            return self.KERNELS[self.kernel]
        return (f"{self.KERNELS[self.kernel]} {self.tile_m}x{self.tile_n} k{self.split_k} "
                f"{self.k_blocks_per_slot}kb/slot x{self.slots} r{self.raster} {self.ctas} CTAs")


# (output, input) -> type index; numbering of the reference's kernel_launcher type_idx.
TYPE_PAIRS = {("f16", "f16"): 0, ("f32", "f16"): 1, ("bf16", "bf16"): 2, ("f32", "bf16"): 3}
_SUFFIX = {0: "f16_f16", 1: "f32_f16", 2: "bf16_bf16", 3: "f32_bf16"}

_GEMM_ARGS = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t,
              ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int, ctypes.c_int, ctypes.c_int,
              ctypes.c_void_p]

# Every symbol include/b200_gemm.h declares: name -> (restype, argtypes)
ABI_SYMBOLS = {
    **{f"rocm_wmma_gemm_{s}": (None, _GEMM_ARGS) for s in _SUFFIX.values()},
    **{f"b200_gemm_{s}": (ctypes.c_int, _GEMM_ARGS) for s in _SUFFIX.values()},
    "b200_gemm_ex": (ctypes.c_int, [ctypes.c_int] + _GEMM_ARGS + [ctypes.POINTER(GemmConfig)]),
    "b200_gemm_splitk_static": (ctypes.c_int, [ctypes.c_int] + _GEMM_ARGS + [ctypes.POINTER(GemmConfig)]),
    "b200_gemm_select_config": (ctypes.c_int, [ctypes.c_size_t] * 3 + [ctypes.c_int] * 4
                                + [ctypes.POINTER(GemmConfig)]),
    "b200_gemm_plan": (ctypes.c_int, [ctypes.c_int] + [ctypes.c_size_t] * 4 + [ctypes.c_int] * 4
                       + [ctypes.POINTER(PlanInfo)]),
    "b200_gemm_host": (ctypes.c_int, [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
                       + [ctypes.c_size_t] * 4 + [ctypes.c_int] * 3),
    "b200_gemm_slab": (ctypes.c_int, [ctypes.c_size_t, ctypes.c_int, ctypes.c_int, ctypes.c_size_t,
                                      ctypes.POINTER(ctypes.c_size_t), ctypes.POINTER(ctypes.c_size_t)]),
    "b200_gemm_workspace_bytes": (ctypes.c_size_t, [ctypes.c_int] + [ctypes.c_size_t] * 4
                                  + [ctypes.c_int] * 3 + [ctypes.POINTER(GemmConfig)]),
    "b200_gemm_device_status": (ctypes.c_int, [ctypes.POINTER(ctypes.c_uint)]),
    "b200_gemm_static_status": (ctypes.c_int, [ctypes.POINTER(ctypes.c_uint)]),
    # multi-GPU column-slab driver
    "b200_gemm_comm_id": (ctypes.c_int, [ctypes.c_void_p]),
    "b200_gemm_comm_create": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_void_p)]),
    "b200_gemm_comm_destroy": (ctypes.c_int, [ctypes.c_void_p]),
    "b200_gemm_comm_barrier": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "b200_gemm_comm_allgather_inplace": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "b200_gemm_peer_alloc": (ctypes.c_int, [ctypes.c_size_t, ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p]),
    "b200_gemm_peer_open": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]),
    "b200_gemm_peer_close": (ctypes.c_int, [ctypes.c_void_p]),
    "b200_gemm_peer_free": (ctypes.c_int, [ctypes.c_void_p]),
    "b200_gemm_slab_allgather": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                                ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int, ctypes.c_size_t, ctypes.c_void_p]),
    "b200_gemm_slab_host": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                           ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int, ctypes.c_int,
                                           ctypes.c_int, ctypes.c_size_t]),
    "b200_gemm_slab_push": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p, ctypes.c_size_t,
                                           ctypes.c_size_t, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_size_t,
                                           ctypes.c_void_p]),
    "b200_gemm_slab_gather": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p, ctypes.c_void_p,
                                             ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int, ctypes.c_int,
                                             ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_size_t, ctypes.c_void_p,
                                             ctypes.POINTER(GemmConfig)]),
    # products with epilogues, grouped products, gradients
    "b200_gemm_fused": (ctypes.c_int, [ctypes.c_int] + _GEMM_ARGS + [ctypes.POINTER(Epilogue)]),
    "b200_gemm_grouped": (ctypes.c_int, [ctypes.c_int] + [ctypes.c_void_p] * 4 + [ctypes.c_size_t] * 4
                          + [ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(Epilogue)]),
    "b200_gemm_grouped_wgrad": (ctypes.c_int, [ctypes.c_int] + [ctypes.c_void_p] * 4 + [ctypes.c_size_t] * 4
                                + [ctypes.c_int, ctypes.c_int, ctypes.c_void_p]),
    "b200_gemm_activation_backward": (ctypes.c_int, [ctypes.c_int] + [ctypes.c_void_p] * 3 + [ctypes.c_size_t] * 3
                                      + [ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
                                         ctypes.c_size_t, ctypes.c_void_p]),
    "b200_gemm_last_status": (ctypes.c_int, []),
    "b200_gemm_last_error": (ctypes.c_char_p, []),
    "b200_gemm_version": (ctypes.c_char_p, []),
    "b200_gemm_launch_count": (ctypes.c_ulonglong, []),
}

_LIB: Optional[ctypes.CDLL] = None


def lib() -> ctypes.CDLL:
    """The loaded shared library.  Raises if it has not been built; never falls back."""
    global _LIB
    if _LIB is None:
        path = _build.LIB_PATH
        if not os.path.exists(path):
            raise RuntimeError(
                f"{path} is missing: run `python -m rocm_wmma_gemm_b200.build` (needs nvcc). "
                "There is no CPU fallback.")
        handle = ctypes.CDLL(path, mode=ctypes.RTLD_LOCAL)
        for name, (res, args) in ABI_SYMBOLS.items():
            fn = getattr(handle, name)  # AttributeError if the library lacks a declared symbol
            fn.restype = res
            fn.argtypes = args
        _LIB = handle
    return _LIB


def _check(status: int) -> None:
    if status != 0:
        raise GemmError(status, lib().b200_gemm_last_error().decode())


def _ptr(x) -> int:
    if x is None:
        return 0
    if isinstance(x, int):
        return x
    return x.data_ptr()  # torch.Tensor


class loader:
    """Counterpart of `rocm_wmma_gemm::loader`: resolves the four C entry points once and
    dispatches `gemm` by (output, input) type pair.

    `gemm(C, A, B, M, N, K, layout_c, layout_a, layout_b, batch_count=1, stream=None)` takes
    torch CUDA tensors or raw device addresses.  Argument order (C, A, B; layouts C, A, B)
    is the reference's.  With `checked=True` (default) the status-returning twin is called
    and a failure raises `GemmError`; with `checked=False` the void reference symbol is
    called, which records failures instead of reporting them.
    """

    def __init__(self):
        self._lib = lib()
        self._fn = {t: getattr(self._lib, f"b200_gemm_{s}") for t, s in _SUFFIX.items()}
        self._fn_ref = {t: getattr(self._lib, f"rocm_wmma_gemm_{s}") for t, s in _SUFFIX.items()}
        self._streams = {}
        self._torch = None

    _DTYPE_INDEX = None  # {(out dtype, in dtype): type index}, filled on first use (needs torch)

    @classmethod
    def _type_index(cls, C, A, types) -> int:
        if types is not None:
            return TYPE_PAIRS[types] if isinstance(types, tuple) else int(types)
        if cls._DTYPE_INDEX is None:
            import torch
            names = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32"}
            cls._DTYPE_INDEX = {(o, i): TYPE_PAIRS[(names[o], names[i])]
                                for o in names for i in names if (names[o], names[i]) in TYPE_PAIRS}
        return cls._DTYPE_INDEX[(C.dtype, A.dtype)]

    def _stream_ptr(self, stream):
        """Pointer to a cell holding the stream handle (cached per handle: the call is hot)."""
        if stream is None:
            if self._torch is None:
                try:
                    import torch
                    self._torch = torch
                except ImportError:
                    self._torch = False
            if self._torch and self._torch.cuda.is_available():
                handle = self._torch.cuda.current_stream().cuda_stream
            else:
                return None
        else:
            handle = int(getattr(stream, "cuda_stream", stream))
        return self._cell(handle)

    def _cell(self, handle):
        cell = self._streams.get(handle)
        if cell is None:
            box = ctypes.c_void_p(handle)
            cell = (box, ctypes.cast(ctypes.pointer(box), ctypes.c_void_p))
            self._streams[handle] = cell
        return cell[1]

    def gemm(self, C, A, B, M, N, K, layout_c=0, layout_a=0, layout_b=0, batch_count=1, stream=None,
             types=None, checked=True, config: Optional[GemmConfig] = None) -> None:
        t = self._type_index(C, A, types)
        sp = self._stream_ptr(stream)
        args = (_ptr(C), _ptr(A), _ptr(B), M, N, K, batch_count, int(layout_c), int(layout_a),
                int(layout_b), sp)
        if config is not None:
            st = self._lib.b200_gemm_ex(t, *args, ctypes.byref(config))
        elif checked:
            st = self._fn[t](*args)
        else:
            self._fn_ref[t](*args)
            return
        if st != 0:
            _check(st)

    def gemm_static(self, C, A, B, M, N, K, layout_c=0, layout_a=0, layout_b=0, batch_count=1, stream=None,
                    types=None, config: Optional[GemmConfig] = None) -> None:
        """`b200_gemm_splitk_static`: the GEMM for callers that may not allocate device memory
        (split-K partials go to the library's built-in workspace; see include/b200_gemm.h)."""
        t = self._type_index(C, A, types)
        sp = self._stream_ptr(stream)
        _check(self._lib.b200_gemm_splitk_static(
            t, _ptr(C), _ptr(A), _ptr(B), M, N, K, batch_count, int(layout_c), int(layout_a), int(layout_b), sp,
            ctypes.byref(config) if config is not None else None))

    def gemm_host(self, C, A, B, M, N, K, layout_c=0, layout_a=0, layout_b=0, batch_count=1,
                  types=None) -> None:
        """Host-buffer call: C, A, B are CPU tensors / host addresses; copies are inside."""
        t = self._type_index(C, A, types)
        _check(self._lib.b200_gemm_host(t, _ptr(C), _ptr(A), _ptr(B), M, N, K, batch_count,
                                        int(layout_c), int(layout_a), int(layout_b)))

    # ---- products with epilogues, grouped products, gradients ------------------------------
    def _types_of(self, C, A, types) -> int:
        """`_type_index` for calls that check their arguments: a pair without a kernel, and `types` that are
        not those of the tensors given, are a ValueError."""
        if types is None:
            try:
                return self._DTYPE_INDEX[C.dtype, A.dtype] if self._DTYPE_INDEX is not None else self._type_index(C, A, None)
            except (KeyError, AttributeError):
                raise ValueError(f"no product {getattr(C, 'dtype', 'of an address')} from {getattr(A, 'dtype', 'an address')}: "
                                 f"one of {', '.join(map(str, TYPE_PAIRS))} (addresses need types)") from None
        pair = types if isinstance(types, tuple) else next((k for k, v in TYPE_PAIRS.items() if v == types), None)
        if pair not in TYPE_PAIRS:
            raise ValueError(f"unknown types {types!r}: one of {', '.join(map(str, TYPE_PAIRS))}")
        for t, name in zip((C, A), pair):
            if t is not None and not isinstance(t, int) and t.dtype != self._torch_type(t, self._TORCH_NAMES[name]):
                raise ValueError(f"types {types!r} do not go with a {t.dtype} tensor")
        return TYPE_PAIRS[pair]

    _TORCH_NAMES = {"f16": "float16", "bf16": "bfloat16", "f32": "float32"}
    _PAIR_DTYPES = None  # type index -> torch's (output, input) dtypes, filled on first use

    @staticmethod
    def _dtypes(t):
        """torch's (output, input) dtypes of type pair t, for calls that name their types: some arguments
        may be addresses, and the tensors among the others must still hold what the kernels read."""
        if loader._PAIR_DTYPES is None:
            try:
                import torch
            except ImportError:
                return None, None  # (so no argument is a tensor)
            loader._PAIR_DTYPES = {i: tuple(getattr(torch, loader._TORCH_NAMES[n]) for n in pair) for pair, i in TYPE_PAIRS.items()}
        return loader._PAIR_DTYPES[t]

    def _arguments(self, stream, spec):
        """(device to make current or None, stream cell, addresses) of a call's array arguments.

        `spec` holds (name, array, elements the call needs, dtype or None).  Tensors must share one
        CUDA device, be dense (contiguous; every shape is given by the sizes of the call) and at
        least as long as the call needs; raw addresses are taken as they are.  The call runs on
        the tensors' device and, where no stream is given, on that device's current stream."""
        device, addresses = None, []
        for name, t, size, dtype in spec:
            if t is None:
                addresses.append(None)
            elif isinstance(t, int):
                addresses.append(t)
            else:
                d = t.get_device()
                if device is None:
                    device = d
                if d < 0 or d != device or t.numel() < size or (dtype is not None and t.dtype != dtype) or not t.is_contiguous():
                    self._refuse(name, t, size, dtype, device)
                addresses.append(t.data_ptr())
        if device is None:
            return None, self._stream_ptr(stream), addresses
        raw_stream, raw_device, _ = loader._cuda or loader._cuda_calls()
        if stream is None:
            handle = raw_stream(device)
        else:
            owner = getattr(stream, "device_index", device)
            if owner != device:
                raise ValueError(f"the stream is on device {owner}, the tensors on device {device}")
            handle = int(getattr(stream, "cuda_stream", stream))
        return (device if raw_device() != device else None), self._cell(handle), addresses

    _cuda = None  # (a device's current raw stream, the current device, torch.cuda), from the first call with tensors on

    @staticmethod
    def _cuda_calls():
        import torch
        stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        calls = (stream, getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device), torch.cuda)
        loader._cuda = calls  # (in one piece: another thread finds all of it or nothing)
        return calls

    @staticmethod
    def _refuse(name, t, size, dtype, device):
        if not t.is_cuda or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous CUDA tensor")
        if t.get_device() != device:
            raise ValueError(f"{name} is on {t.device}, other arguments on device {device}")
        if t.numel() < size:
            raise ValueError(f"{name} holds {t.numel()} elements, the call needs {size}")
        raise ValueError(f"{name} is {t.dtype}, not {dtype}")

    @staticmethod
    def _on(device, call, *args) -> None:
        if device is None:
            st = call(*args)
        else:
            with loader._cuda[2].device(device):
                st = call(*args)
        if st != 0:
            _check(st)

    @staticmethod
    def _activation(activation) -> int:
        act = ACTIVATIONS.get(activation, activation)
        if not isinstance(act, int):
            raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
        return act

    _TORCH_TYPES = {}  # name -> torch's dtype, filled on first use

    @staticmethod
    def _torch_type(t, name):
        """torch's dtype `name` where t is a tensor (raw addresses need no torch)."""
        if t is None or isinstance(t, int):
            return None
        dtype = loader._TORCH_TYPES.get(name)
        if dtype is None:
            import torch
            dtype = loader._TORCH_TYPES[name] = getattr(torch, name)
        return dtype

    def gemm_fused(self, C, A, B, M, N, K, layout_c=0, layout_a=0, layout_b=0, batch_count=1, activation="none",
                   bias=None, residual=None, preact=None, gradient=False, bias_grad=None, bias_stride=0,
                   stream=None, types=None) -> None:
        """`b200_gemm_fused`: a product and what a layer does around it, in one kernel.

        Forward: `C = act(A*B + bias) + residual`; with `preact` given it receives `A*B + bias`.
        `gradient=True`: `C = (A*B) * act'(preact)`, and `bias_grad` (float32) receives the column
        sums of C.  `activation` is one of `ACTIVATIONS`; bias, residual and preact have C's type,
        residual and preact C's layout; residual (forward) or preact (gradient) may be C itself.
        With batch_count > 1, `bias_stride` 0 shares one bias among the items (its gradient is
        the sum over them), N or more gives each its own."""
        t = self._types_of(C, A, types)
        mn, vec = batch_count * M * N, N + (batch_count - 1) * bias_stride if N else 0
        ct, it = (C.dtype, A.dtype) if types is None else self._dtypes(t)
        dev, sp, (c, a, b, bi, re, pr, bg) = self._arguments(stream, (
            ("C", C, mn, None), ("A", A, batch_count * M * K, None), ("B", B, batch_count * K * N, it),
            ("bias", bias, vec, ct), ("residual", residual, mn, ct), ("preact", preact, mn, ct),
            ("bias_grad", bias_grad, vec, self._torch_type(bias_grad, "float32"))))
        epi = Epilogue(self._activation(activation), int(gradient), bi, re, pr, bg, bias_stride)
        self._on(dev, self._lib.b200_gemm_fused, t, c, a, b, M, N, K, batch_count, int(layout_c), int(layout_a),
                 int(layout_b), sp, ctypes.byref(epi))

    def gemm_grouped(self, C, A, B, offsets, rows, N, K, groups, layout_b=0, activation="none", bias=None,
                     residual=None, preact=None, gradient=False, bias_grad=None, stream=None, types=None) -> None:
        """`b200_gemm_grouped`: rows [offsets[e], offsets[e+1]) of A (rows x K) times matrix e of B
        (groups x K x N, each in layout_b), with the epilogues of `gemm_fused`.  `offsets` is an
        int32 tensor of groups + 1 on the device; rows outside [offsets[0], offsets[groups]) are
        left as they are.  bias and bias_grad are groups x N.  The input gradient is the same call
        on the output's gradient with layout_b flipped and N and K exchanged."""
        t = self._types_of(C, A, types)
        mn = rows * N
        ct, it = (C.dtype, A.dtype) if types is None else self._dtypes(t)
        dev, sp, (c, a, b, bi, re, pr, bg, off) = self._arguments(stream, (
            ("C", C, mn, None), ("A", A, rows * K, None), ("B", B, groups * K * N, it),
            ("bias", bias, groups * N, ct), ("residual", residual, mn, ct), ("preact", preact, mn, ct),
            ("bias_grad", bias_grad, groups * N, self._torch_type(bias_grad, "float32")),
            ("offsets", offsets, groups + 1, self._torch_type(offsets, "int32"))))
        epi = Epilogue(self._activation(activation), int(gradient), bi, re, pr, bg, 0)
        self._on(dev, self._lib.b200_gemm_grouped, t, c, a, b, off, rows, N, K, groups, int(layout_b), sp,
                 ctypes.byref(epi))

    def gemm_grouped_wgrad(self, C, A, B, offsets, rows, M, N, groups, layout_c=0, accumulate=False, stream=None,
                           types=None) -> None:
        """`b200_gemm_grouped_wgrad`: for every group `C_e = A[rows of e]^T * B[rows of e]` (added to
        C_e with `accumulate`), A rows x M, B rows x N, C groups x M x N, each C_e in layout_c.
        An empty group's C_e is zero."""
        t = self._types_of(C, A, types)
        dev, sp, (c, a, b, off) = self._arguments(stream, (
            ("C", C, groups * M * N, None), ("A", A, rows * M, None), ("B", B, rows * N, A.dtype if types is None else self._dtypes(t)[1]),
            ("offsets", offsets, groups + 1, self._torch_type(offsets, "int32"))))
        self._on(dev, self._lib.b200_gemm_grouped_wgrad, t, c, a, b, off, rows, M, N, groups, int(layout_c),
                 int(accumulate), sp)

    _OUT_TYPES = None  # torch dtype of C -> a type pair with that output

    def activation_backward(self, dZ, dY, preact, M, N, layout=0, batch_count=1, activation="none", bias_grad=None,
                            bias_stride=0, offsets=None, groups=0, stream=None, types=None) -> None:
        """`b200_gemm_activation_backward`: `dZ = dY * act'(preact)` and `bias_grad` (float32), the
        column sums of dZ, for M x N matrices.  dZ may be None (only the sums), dY or preact
        itself.  With `offsets` (int32 on the device, `groups` + 1) the rows are those of
        `gemm_grouped` and bias_grad is groups x N."""
        if types is None:
            if loader._OUT_TYPES is None:
                import torch
                loader._OUT_TYPES = {torch.float16: 0, torch.float32: 3, torch.bfloat16: 2}
            t = loader._OUT_TYPES.get(getattr(dY, "dtype", None))
            if t is None:
                raise ValueError(f"dY is {getattr(dY, 'dtype', 'an address')}: a float16, bfloat16 or float32 tensor, or give types")
        else:
            t = self._types_of(dY, None, types)
        mn, ct = batch_count * M * N, dY.dtype if types is None else self._dtypes(t)[0]
        vec = groups * N if groups else (N + (batch_count - 1) * bias_stride if N else 0)
        dev, sp, (dz, dy, z, bg, off) = self._arguments(stream, (
            ("dZ", dZ, mn, ct), ("dY", dY, mn, None), ("preact", preact, mn, ct),
            ("bias_grad", bias_grad, vec, self._torch_type(bias_grad, "float32")),
            ("offsets", offsets, groups + 1, self._torch_type(offsets, "int32"))))
        self._on(dev, self._lib.b200_gemm_activation_backward, t, dz, dy, z, M, N, batch_count, int(layout),
                 self._activation(activation), bg, bias_stride, off, groups, sp)


def get_gemm_params(m: int, n: int, k: int, layout_c=0, layout_a=0, layout_b=0, type_group: int = 0):
    """Tuned parameters for a problem (same argument order as the reference's
    `get_gemm_params(m, n, k, layout_c, layout_a, layout_b, type_group)`).
    Returns (GemmConfig, index into the compiled config list)."""
    cfg = GemmConfig()
    types = 1 if type_group == 1 else 0
    idx = lib().b200_gemm_select_config(m, n, k, types, int(layout_c), int(layout_a), int(layout_b),
                                        ctypes.byref(cfg))
    if idx < 0:
        raise GemmError(-idx, lib().b200_gemm_last_error().decode())
    return cfg, idx


def plan(m: int, n: int, k: int, layout_c=0, layout_a=0, layout_b=0, types: int = 0, batch_count: int = 1,
         sm_count: int = 0) -> PlanInfo:
    """What a call with these arguments would launch (`b200_gemm_plan`): kernel family, tile,
    K partitions, ring geometry, CTA count.  Host code only; `sm_count` 0 = the current
    device's, or 148 without a device."""
    info = PlanInfo()
    _check(lib().b200_gemm_plan(int(types), m, n, k, batch_count, int(layout_c), int(layout_a), int(layout_b),
                                int(sm_count), ctypes.byref(info)))
    return info


def slab(n: int, world: int, rank: int, align: int = 256):
    """Columns [begin, begin + count) of B and C that `rank` of `world` devices owns."""
    b, c = ctypes.c_size_t(), ctypes.c_size_t()
    _check(lib().b200_gemm_slab(n, world, rank, align, ctypes.byref(b), ctypes.byref(c)))
    return b.value, c.value


def device_status() -> int:
    """Synchronises and raises GemmError if a kernel gave up on a bounded wait."""
    word = ctypes.c_uint(0)
    _check(lib().b200_gemm_device_status(ctypes.byref(word)))
    return word.value


def static_status() -> int:
    """`device_status` for the kernels launched by `gemm_static` (their own status word)."""
    word = ctypes.c_uint(0)
    _check(lib().b200_gemm_static_status(ctypes.byref(word)))
    return word.value


RASTER_SNAKE = 128  # B200_GEMM_RASTER_SNAKE


def launch_count() -> int:
    return int(lib().b200_gemm_launch_count())
