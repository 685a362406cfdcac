"""Products with 4-bit weights for few tokens (`retro_b200_w4_*` in include/retro_b200.h) on torch CUDA tensors.

The tensors' memory goes to the library as it is: rows may be strided, calls run on the current stream of the tensors' device
(or the one given) and can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _ffi
from .engine import EngineError, InvalidArgument, _check, _last_error

_TYPES: dict = {}       # torch dtype -> GGML type code


def _torch():
    import torch

    if not _TYPES:
        _TYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 30})
    return torch


class W4Matrix:
    """A matrix, or a bank of `n_expert` matrices, of 4-bit weights laid out on a GPU.

    `rows` are the stored GGUF rows (bytes, a numpy uint8 array or a torch uint8 tensor, on the host or a GPU) of `ggml_type` 2 (Q4_0) or
    39 (MXFP4); they are read before the constructor returns and need not be kept. `device`: a CUDA device index; by default
    that of a CUDA tensor, else the current device."""

    def __init__(self, ggml_type: int, rows, n_out: int, n_in: int, n_expert: int = 1, device: int | None = None) -> None:
        self._h = None
        self._lib = lib = _ffi.load_library()
        for value in (ggml_type, n_out, n_in, n_expert):
            if not 0 <= value < 1 << 32:
                raise InvalidArgument("w4_new: a size is negative or above 32 bits")
        want = n_expert * n_out * (n_in // 32) * {2: 18, 39: 17}.get(ggml_type, 0)
        if hasattr(rows, "data_ptr"):
            if rows.element_size() != 1 or not rows.is_contiguous():
                raise InvalidArgument("w4_new: rows must be contiguous bytes")
            got, pointer = rows.numel(), rows.data_ptr()
            if rows.is_cuda and device is None:
                device = rows.device.index
        else:
            rows = np.ascontiguousarray(rows if isinstance(rows, np.ndarray) else np.frombuffer(rows, dtype=np.uint8))
            got, pointer = rows.nbytes, rows.ctypes.data
        if want and got != want:
            raise InvalidArgument(f"w4_new: rows hold {got} bytes, the shape needs {want}")
        if device is None:
            h = lib.retro_b200_w4_new(ggml_type, pointer, n_out, n_in, n_expert)
        else:
            torch = _torch()
            with torch.cuda.device(device):
                if hasattr(rows, "is_cuda") and rows.is_cuda:
                    torch.cuda.synchronize(rows.device)
                h = lib.retro_b200_w4_new(ggml_type, pointer, n_out, n_in, n_expert)
        if not h:
            raise InvalidArgument(_last_error()) if _last_error().startswith("w4_new: ") else EngineError(_last_error())
        self._h = h
        nbytes, where = C.c_uint64(), C.c_int()
        _check(lib.retro_b200_w4_info(h, None, None, C.byref(nbytes), C.byref(where)))
        self.ggml_type, self.n_out, self.n_in, self.n_expert = ggml_type, n_out, n_in, n_expert
        self.nbytes, self.device = nbytes.value, where.value

    def close(self) -> None:
        """Frees the device memory; no call that uses the matrix may be pending."""
        if self._h:
            self._lib.retro_b200_w4_free(self._h)
            self._h = None

    def __del__(self) -> None:
        try:
            self.close()
        except Exception:       # the interpreter is shutting down
            pass


def _rows(op: str, name: str, t, width: int, device: int, tokens: int = -1):
    """Pointer, type code and row stride of a [tokens, width] tensor."""
    code = _TYPES.get(t.dtype)
    shape = t.shape
    if code is None:
        raise InvalidArgument(f"{op}: {name} must be float32, float16 or bfloat16")
    if len(shape) != 2 or shape[1] != width or (tokens >= 0 and shape[0] != tokens):
        raise InvalidArgument(f"{op}: {name} has the shape {tuple(shape)}, expected [{tokens if tokens >= 0 else 'tokens'}, {width}]")
    if t.get_device() != device:
        raise InvalidArgument(f"{op}: {name} is not on the weights' device")
    ld, inner = t.stride()
    if inner != 1 and width > 1:
        raise InvalidArgument(f"{op}: the elements of a row of {name} must be consecutive")
    return t.data_ptr(), code, ld


def _vector(op: str, name: str, t, n: int, device: int):
    if t is None:
        return None
    torch = _torch()
    if t.dtype != torch.float32 or t.numel() != n or t.get_device() != device or not t.is_contiguous():
        raise InvalidArgument(f"{op}: {name} must be {n} consecutive float32 on the weights' device")
    return t.data_ptr()


def _open(op: str, *matrices) -> int:
    for m in matrices:
        if not m._h:
            raise InvalidArgument(f"{op}: the matrix is closed")
        if m.device != matrices[0].device:
            raise InvalidArgument(f"{op}: the matrices are on different devices")
    return matrices[0].device


def _result(torch, op, x, out, tokens, width, device):
    if out is None:
        return torch.empty(tokens, width, dtype=x.dtype, device=x.device)
    return out


def _stream(torch, stream, device):
    return torch.cuda.current_stream(device).cuda_stream if stream is None else getattr(stream, "cuda_stream", stream)


def w4_matvec(w: W4Matrix, x, *, norm=None, eps: float = 1e-5, bias=None, residual=None, out=None, stream=None):
    """y = xn W^T + bias + residual for x [tokens, n_in]; xn is x, or its RMSNorm with the weights `norm`. `out` (any of the three
    element types, may be `residual`) or a new tensor of x's type is returned; a residual has the result's type."""
    torch = _torch()
    device = _open("w4_matvec", w)
    n_in, n_out = w.n_in, w.n_out
    px, tx, ldx = _rows("w4_matvec", "x", x, n_in, device)
    tokens = x.shape[0]
    y = _result(torch, "w4_matvec", x, out, tokens, n_out, device)
    py, ty, ldy = _rows("w4_matvec", "out", y, n_out, device, tokens)
    pr, ldr = None, 0
    if residual is not None:
        pr, tr, ldr = _rows("w4_matvec", "residual", residual, n_out, device, tokens)
        if tr != ty:
            raise InvalidArgument("w4_matvec: residual must have the result's element type")
    if tokens:
        _check(w._lib.retro_b200_w4_matvec(w._h, px, tx, ldx, tokens, _vector("w4_matvec", "norm", norm, n_in, device), eps,
                                           _vector("w4_matvec", "bias", bias, n_out, device), pr, ldr, py, ty, ldy, _stream(torch, stream, device)))
    return y


def w4_glu(gate: W4Matrix, up: W4Matrix, x, *, norm=None, eps: float = 1e-5, out=None, stream=None):
    """y = silu(xn Wgate^T) * (xn Wup^T) for x [tokens, n_in]: the first half of a gated FFN."""
    torch = _torch()
    device = _open("w4_glu", gate, up)
    px, tx, ldx = _rows("w4_glu", "x", x, gate.n_in, device)
    tokens = x.shape[0]
    y = _result(torch, "w4_glu", x, out, tokens, gate.n_out, device)
    py, ty, ldy = _rows("w4_glu", "out", y, gate.n_out, device, tokens)
    if tokens:
        _check(gate._lib.retro_b200_w4_glu(gate._h, up._h, px, tx, ldx, tokens, _vector("w4_glu", "norm", norm, gate.n_in, device), eps, py, ty, ldy,
                                           _stream(torch, stream, device)))
    return y
