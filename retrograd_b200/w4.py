"""Products with 4-bit weights for few tokens (`retro_b200_w4_*` in include/retro_b200.h) on torch CUDA tensors.

The tensors' memory goes to the library as it is: rows may be strided, calls run on the current stream of the tensors' device
(or the one given, as a torch stream or its handle) and can be captured into a CUDA graph. A call on a given stream does not order it behind
the current one: the caller does, before the call for its operands and behind it for the result. Operands may be dropped
at once, their memory is not handed out again before the call is done. There is no backward pass: where gradients are recorded, an
operand that requires one is refused.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _ffi
from .engine import EngineError, InvalidArgument, _check, _last_error

_TYPES: dict = {}       # torch dtype -> GGML type code
_raw_stream = None      # current stream handle of a device
_recording = None       # whether gradients are recorded
_bump = None            # counts a tensor's version up


def _torch():
    import torch

    global _raw_stream, _recording, _bump
    if not _TYPES:
        _recording, _bump = torch.is_grad_enabled, torch.autograd.graph.increment_version
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)
        _TYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 30})      # last: another thread takes a filled table for all of it
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
                if hasattr(rows, "is_cuda") and rows.is_cuda and rows.device.index != device:     # (the call waits for its own device)
                    torch.cuda.synchronize(rows.device)
                h = lib.retro_b200_w4_new(ggml_type, pointer, n_out, n_in, n_expert)
        if not h:
            raise InvalidArgument(_last_error()) if _last_error().startswith("w4_new: ") else EngineError(_last_error())
        self._h = h
        nbytes, where = C.c_uint64(), C.c_int()
        _check(lib.retro_b200_w4_info(h, None, None, C.byref(nbytes), C.byref(where)))
        self.ggml_type, self.n_out, self.n_in, self.n_expert = ggml_type, n_out, n_in, n_expert
        self.nbytes, self.device = nbytes.value, where.value
        self._workspace: dict = {}      # bytes of w4_moe's workspace by (tokens of a pass, experts per token)

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


def _no_backward(op: str, name: str) -> None:
    if _recording():
        raise InvalidArgument(f"{op}: {name} requires a gradient, but there is no backward pass: call it under torch.no_grad()")


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
    if t.requires_grad:
        _no_backward(op, name)
    return t.data_ptr(), code, ld


def _vector(op: str, name: str, t, n: int, device: int):
    if t is None:
        return None
    if _TYPES.get(t.dtype) != 0 or t.numel() != n or t.get_device() != device or not t.is_contiguous():
        raise InvalidArgument(f"{op}: {name} must be {n} consecutive float32 on the weights' device")
    if t.requires_grad:
        _no_backward(op, name)
    return t.data_ptr()


def _open(op: str, *matrices) -> int:
    for m in matrices:
        if not m._h:
            raise InvalidArgument(f"{op}: the matrix is closed")
        if m.device != matrices[0].device:
            raise InvalidArgument(f"{op}: the matrices are on different devices")
    return matrices[0].device


def _other(stream, device: int):
    """The stream a call is given, as torch's object, when it is not the current one."""
    if stream is None or getattr(stream, "cuda_stream", stream) == _raw_stream(device):
        return None
    return stream if hasattr(stream, "cuda_stream") else _torch().cuda.ExternalStream(stream, device=device)


def _new(make, stream, device: int):
    """The tensor that make() makes, on the stream the call runs on: the allocator hands its memory to no other stream before."""
    other = _other(stream, device)
    if other is None:
        return make()
    with _torch().cuda.stream(other):
        return make()


def _written(*tensors) -> None:
    """Tells autograd that a call wrote these: a backward pass that has saved one refuses it, as after torch's own in-place operations."""
    for t in tensors:
        if t is not None and not t.is_inference():
            _bump(t)


def _used(stream, device: int, *tensors) -> None:
    """Tells the allocator that a call used these on `stream`: it hands their memory out again only behind that."""
    other = _other(stream, device)
    if other is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(other)


def _result(op: str, x, tx: int, out, tokens: int, width: int, device: int, stream):
    """The result tensor (a new one of x's type unless `out` is given), its pointer, type code and row stride."""
    if out is None:
        y = x.new_empty(tokens, width) if stream is None else _new(lambda: x.new_empty(tokens, width), stream, device)
        return y, y.data_ptr(), tx, width
    return (out, *_rows(op, "out", out, width, device, tokens))


def _residual(op: str, residual, code: int, width: int, device: int, tokens: int):
    if residual is None:
        return None, 0
    pointer, own, ld = _rows(op, "residual", residual, width, device, tokens)
    if own != code:
        raise InvalidArgument(f"{op}: residual must have the result's element type")
    return pointer, ld


def _stream(stream, device: int):
    return _raw_stream(device) if stream is None else getattr(stream, "cuda_stream", stream)


def w4_matvec(w: W4Matrix, x, *, norm=None, eps: float = 1e-5, bias=None, residual=None, out=None, stream=None):
    """y = xn W^T + bias + residual for x [tokens, n_in]; xn is x, or its RMSNorm with the weights `norm`. `out` (any of the three
    element types, may be `residual`) or a new tensor of x's type is returned; a residual has the result's type."""
    _TYPES or _torch()
    device = w.device
    if not w._h:
        _open("w4_matvec", w)
    px, tx, ldx = _rows("w4_matvec", "x", x, w.n_in, device)
    tokens = x.shape[0]
    y, py, ty, ldy = _result("w4_matvec", x, tx, out, tokens, w.n_out, device, stream)
    pr, ldr = (None, 0) if residual is None else _residual("w4_matvec", residual, ty, w.n_out, device, tokens)
    if tokens:
        status = w._lib.retro_b200_w4_matvec(w._h, px, tx, ldx, tokens, None if norm is None else _vector("w4_matvec", "norm", norm, w.n_in, device), eps,
                                             None if bias is None else _vector("w4_matvec", "bias", bias, w.n_out, device), pr, ldr, py, ty, ldy, _stream(stream, device))
        if status:
            _check(status)
        if out is not None:
            _written(out)
        if stream is not None:
            _used(stream, device, x, norm, bias, residual, out)
    return y


def w4_glu(gate: W4Matrix, up: W4Matrix, x, *, norm=None, eps: float = 1e-5, out=None, stream=None):
    """y = silu(xn Wgate^T) * (xn Wup^T) for x [tokens, n_in]: the first half of a gated FFN."""
    _TYPES or _torch()
    device = _open("w4_glu", gate, up)
    px, tx, ldx = _rows("w4_glu", "x", x, gate.n_in, device)
    tokens = x.shape[0]
    y, py, ty, ldy = _result("w4_glu", x, tx, out, tokens, gate.n_out, device, stream)
    if tokens:
        status = gate._lib.retro_b200_w4_glu(gate._h, up._h, px, tx, ldx, tokens, _vector("w4_glu", "norm", norm, gate.n_in, device), eps, py, ty, ldy,
                                             _stream(stream, device))
        if status:
            _check(status)
        if out is not None:
            _written(out)
        if stream is not None:
            _used(stream, device, x, norm, out)
    return y


def w4_moe(router, gate: W4Matrix, up: W4Matrix, down: W4Matrix, x, n_used: int, *, normalise: bool = False, norm=None, eps: float = 1e-5,
           residual=None, out=None, ids=None, weights=None, workspace=None, stream=None):
    """A mixture-of-experts layer for x [tokens, n_in]: y = residual + sum over the n_used likeliest experts of their probability times
    down(silu(gate xn) * (up xn)). `ids` (int32) and `weights` (float32), [tokens, n_used], receive the routing. `workspace` is a
    CUDA byte tensor of at least `w4_moe_workspace(gate, tokens, n_used)` bytes that no other pending call uses; by default one is
    allocated for the call."""
    torch = _torch()
    device = _open("w4_moe", gate, up, down)
    n_in = gate.n_in
    px, tx, ldx = _rows("w4_moe", "x", x, n_in, device)
    tokens = x.shape[0]
    y, py, ty, ldy = _result("w4_moe", x, tx, out, tokens, n_in, device, stream)
    pr, ldr = _residual("w4_moe", residual, ty, n_in, device, tokens)
    if not 1 <= n_used <= min(gate.n_expert, 32):
        raise InvalidArgument("w4_moe: n_used must be 1 to n_expert, at most 32")
    for name, t, dtype in (("ids", ids, torch.int32), ("weights", weights, torch.float32)):
        if t is not None and (t.dtype != dtype or tuple(t.shape) != (tokens, n_used) or t.get_device() != device or not t.is_contiguous()):
            raise InvalidArgument(f"w4_moe: {name} must be contiguous {dtype} [{tokens}, {n_used}] on the weights' device")
        if t is not None and t.requires_grad:
            _no_backward("w4_moe", name)
    if not tokens:
        return y
    on, given = _stream(stream, device), workspace
    if workspace is None:
        need = w4_moe_workspace(gate, tokens, n_used)
        workspace = _new(lambda: torch.empty(need, dtype=torch.uint8, device=x.device), stream, device)
    elif workspace.get_device() != device or not workspace.is_contiguous():
        raise InvalidArgument("w4_moe: the workspace must be contiguous on the weights' device")
    _check(gate._lib.retro_b200_w4_moe(_vector("w4_moe", "router", router, gate.n_expert * n_in, device), gate._h, up._h, down._h, px, tx, ldx, tokens, n_used,
                                       normalise, _vector("w4_moe", "norm", norm, n_in, device), eps, pr, ldr, py, ty, ldy,
                                       None if ids is None else ids.data_ptr(), None if weights is None else weights.data_ptr(),
                                       workspace.data_ptr(), workspace.numel() * workspace.element_size(), on))
    _written(out, ids, weights)
    if stream is not None:
        _used(stream, device, router, x, norm, residual, out, ids, weights, given)
    return y


def w4_moe_workspace(gate: W4Matrix, tokens: int, n_used: int) -> int:
    """Bytes of workspace a `w4_moe` call of `tokens` tokens needs."""
    key = min(tokens, 16), n_used
    known = gate._workspace.get(key)
    if known is None:
        _open("w4_moe_workspace", gate)
        n = C.c_size_t()
        _check(gate._lib.retro_b200_w4_moe_workspace(gate._h, key[0], n_used, C.byref(n)))
        known = gate._workspace[key] = n.value
    return known
