"""Host side of the root-mean-square norm with the residual's addition (include/metalllm_attn.h): ctypes
bindings of rmsnormForward, rmsnormForwardFp8 and rmsnormBackward. (The reference's block has a layernorm and a
residual addition of their own, /root/reference/layernorm.metal:10-127, elementwise.metal:7-17.)

Tensors are contiguous: activations torch.bfloat16 [..., cols], gamma torch.bfloat16 [cols], rstd
torch.float32 [rows], dgamma torch.float32 [cols], 8-bit outputs torch.float8_e4m3fn with scales
torch.float32 [rows, ceil(cols/group)]. No CPU fallback.
"""
from __future__ import annotations

import ctypes

from .attention import _check, _lib
from .window import on_device, raw_stream, torch_

MAX_COLS = 8192  # METALLLM_RMSNORM_MAX_COLS


class RmsnormParams(ctypes.Structure):
    """metalllmRmsnormParams."""
    _fields_ = [("rows", ctypes.c_uint32), ("cols", ctypes.c_uint32), ("eps", ctypes.c_float), ("group", ctypes.c_uint32)]

    @classmethod
    def of(cls, rows: int, cols: int, eps: float = 1e-5, group: int = 0) -> "RmsnormParams":
        if not 0 <= rows < 1 << 32 or not 0 <= cols < 1 << 32 or not 0 <= group < 1 << 32:
            raise ValueError("rows, cols and group are unsigned 32-bit numbers")
        return cls(rows, cols, eps, group)


_BOUND = False


def _L():
    global _BOUND
    L = _lib()
    if not _BOUND:
        vp, u64, pp = ctypes.c_void_p, ctypes.c_uint64, ctypes.POINTER(RmsnormParams)
        L.rmsnormForward.argtypes = [vp] * 6 + [pp, vp]
        L.rmsnormForwardFp8.argtypes = [vp] * 7 + [pp, vp]
        L.rmsnormBackward.argtypes = [vp] * 8 + [u64, pp, vp]
        L.metalllmRmsnormBackwardWorkspaceSize.argtypes = [pp, ctypes.POINTER(u64)]
        for f in (L.rmsnormForward, L.rmsnormForwardFp8, L.rmsnormBackward, L.metalllmRmsnormBackwardWorkspaceSize):
            f.restype = ctypes.c_int
        _BOUND = True
    return L


def _shape(t):
    cols = t.shape[-1]
    return (t.numel() // cols if cols else 0), cols


def _are(dtype, count, *tensors):
    """The addresses of contiguous tensors (or None) of `count` values."""
    at = []
    for t in tensors:
        if t is None:
            at.append(None)
            continue
        if t.dtype is not dtype or t.numel() != count:
            raise ValueError(f"tensor must hold {count} values of {dtype}")
        if not t.is_contiguous():
            raise ValueError("tensor must be contiguous")
        at.append(t.data_ptr())
    return at


def rmsnormForward(x, residual, sum, out, gamma, rstd=None, eps: float = 1e-5, stream=None):
    """h = x + residual, sum = bf16(h), rstd = 1/sqrt(mean(h^2) + eps), out = bf16(h rstd gamma). residual,
    sum and rstd may be None (a residual needs sum)."""
    rows, cols = _shape(x)
    here, T = on_device(x, residual, sum, out, gamma, rstd), torch_()
    _check(_L().rmsnormForward(*_are(T.bfloat16, rows * cols, x, residual, sum, out), *_are(T.bfloat16, cols, gamma),
                               *_are(T.float32, rows, rstd), ctypes.byref(RmsnormParams.of(rows, cols, eps)),
                               raw_stream(stream, here)), "rmsnormForward")


def rmsnormForwardFp8(x, residual, sum, out, scales, gamma, rstd=None, eps: float = 1e-5, group: int = 128, stream=None):
    """rmsnormForward with out = e4m3(h rstd gamma / scale), one scale per `group` columns of a row (0: per row)."""
    rows, cols = _shape(x)
    here, T = on_device(x, residual, sum, out, scales, gamma, rstd), torch_()
    _check(_L().rmsnormForwardFp8(*_are(T.bfloat16, rows * cols, x, residual, sum), *_are(T.float8_e4m3fn, rows * cols, out),
                                  *_are(T.float32, rows * (-(-cols // group) if group > 0 else 1), scales),
                                  *_are(T.bfloat16, cols, gamma), *_are(T.float32, rows, rstd),
                                  ctypes.byref(RmsnormParams.of(rows, cols, eps, group)), raw_stream(stream, here)),
           "rmsnormForwardFp8")


def backward_workspace_bytes(rows: int, cols: int) -> int:
    """Device workspace of rmsnormBackward."""
    n = ctypes.c_uint64()
    _check(_L().metalllmRmsnormBackwardWorkspaceSize(ctypes.byref(RmsnormParams.of(rows, cols)), ctypes.byref(n)),
           "metalllmRmsnormBackwardWorkspaceSize")
    return n.value


def rmsnormBackward(dOut, dSum, h, gamma, rstd, dX, dgamma, workspace, stream=None):
    """dX = dSum + gradient through the norm (the gradient of x and of residual), dgamma written. h is the
    forward's sum; dSum (the residual stream's gradient) may be None; workspace: a tensor of
    backward_workspace_bytes(rows, cols) bytes."""
    rows, cols = _shape(h)
    here, T = on_device(dOut, dSum, h, gamma, rstd, dX, dgamma, workspace), torch_()
    at = None
    if workspace is not None:
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        at = workspace.data_ptr()
    n = 0 if workspace is None else workspace.numel() * workspace.element_size()
    dy, ds, hp, dx = _are(T.bfloat16, rows * cols, dOut, dSum, h, dX)
    _check(_L().rmsnormBackward(dy, ds, hp, *_are(T.bfloat16, cols, gamma), *_are(T.float32, rows, rstd), dx,
                                *_are(T.float32, cols, dgamma), at, n, ctypes.byref(RmsnormParams.of(rows, cols)),
                                raw_stream(stream, here)), "rmsnormBackward")
