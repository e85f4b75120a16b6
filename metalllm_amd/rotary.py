"""Host side of the rotary positions (include/metalllm_attn.h): ctypes bindings of rotaryForward and
rotaryBackward, which turn q and k between computeQKV and the attention. (The reference has learned
positions at the embedding instead, /root/reference/embed.metal:1-34.)

Tensors: q torch.bfloat16 [B, T, NH, D], k torch.bfloat16 [B, T, NKV, D] (or None), heads beside each
other in a row; positions torch.int32 [B, T], contiguous, or None. No CPU fallback.
"""
from __future__ import annotations

import ctypes

from .attention import _check, _lib
from .window import on_device, raw_stream, row_seq, torch_

PAIRS = 128  # METALLLM_ROTARY_PAIRS
SCALING = {"none": 0, "linear": 1, "parts": 2}


class RotaryScaling(ctypes.Structure):
    """metalllmRotaryScaling."""
    _fields_ = [("kind", ctypes.c_int32), ("magnitude", ctypes.c_float), ("factor", ctypes.c_double),
                ("original", ctypes.c_double), ("low", ctypes.c_double), ("high", ctypes.c_double)]


class RotaryPlan(ctypes.Structure):
    """metalllmRotaryPlan: the frequencies of a head's pairs, in host memory."""
    _fields_ = [("turns", ctypes.c_double * PAIRS), ("magnitude", ctypes.c_float), ("dims", ctypes.c_uint32),
                ("interleaved", ctypes.c_uint32), ("reserved", ctypes.c_uint32)]

    @classmethod
    def of(cls, dims: int, base: float = 10000.0, interleaved: bool = False, scaling: str = "none", factor: float = 1.0,
           original: float = 1.0, low: float = 1.0, high: float = 32.0, magnitude: float = 1.0) -> "RotaryPlan":
        if scaling not in SCALING:
            raise ValueError(f"scaling is one of {', '.join(SCALING)}")
        if not 0 <= dims < 1 << 32:
            raise ValueError("dims is an unsigned number")
        plan, s = cls(), RotaryScaling(SCALING[scaling], magnitude, factor, original, low, high)
        _check(_L().metalllmRotaryPlanInit(dims, base, int(interleaved), ctypes.byref(s), ctypes.byref(plan)),
               "metalllmRotaryPlanInit")
        return plan


class RotaryParams(ctypes.Structure):
    """metalllmRotaryParams."""
    _fields_ = [(n, ctypes.c_uint32) for n in ("B", "T", "NH", "NKV", "D", "reserved")] + \
               [(n, ctypes.c_uint64) for n in ("q_row", "q_seq", "k_row", "k_seq", "qo_row", "qo_seq", "ko_row", "ko_seq")]


_BOUND = False


def _L():
    global _BOUND
    L = _lib()
    if not _BOUND:
        vp = ctypes.c_void_p
        L.metalllmRotaryPlanInit.argtypes = [ctypes.c_uint32, ctypes.c_double, ctypes.c_int,
                                             ctypes.POINTER(RotaryScaling), ctypes.POINTER(RotaryPlan)]
        for f in (L.rotaryForward, L.rotaryBackward):
            f.argtypes = [vp] * 5 + [ctypes.POINTER(RotaryPlan), ctypes.POINTER(RotaryParams), vp]
        for f in (L.metalllmRotaryPlanInit, L.rotaryForward, L.rotaryBackward):
            f.restype = ctypes.c_int
        _BOUND = True
    return L


def _rotary(name, q, k, q_out, k_out, positions, plan, stream):
    if (k is None) != (k_out is None):
        raise ValueError("k and k_out go together")
    here = on_device(q, k, q_out, k_out, positions)
    bf16, shape = torch_().bfloat16, q.shape
    if q.dtype is not bf16 or q_out.dtype is not bf16 or (k is not None and (k.dtype is not bf16 or k_out.dtype is not bf16)):
        raise ValueError("tensors must be bfloat16")
    if len(shape) != 4 or q_out.shape != shape:
        raise ValueError("q, q_out: [B, T, NH, D]")
    B, T, NH, D = shape
    NKV, kp, kop, kr, kor = 0, None, None, (0, 0), (0, 0)
    if k is not None:
        if k_out.shape != k.shape or len(k.shape) != 4 or k.shape[:2] != shape[:2] or k.shape[3] != D:
            raise ValueError("k, k_out: [B, T, NKV, D]")
        NKV, kp, kop, kr, kor = k.shape[2], k.data_ptr(), k_out.data_ptr(), row_seq(k), row_seq(k_out)
    at = None
    if positions is not None:
        if positions.dtype is not torch_().int32 or positions.shape != shape[:2] or not positions.is_contiguous():
            raise ValueError("positions must be int32 [B, T], contiguous")
        at = positions.data_ptr()
    if max(B, T, NH, NKV, D) >= 1 << 32:
        raise ValueError("sizes are unsigned 32-bit numbers")
    p = RotaryParams(B, T, NH, NKV, D, 0, *row_seq(q), *kr, *row_seq(q_out), *kor)
    _check(getattr(_L(), name)(q.data_ptr(), kp, q_out.data_ptr(), kop, at, ctypes.byref(plan), ctypes.byref(p),
                               raw_stream(stream, here)), name)


def rotaryForward(q, k, q_out, k_out, positions, plan: RotaryPlan, stream=None):
    """q_out, k_out = q, k turned to their positions (None: token t at t). In place: q_out is q."""
    _rotary("rotaryForward", q, k, q_out, k_out, positions, plan, stream)


def rotaryBackward(dq, dk, dq_out, dk_out, positions, plan: RotaryPlan, stream=None):
    """The gradient: dq_out, dk_out = gradients at q and k from those at the turned ones."""
    _rotary("rotaryBackward", dq, dk, dq_out, dk_out, positions, plan, stream)
