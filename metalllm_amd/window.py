"""Host side of the window attention (include/metalllm_attn.h): ctypes bindings of
windowAttentionForward and windowAttentionBackward. The reference's attention is causal over every key
(/root/reference/attention.metal:56-299); here a query row at position pos sees key j where j <= pos and
(pos - j < window or j < sinks), with any number of rows, fewer key heads than query heads, sequence
lengths on the device, and strided tensors.

Tensors: q, out, dO, O, dQ are torch.bfloat16 [B, TQ, NH, D]; k, v, dK, dV are torch.bfloat16
[B, TK, NKV, D]; l is torch.float32 [B, NH, TQ], contiguous; lengths are torch.int32 [B]. Heads lie beside
each other in a row, rows and sequences at any stride that is a multiple of 8. No CPU fallback.
"""
from __future__ import annotations

import ctypes

from .attention import _check, _lib

FULL = (1 << 32) - 1  # a window that holds every key


class WindowParams(ctypes.Structure):
    """metalllmWindowParams."""
    _fields_ = [(n, ctypes.c_uint32) for n in ("B", "TQ", "TK", "NH", "NKV", "D", "window", "sinks")] + \
               [(n, ctypes.c_uint64) for n in ("q_row", "q_seq", "k_row", "k_seq", "v_row", "v_seq", "o_row", "o_seq")]

    @classmethod
    def of(cls, q, k, v, out, window: int | None = None, sinks: int = 0) -> "WindowParams":
        """From the tensors of a forward call (window None: every key). Buffers that keep their shapes and
        strides can keep the params."""
        if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or out.shape != q.shape:
            raise ValueError("q, out: [B, TQ, NH, D]; k, v: [B, TK, NKV, D]")
        B, TQ, NH, D = q.shape
        TK, NKV = k.shape[1], k.shape[2]
        if max(B, TQ, TK, NH, NKV, D) > FULL:
            raise ValueError("sizes are unsigned 32-bit numbers")
        if k.shape[0] != B or k.shape[3] != D:
            raise ValueError("q and k disagree about B or D")
        window = FULL if window is None else window
        if not 0 <= window <= FULL or not 0 <= sinks <= FULL:
            raise ValueError("window and sinks are unsigned 32-bit numbers")
        return cls(B, TQ, TK, NH, NKV, D, window, sinks, *row_seq(q), *row_seq(k), *row_seq(v), *row_seq(out))


def row_seq(t):
    """Elements from a token to the next and from a sequence to the next of a [B, T, heads, D] tensor."""
    B, T, H, D = t.shape
    if t.is_contiguous():
        return H * D, T * H * D
    s, r, h, e = t.stride()
    if (e != 1 and D > 1) or (h != D and H > 1):
        raise ValueError("a row's heads must lie beside each other (strides ..., D, 1)")
    if T == 1:
        r = H * D  # no second row: any stride stands
        if B > 1 and s < r:
            raise ValueError("sequences overlap")
    return r, (s if B > 1 else T * r)


_BOUND = False


def _L():
    global _BOUND
    L = _lib()
    if not _BOUND:
        vp, u64, pp = ctypes.c_void_p, ctypes.c_uint64, ctypes.POINTER(WindowParams)
        L.windowAttentionForward.argtypes = [vp] * 8 + [u64, pp, vp]
        L.windowAttentionBackward.argtypes = [vp] * 12 + [u64, pp, vp]
        for f in (L.metalllmWindowForwardWorkspaceSize, L.metalllmWindowBackwardWorkspaceSize):
            f.argtypes = [pp, ctypes.POINTER(u64)]
        for f in (L.windowAttentionForward, L.windowAttentionBackward, L.metalllmWindowForwardWorkspaceSize,
                  L.metalllmWindowBackwardWorkspaceSize):
            f.restype = ctypes.c_int
        _BOUND = True
    return L


def forward_workspace_bytes(p: WindowParams) -> int:
    """Device workspace of windowAttentionForward (0 for all but a few query rows over many keys)."""
    n = ctypes.c_uint64()
    _check(_L().metalllmWindowForwardWorkspaceSize(ctypes.byref(p), ctypes.byref(n)), "metalllmWindowForwardWorkspaceSize")
    return n.value


def backward_workspace_bytes(p: WindowParams) -> int:
    """Device workspace of windowAttentionBackward."""
    n = ctypes.c_uint64()
    _check(_L().metalllmWindowBackwardWorkspaceSize(ctypes.byref(p), ctypes.byref(n)), "metalllmWindowBackwardWorkspaceSize")
    return n.value


_T = None  # torch, and its current device and raw current stream, from the first call on


def torch_():
    global _T, _device, _raw_stream
    if _T is None:
        import torch
        torch.cuda.init()
        _T, _device, _raw_stream = torch, torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    return _T


def on_device(*tensors):
    """The current GPU, which the call launches on; raises unless every tensor (or None) lives there."""
    at = {t.get_device() for t in tensors if t is not None}
    if -1 in at:
        raise ValueError("tensor must live on the GPU")
    torch_()
    here = _device()
    if at != {here}:
        raise ValueError("tensor must live on the current GPU")
    return here


def raw_stream(stream, here: int):
    """The handle of `stream`, which has to be of the GPU `here`; None: its current stream."""
    if stream is None:
        return _raw_stream(here)
    if getattr(stream, "device_index", here) != here:
        raise ValueError("stream must be of the current GPU")
    return stream.cuda_stream


def _bf16(shape, row, seq, *tensors):
    for t in tensors:
        if t.dtype is not _T.bfloat16:
            raise ValueError("tensor must be bfloat16")
        if t.shape != shape or row_seq(t) != (row, seq):
            raise ValueError(f"tensor must have shape {shape}, its rows {row} and its sequences {seq} elements apart")


def _logsumexp(p, l):
    if l is not None and (l.dtype is not _T.float32 or l.shape != (p.B, p.NH, p.TQ) or not l.is_contiguous()):
        raise ValueError("l must be float32 [B, NH, TQ], contiguous")


def _lengths(p, *lengths):
    for t in lengths:
        if t is not None and (t.dtype is not _T.int32 or t.shape != (p.B,) or not t.is_contiguous()):
            raise ValueError("lengths must be int32 [B], contiguous")


def _address(t):
    return None if t is None else t.data_ptr()


def _room(workspace):
    if workspace is None:
        return None, 0
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def windowAttentionForward(q, k, v, out, l=None, q_len=None, k_len=None, workspace=None, stream=None,
                           params: WindowParams | None = None, window: int | None = None, sinks: int = 0):
    """out = attention of q over the visible keys, l = logsumexp (None: not kept). params (or window and
    sinks), lengths and workspace (a tensor of forward_workspace_bytes bytes; None where that is 0) as in
    include/metalllm_attn.h."""
    p = params or WindowParams.of(q, k, v, out, window, sinks)
    here = on_device(q, k, v, out, l, q_len, k_len, workspace)
    B, D = p.B, p.D
    rows, keys = (B, p.TQ, p.NH, D), (B, p.TK, p.NKV, D)
    _bf16(rows, p.q_row, p.q_seq, q), _bf16(keys, p.k_row, p.k_seq, k)
    _bf16(keys, p.v_row, p.v_seq, v), _bf16(rows, p.o_row, p.o_seq, out)
    _logsumexp(p, l), _lengths(p, q_len, k_len)
    wp, wn = _room(workspace)
    _check(_L().windowAttentionForward(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _address(l),
                                       _address(q_len), _address(k_len), wp, wn, ctypes.byref(p), raw_stream(stream, here)),
           "windowAttentionForward")


def windowAttentionBackward(dO, O, l, q, k, v, dQ, dK, dV, q_len=None, k_len=None, workspace=None, stream=None,
                            params: WindowParams | None = None, window: int | None = None, sinks: int = 0):
    """dQ, dK, dV of windowAttentionForward's out = O, l. dO has O's layout, dQ q's, dK k's and dV v's."""
    p = params or WindowParams.of(q, k, v, O, window, sinks)
    here = on_device(dO, O, l, q, k, v, dQ, dK, dV, q_len, k_len, workspace)
    B, D = p.B, p.D
    rows, keys = (B, p.TQ, p.NH, D), (B, p.TK, p.NKV, D)
    _bf16(rows, p.q_row, p.q_seq, q, dQ), _bf16(keys, p.k_row, p.k_seq, k, dK)
    _bf16(keys, p.v_row, p.v_seq, v, dV), _bf16(rows, p.o_row, p.o_seq, O, dO)
    _logsumexp(p, l), _lengths(p, q_len, k_len)
    wp, wn = _room(workspace)
    _check(_L().windowAttentionBackward(dO.data_ptr(), O.data_ptr(), _address(l), q.data_ptr(), k.data_ptr(),
                                        v.data_ptr(), dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), _address(q_len),
                                        _address(k_len), wp, wn, ctypes.byref(p), raw_stream(stream, here)),
           "windowAttentionBackward")


def window_attention_forward(q, k, v, window: int | None = None, sinks: int = 0, q_len=None, k_len=None, stream=None):
    """Allocating form: returns (out, l). Rows behind a sequence's length hold zeros."""
    import torch
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    l = torch.zeros((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device)
    p = WindowParams.of(q, k, v, out, window, sinks)
    n = forward_workspace_bytes(p)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    _with_stream(stream, out, l, ws)
    windowAttentionForward(q, k, v, out, l, q_len, k_len, ws, stream, p)
    return out, l


def window_attention_backward(dO, q, k, v, out, l, window: int | None = None, sinks: int = 0, q_len=None, k_len=None,
                              stream=None):
    """Allocating form: returns (dQ, dK, dV). Rows behind a sequence's lengths hold zeros."""
    import torch
    dQ, dK, dV = (torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device).zero_() for t in (q, k, v))
    p = WindowParams.of(q, k, v, out, window, sinks)
    ws = torch.empty(backward_workspace_bytes(p), dtype=torch.uint8, device=q.device)
    _with_stream(stream, dQ, dK, dV, ws)
    windowAttentionBackward(dO, out, l, q, k, v, dQ, dK, dV, q_len, k_len, ws, stream, p)
    return dQ, dK, dV


def _with_stream(stream, *tensors):
    """Tensors allocated on the current stream, used on another: that one waits for their zeros, and the
    allocator for it."""
    if stream is None:
        return
    import torch
    stream.wait_stream(torch.cuda.current_stream())
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
