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

from .attention import _check, _lib, _stream

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
        if k.shape[0] != B or k.shape[3] != D:
            raise ValueError("q and k disagree about B or D")
        window = FULL if window is None else window
        if not 0 <= window <= FULL or not 0 <= sinks <= FULL:
            raise ValueError("window and sinks are unsigned 32-bit numbers")
        p = cls(B, TQ, TK, NH, NKV, D, window, sinks, *row_seq(q), *row_seq(k), *row_seq(v), *row_seq(out))
        p.q_is, p.k_is, p.v_is, p.o_is = (_layout(t) for t in (q, k, v, out))
        return p


def _layout(t):
    return t.shape, t.stride()


def row_seq(t):
    """Elements from a token to the next and from a sequence to the next of a [B, T, heads, D] tensor."""
    B, T, H, D = t.shape
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


_CURRENT = None  # torch.cuda.current_device, imported on the first call


def on_device(*tensors):
    """Raises unless every tensor (or None) lives on the current GPU, which the call launches on."""
    global _CURRENT
    if _CURRENT is None:
        import torch
        _CURRENT = torch.cuda.current_device
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("tensor must live on the GPU")
    here = _CURRENT()
    for t in tensors:
        if t is not None and t.get_device() != here:
            raise ValueError("tensor must live on the current GPU")


def _bf16(layout, *tensors):
    import torch
    for t in tensors:
        if t.dtype != torch.bfloat16:
            raise ValueError("tensor must be bfloat16")
        if t.shape != layout[0] or t.stride() != layout[1]:
            raise ValueError(f"tensor must have shape {tuple(layout[0])} and strides {layout[1]}")


def _logsumexp(p, l):
    import torch
    if l is not None and (l.dtype != torch.float32 or l.shape != (p.B, p.NH, p.TQ) or not l.is_contiguous()):
        raise ValueError("l must be float32 [B, NH, TQ], contiguous")


def _lengths(p, *lengths):
    import torch
    for t in lengths:
        if t is not None and (t.dtype != torch.int32 or t.shape != (p.B,) or not t.is_contiguous()):
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
    on_device(q, k, v, out, l, q_len, k_len, workspace)
    _bf16(p.q_is, q), _bf16(p.k_is, k), _bf16(p.v_is, v), _bf16(p.o_is, out)
    _logsumexp(p, l), _lengths(p, q_len, k_len)
    wp, wn = _room(workspace)
    _check(_L().windowAttentionForward(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _address(l),
                                       _address(q_len), _address(k_len), wp, wn, ctypes.byref(p), _stream(stream)),
           "windowAttentionForward")


def windowAttentionBackward(dO, O, l, q, k, v, dQ, dK, dV, q_len=None, k_len=None, workspace=None, stream=None,
                            params: WindowParams | None = None, window: int | None = None, sinks: int = 0):
    """dQ, dK, dV of windowAttentionForward's out = O, l. dO has O's layout, dQ q's, dK k's and dV v's."""
    p = params or WindowParams.of(q, k, v, O, window, sinks)
    on_device(dO, O, l, q, k, v, dQ, dK, dV, q_len, k_len, workspace)
    _bf16(p.q_is, q, dQ), _bf16(p.k_is, k, dK), _bf16(p.v_is, v, dV), _bf16(p.o_is, O, dO)
    _logsumexp(p, l), _lengths(p, q_len, k_len)
    wp, wn = _room(workspace)
    _check(_L().windowAttentionBackward(dO.data_ptr(), O.data_ptr(), _address(l), q.data_ptr(), k.data_ptr(),
                                        v.data_ptr(), dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), _address(q_len),
                                        _address(k_len), wp, wn, ctypes.byref(p), _stream(stream)),
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
