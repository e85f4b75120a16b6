"""The window attention's refusals, sizes and host-side checks: no GPU."""
import ctypes

import pytest

import metalllm_amd as M
import metalllm_amd.window as W

AT = lambda i: ctypes.c_void_p((1 << 40) + (i << 34))  # never dereferenced


def params(**change):
    f = dict(B=2, TQ=100, TK=130, NH=4, NKV=2, D=64, window=50, sinks=4, q_row=256, q_seq=25600, k_row=128, k_seq=16640,
             v_row=128, v_seq=16640, o_row=256, o_seq=25600)
    f.update(change)
    return W.WindowParams(**f)


def forward(p, at=None, n=1 << 40, **change):
    a = {m: AT(i) for i, m in enumerate(("q", "k", "v", "out", "l", "q_len", "k_len", "workspace"))}
    a.update(change)
    return W._L().windowAttentionForward(*a.values(), n, p and ctypes.byref(p), None)


def backward(p, n=1 << 33, **change):
    a = {m: AT(i) for i, m in enumerate(("dO", "O", "l", "q", "k", "v", "dQ", "dK", "dV", "q_len", "k_len", "workspace"))}
    a.update(change)
    return W._L().windowAttentionBackward(*a.values(), n, p and ctypes.byref(p), None)


@pytest.mark.parametrize("change,code", [
    (dict(D=32), -3), (dict(D=96), -3), (dict(TQ=0), -4), (dict(TK=0), -4), (dict(B=0), -4), (dict(NH=0), -4), (dict(NKV=0), -4),
    (dict(NKV=3), -4), (dict(window=0), -10), (dict(sinks=65), -10), (dict(TQ=(1 << 24) + 1), -5), (dict(TK=(1 << 24) + 1), -5),
    (dict(B=1 << 20, NH=64, NKV=64), -5), (dict(B=1 << 12, NH=16, TQ=1 << 22), -5), (dict(q_row=255), -4), (dict(q_row=260), -4),
    (dict(q_row=248), -4), (dict(k_row=120), -4), (dict(v_row=1 << 22, v_seq=1 << 40), -4), (dict(o_seq=25592), -4),
    (dict(q_seq=25604), -4), (dict(k_seq=1 << 48), -4), (dict(k_seq=64), -4), (dict(k_seq=0), -4),
])
def test_bad_params(change, code):
    p, n = params(**change), ctypes.c_uint64()
    assert forward(p) == code and backward(p) == code
    assert W._L().metalllmWindowForwardWorkspaceSize(ctypes.byref(p), ctypes.byref(n)) == code
    assert W._L().metalllmWindowBackwardWorkspaceSize(ctypes.byref(p), ctypes.byref(n)) == code


def test_null_and_alignment():
    p = params()
    assert forward(None) == -1 and backward(None) == -1
    for n in ("q", "k", "v", "out"):
        assert forward(p, **{n: None}) == -1
    for n in ("q", "k", "v", "out", "l"):
        assert forward(p, **{n: ctypes.c_void_p((1 << 50) + 8)}) == -6
    for n in ("q_len", "k_len"):
        assert forward(p, **{n: ctypes.c_void_p((1 << 50) + 2)}) == -6
        assert backward(p, **{n: ctypes.c_void_p((1 << 50) + 2)}) == -6
    for n in ("dO", "O", "l", "q", "k", "v", "dQ", "dK", "dV", "workspace"):
        assert backward(p, **{n: None}) == -1
        assert backward(p, **{n: ctypes.c_void_p((1 << 50) + 8)}) == -6
    assert W._L().metalllmWindowForwardWorkspaceSize(ctypes.byref(p), None) == -1
    assert W._L().metalllmWindowBackwardWorkspaceSize(ctypes.byref(p), None) == -1


def test_workspace():
    rows, token = params(), params(TQ=1, TK=9000, window=8000, q_seq=256, o_seq=256, k_seq=9000 * 128, v_seq=9000 * 128)
    assert W.forward_workspace_bytes(rows) == 0
    n = W.forward_workspace_bytes(token)
    assert n > 0 and n % 4 == 0
    assert forward(token, workspace=None) == -1
    assert forward(token, workspace=ctypes.c_void_p((1 << 50) + 4)) == -6
    assert forward(token, n=n - 1) == -5
    # two numbers for every row and head, and the sinks' parts where rows lie beyond block 0's windows
    assert W.backward_workspace_bytes(params(TK=100, sinks=0)) == 4 * 2 * 2 * 4 * 100
    assert W.backward_workspace_bytes(params(sinks=0)) == 4 * 2 * 2 * 4 * 100
    big = params(TK=1000, TQ=1000, q_seq=256000, o_seq=256000, k_seq=128000, v_seq=128000)
    n = W.backward_workspace_bytes(big)
    assert n > 4 * 2 * 2 * 4 * 1000
    assert backward(big, n=n - 1) == -5


def test_shared_memory():
    p = params()
    e = 2 * 25600 * 2  # bytes of q
    inside = lambda i, more: ctypes.c_void_p(AT(i).value + more)
    assert forward(p, out=AT(0)) == -11 and forward(p, out=inside(0, e - 16)) == -11
    assert forward(p, out=inside(1, 2 * (16640 + 129 * 128))) == -11  # k's last row
    assert forward(p, l=AT(3)) == -11 and forward(p, l=AT(2)) == -11 and forward(p, l=AT(5)) == -11
    for out in ("dQ", "dK", "dV"):
        for i in range(6):
            assert backward(p, **{out: AT(i)}) == -11
    assert backward(p, dK=AT(6)) == -11 and backward(p, dV=AT(7)) == -11
    for i in range(9):
        assert backward(p, workspace=AT(i)) == -11
    token = params(TQ=1, TK=9000, window=8000, q_seq=256, o_seq=256, k_seq=9000 * 128, v_seq=9000 * 128)
    for i in range(5):
        assert forward(token, workspace=AT(i)) == -11


def test_python_checks():
    import torch
    q, k = torch.zeros(2, 100, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 130, 2, 64, dtype=torch.bfloat16)
    p = W.WindowParams.of(q, k, k, q, 50, 4)
    assert [getattr(p, n) for n, _ in p._fields_] == [getattr(params(), n) for n, _ in p._fields_]
    assert W.WindowParams.of(q, k, k, q).window == W.FULL
    for bad in ((q[0], k, k, q), (q, k, k[:, 1:], q), (q, k, k, q[:, 1:]), (q, k[:1], k[:1], q), (q[..., :32], k, k, q[..., :32])):
        with pytest.raises(ValueError):
            W.WindowParams.of(*bad, 50, 4)
    for window, sinks in ((-1, 0), (1 << 32, 0), (5, -1)):
        with pytest.raises(ValueError):
            W.WindowParams.of(q, k, k, q, window, sinks)
    # a head's values, or the heads of a row, that do not lie beside each other
    for t in (torch.zeros(2, 100, 64, 4, dtype=torch.bfloat16).transpose(2, 3), torch.zeros(2, 4, 100, 64).transpose(1, 2)):
        with pytest.raises(ValueError):
            W.row_seq(t)
    # strides of dimensions of one are no strides
    assert W.row_seq(torch.zeros(1, 9, 4, 64)[:, 4:5]) == (256, 256)
    assert W.row_seq(torch.zeros(3, 9, 4, 64)[:, 4:5]) == (256, 9 * 256)
    with pytest.raises(ValueError, match="GPU"):
        W.windowAttentionForward(q, k, k.clone(), q.clone(), None, params=p)


def test_error_strings():
    for code in (-10, -11):
        assert b"unknown" not in M.library().metalllmAttnErrorString(code)
        assert str(M.AttentionError(code, "x")).startswith("x: E_")
