"""Refusals and host arithmetic of the rotary positions and the root-mean-square norm: no GPU."""
import ctypes
import math

import pytest

import metalllm_amd.rmsnorm as N
import metalllm_amd.rotary as R
from metalllm_amd import AttentionError

AT = lambda i: ctypes.c_void_p((1 << 40) + (i << 34))  # never dereferenced


def test_plan():
    p = R.RotaryPlan.of(64, base=500.0, interleaved=True, magnitude=1.5)
    assert (p.dims, p.interleaved, p.magnitude) == (64, 1, 1.5)
    for i in range(32):
        assert math.isclose(p.turns[i], 500.0 ** (-2 * i / 64) / (2 * math.pi), rel_tol=1e-14)
    assert all(p.turns[i] == 0 for i in range(32, 128))
    q = R.RotaryPlan.of(64, base=500.0, scaling="linear", factor=4.0)
    assert all(math.isclose(q.turns[i], p.turns[i] / 4, rel_tol=1e-14) for i in range(32))
    q = R.RotaryPlan.of(64, base=500.0, scaling="parts", factor=4.0, original=100.0, low=1.0, high=8.0)
    for i in range(32):
        keep = min(1.0, max(0.0, (100.0 * p.turns[i] - 1) / 7))
        assert math.isclose(q.turns[i], p.turns[i] * (keep + (1 - keep) / 4), rel_tol=1e-13)
    assert q.turns[0] == p.turns[0] and math.isclose(q.turns[31], p.turns[31] / 4, rel_tol=1e-13)
    nan, inf = float("nan"), float("inf")
    for bad in (dict(dims=0), dict(dims=63), dict(dims=258), dict(dims=64, base=0.0), dict(dims=64, base=-1.0),
                dict(dims=64, base=nan), dict(dims=64, base=inf), dict(dims=64, magnitude=nan),
                dict(dims=64, scaling="linear", factor=0.0), dict(dims=64, scaling="linear", factor=nan),
                dict(dims=64, scaling="parts", factor=2.0, original=0.0), dict(dims=64, scaling="parts", factor=2.0, original=9.0, low=3.0, high=3.0),
                dict(dims=64, scaling="parts", factor=2.0, original=9.0, low=nan)):
        with pytest.raises(AttentionError):
            R.RotaryPlan.of(**bad)
    with pytest.raises(ValueError):
        R.RotaryPlan.of(64, scaling="other")
    with pytest.raises(ValueError):
        R.RotaryPlan.of(-2)
    assert R._L().metalllmRotaryPlanInit(64, 10000.0, 0, None, None) == -1
    assert R._L().metalllmRotaryPlanInit(64, 10000.0, 0, None, ctypes.byref(p)) == 0 and p.magnitude == 1.0
    s = R.RotaryScaling(7, 1.0, 1.0, 1.0, 1.0, 2.0)
    assert R._L().metalllmRotaryPlanInit(64, 10000.0, 0, ctypes.byref(s), ctypes.byref(p)) == -4


def rotary_params(**change):
    f = dict(B=2, T=10, NH=4, NKV=2, D=64, reserved=0, q_row=256, q_seq=2560, k_row=128, k_seq=1280, qo_row=256, qo_seq=2560,
             ko_row=128, ko_seq=1280)
    f.update(change)
    return R.RotaryParams(**f)


@pytest.mark.parametrize("name", ["rotaryForward", "rotaryBackward"])
def test_rotary_refusals(name):
    plan = R.RotaryPlan.of(64)

    def call(p=None, plan=plan, **change):
        a = {m: AT(i) for i, m in enumerate(("q", "k", "qo", "ko", "pos"))}
        a.update(change)
        p = p or rotary_params()
        return getattr(R._L(), name)(*a.values(), plan and ctypes.byref(plan), ctypes.byref(p), None)

    assert call(plan=None) == -1
    assert getattr(R._L(), name)(AT(0), AT(1), AT(2), AT(3), AT(4), ctypes.byref(plan), None, None) == -1
    for n in ("q", "k", "qo", "ko"):
        assert call(**{n: None}) == -1
        assert call(**{n: ctypes.c_void_p((1 << 50) + 2)}) == -6
    assert call(pos=ctypes.c_void_p((1 << 50) + 2)) == -6
    for change, code in ((dict(D=0), -3), (dict(D=60), -3), (dict(D=264), -3), (dict(B=0), -4), (dict(T=0), -4), (dict(NH=0), -4),
                         (dict(D=56), -4), (dict(q_row=248), -4), (dict(k_row=132), -4), (dict(qo_seq=2552), -4),
                         (dict(ko_seq=100), -4), (dict(B=1 << 25), -5), (dict(T=1 << 25, B=1), -5),
                         (dict(B=1, T=1 << 24, NH=1 << 13, NKV=0, q_row=1 << 20, qo_row=1 << 20), -5)):
        assert call(rotary_params(**change)) == code, change
    broken = R.RotaryPlan.of(64)
    broken.dims = 63
    assert call(plan=broken) == -4
    broken.dims = 0
    assert call(plan=broken) == -4
    # shared memory: in place with other strides, half over an input, outputs over each other
    assert call(rotary_params(qo_row=512, qo_seq=5120), qo=AT(0)) == -11
    near = ctypes.c_void_p(AT(0).value + 256)
    assert call(qo=near) == -11 and call(ko=near) == -11 and call(qo=AT(1)) == -11 and call(ko=AT(2)) == -11
    assert call(pos=AT(2)) == -11 and call(pos=AT(3)) == -11


def norm_params(rows=10, cols=768, eps=1e-5, group=0):
    return N.RmsnormParams(rows, cols, eps, group)


def test_norm_refusals():
    L = N._L()
    fwd = lambda p, *a: L.rmsnormForward(*a, p and ctypes.byref(p), None)
    fp8 = lambda p, *a: L.rmsnormForwardFp8(*a, p and ctypes.byref(p), None)
    bwd = lambda p, *a, n=1 << 30: L.rmsnormBackward(*a, n, p and ctypes.byref(p), None)
    six, seven, eight = ([AT(i) for i in range(n)] for n in (6, 7, 8))
    n = ctypes.c_uint64()
    for p, code in ((None, -1), (norm_params(rows=0), -4), (norm_params(cols=0), -4), (norm_params(cols=12), -4),
                    (norm_params(cols=8200), -4), (norm_params(eps=-1.0), -4), (norm_params(eps=float("nan")), -4),
                    (norm_params(eps=float("inf")), -4), (norm_params(group=16), -4), (norm_params(group=256), -4),
                    (norm_params(rows=1 << 24), -5)):
        assert fwd(p, *six) == code and fp8(p, *seven) == code and bwd(p, *eight) == code
        assert L.metalllmRmsnormBackwardWorkspaceSize(p and ctypes.byref(p), ctypes.byref(n)) == code
    p = norm_params()
    bad = ctypes.c_void_p((1 << 50) + 2)
    put = lambda a, i, x: a[:i] + [x] + a[i + 1:]
    for i in range(6):  # x, residual, sum, out, gamma, rstd
        assert fwd(p, *put(six, i, bad)) == -6
        if i in (0, 2, 3, 4):
            assert fwd(p, *put(six, i, None)) == -1
    for i in range(7):  # x, residual, sum, out, scales, gamma, rstd
        assert fp8(p, *put(seven, i, bad)) == -6
        if i in (0, 2, 3, 4, 5):
            assert fp8(p, *put(seven, i, None)) == -1
    for i in range(8):  # dOut, dSum, h, gamma, rstd, dX, dgamma, workspace
        assert bwd(p, *put(eight, i, bad)) == -6
        if i != 1:
            assert bwd(p, *put(eight, i, None)) == -1
    assert L.metalllmRmsnormBackwardWorkspaceSize(ctypes.byref(p), None) == -1
    need = N.backward_workspace_bytes(10, 768)
    assert need > 0 and bwd(p, *eight, n=need - 1) == -5
    # shared memory that is not allowed
    half = lambda i: ctypes.c_void_p(AT(i).value + 16)
    for i, x in ((2, half(0)), (3, half(1)), (3, AT(2)), (5, AT(0)), (5, AT(3)), (3, AT(4)), (2, AT(4))):
        assert fwd(p, *put(six, i, x)) == -11
    for i, x in ((3, AT(0)), (4, AT(1)), (4, AT(3)), (6, AT(4))):
        assert fp8(p, *put(seven, i, x)) == -11
    for i, x in ((5, half(0)), (5, half(2)), (5, AT(6)), (6, AT(0)), (7, AT(2)), (7, AT(5)), (6, AT(3)), (5, AT(4))):
        assert bwd(p, *put(eight, i, x)) == -11


def test_python_checks():
    import torch
    x = torch.zeros(4, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        N.rmsnormForward(x, None, None, x, x[0])
    with pytest.raises(ValueError, match="GPU"):
        R.rotaryForward(x.view(1, 1, 4, 16), None, x.view(1, 1, 4, 16), None, None, R.RotaryPlan.of(16))
    with pytest.raises(ValueError, match="together"):
        R.rotaryForward(x, x, x, None, None, R.RotaryPlan.of(16))
    with pytest.raises(ValueError):
        N.RmsnormParams.of(-1, 8)
