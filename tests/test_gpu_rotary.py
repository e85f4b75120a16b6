"""rotaryForward and rotaryBackward on the GPU against the definition in 64 bits.

Tolerance: y = m (x1 c - x2 s), rounded once to bf16 (u = 2^-8 of the value). The hardware sine and cosine of
an angle in turns are taken to be off by at most 2^-16 (they are documented for 32-bit arguments with errors
near 2^-20; the angle's own rounding to 32 bits, at most 2^-26 turns, adds 2pi 2^-26)."""
import math

import numpy as np
import pytest

from tests.window_case import bf16

pytestmark = pytest.mark.gpu


def frequencies(R, base, scaling, k):
    f = base ** (-2.0 * np.arange(R // 2) / R)
    if scaling == "linear":
        f = f / k["factor"]
    if scaling == "parts":
        keep = np.clip((k["original"] * f / (2 * math.pi) - k["low"]) / (k["high"] - k["low"]), 0, 1)
        f = f * keep + f / k["factor"] * (1 - keep)
    return f


def turned(x, pos, R, interleaved, f, m, back):
    x = x.double().numpy()
    y, t = x.copy(), np.zeros_like(x)
    a = pos.astype(np.float64)[..., None] * f
    c, s = np.cos(a)[:, :, None] * m, np.sin(a)[:, :, None] * m * (-1 if back else 1)
    i1 = np.arange(0, R, 2) if interleaved else np.arange(R // 2)
    i2 = i1 + 1 if interleaved else i1 + R // 2
    x1, x2 = x[..., i1], x[..., i2]
    y[..., i1], y[..., i2] = x1 * c - x2 * s, x1 * s + x2 * c
    for i in (i1, i2):
        t[..., i] = 2.0 ** -8 * np.abs(y[..., i]) + abs(m) * (np.abs(x1) + np.abs(x2)) * 2.0 ** -16
    return y, t


CASES = [
    # B, T, NH, NKV, D, R, interleaved, scaling, most, in place
    (1, 1, 1, 1, 64, 64, False, "none", 1, False), (3, 5, 4, 2, 128, 128, False, "parts", 1000000, False),
    (2, 7, 3, 3, 64, 48, True, "none", 4000, True), (2, 9, 5, 1, 128, 96, True, "linear", 100000, False),
    (1, 33, 2, 2, 64, 10, False, "none", 500, False), (2, 6, 3, 1, 128, 2, True, "parts", 500, False),
    (2, 11, 7, 1, 64, 30, True, "linear", 9000, True), (1, 3, 2, 1, 8, 8, False, "none", 100, False),
    (1, 3, 9, 1, 24, 16, False, "none", 100, True), (2, 130, 12, 4, 256, 256, False, "parts", 2000000000, False),
]


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("B,T,NH,NKV,D,R,inter,scaling,most,place", CASES)
def test_rotary(gpu, B, T, NH, NKV, D, R, inter, scaling, most, place, back):
    import torch
    import metalllm_amd.rotary as M
    print(f"case {(B, T, NH, NKV, D, R, inter, scaling, most, place, back)}", flush=True)
    rng = np.random.default_rng(B * T + D + R)
    k = dict(factor=8.0, original=2048.0, low=1.0, high=16.0) if scaling != "none" else {}
    m = 1.25 if scaling == "parts" else 1.0
    q, kk = bf16(rng.standard_normal((B, T, NH, D))), bf16(rng.standard_normal((B, T, NKV, D)))
    pos = rng.integers(-most if most > 1 else 0, most, (B, T)).astype(np.int32)
    plan = M.RotaryPlan.of(R, 10000.0, inter, scaling, magnitude=m, **k)
    tq, tk = q.to(gpu), kk.to(gpu)
    oq, ok = (tq, tk) if place else (torch.full_like(tq, float("nan")), torch.full_like(tk, float("nan")))
    (M.rotaryBackward if back else M.rotaryForward)(tq, tk, oq, ok, torch.from_numpy(pos).to(gpu), plan)
    torch.cuda.synchronize()
    f = frequencies(R, 10000.0, scaling, k)
    for x, y in ((q, oq), (kk, ok)):
        want, tol = turned(x, pos, R, inter, f, m, back)
        got = y.double().cpu().numpy()
        assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) - tol).max()
        assert np.array_equal(got[..., R:], want[..., R:])


def test_default_positions_q_alone_and_strides(gpu):
    import torch
    import metalllm_amd.rotary as M
    rng = np.random.default_rng(3)
    plan = M.RotaryPlan.of(64)
    x = bf16(rng.standard_normal((2, 19, 6 * 64 + 2 * 128))).to(gpu)
    q, k = x[..., :384].unflatten(2, (6, 64)), x[..., 384:512].unflatten(2, (2, 64))
    f = frequencies(64, 10000.0, "none", {})
    pos = np.tile(np.arange(19), (2, 1))
    before = x.clone()
    wq, wk = turned(q.cpu(), pos, 64, False, f, 1.0, False), turned(k.cpu(), pos, 64, False, f, 1.0, False)
    alone = torch.empty(2, 19, 6, 64, dtype=torch.bfloat16, device=gpu)
    M.rotaryForward(q, None, alone, None, None, plan)
    M.rotaryForward(q, k, q, k, None, plan)  # in place, in a packed buffer
    torch.cuda.synchronize()
    for y, (w, t) in ((alone, wq), (q, wq), (k, wk)):
        assert (np.abs(y.double().cpu().numpy() - w) <= t).all()
    assert torch.equal(x[..., 512:], before[..., 512:])


def test_backward_is_the_transpose(gpu):
    """<turned(x), y> = <x, turned back(y)>, up to one rounding of each value."""
    import torch
    import metalllm_amd.rotary as M
    rng = np.random.default_rng(4)
    x, y = bf16(rng.standard_normal((1, 50, 2, 64))).to(gpu), bf16(rng.standard_normal((1, 50, 2, 64))).to(gpu)
    plan = M.RotaryPlan.of(32, interleaved=True, scaling="linear", factor=3.0, magnitude=0.7)
    a, b = torch.empty_like(x), torch.empty_like(y)
    M.rotaryForward(x, None, a, None, None, plan)
    M.rotaryBackward(y, None, b, None, None, plan)
    left, right = (a.double() * y.double()), (x.double() * b.double())
    tol = 2.0 ** -8 * (left.abs().sum() + right.abs().sum()) + 1e-3
    assert (left.sum() - right.sum()).abs() <= tol


def test_captured_and_replayed(gpu):
    import torch
    import metalllm_amd.rotary as M
    q, k = (torch.randn(2, 9, h, 128, device=gpu).to(torch.bfloat16) for h in (4, 2))
    pos = torch.zeros(2, 9, dtype=torch.int32, device=gpu)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    plan = M.RotaryPlan.of(128, scaling="parts", factor=4.0, original=100.0)
    graph = torch.cuda.CUDAGraph()
    M.rotaryForward(q, k, qo, ko, pos, plan)
    with torch.cuda.graph(graph):
        M.rotaryForward(q, k, qo, ko, pos, plan)
    del plan  # calls copy it
    plan = M.RotaryPlan.of(128, scaling="parts", factor=4.0, original=100.0)
    for n in (5, 1234567):
        pos.copy_(torch.arange(18, device=gpu, dtype=torch.int32).view(2, 9) * n)
        graph.replay()
        torch.cuda.synchronize()
        a, b = qo.clone(), ko.clone()
        M.rotaryForward(q, k, qo, ko, pos, plan)
        torch.cuda.synchronize()
        assert torch.equal(a, qo) and torch.equal(b, ko)
