"""The attention half of a block from the operators together, as a program runs it: norm with the residual,
computeQKV, rotary positions in place, window attention, projForward, and the gradients back through them; and
the next tokens over the cache that a prompt left. Against the same chain in 64 bits.

Tolerance of the chain: every stored activation is rounded once to bf16, off by at most u = 2^-8 of its size.
The output passes 6 such roundings (norm, q or k or v, turned q or k, weight, attention output, output); scores
here are below 4 in magnitude, and a score's error of 2u of it (two rounded factors, each rounded twice) moves its
weight by as much, so the relative 2-norm error is at most (6 + 2 * 2 * 4) u = 22 u = 0.086. The gradients pass
the same ones and as many on the way back: 44 u = 0.17. Sums over many elements of independent roundings stay
far inside."""
import math

import numpy as np
import pytest

from tests.window_case import bf16, far, make, reference

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def inputs(B, T, H, D, seed=0):
    rng = np.random.default_rng(seed)
    C = H * D
    n = lambda *s, scale=1.0: bf16(rng.standard_normal(s) * scale)
    return dict(x=n(B, T, C), res=n(B, T, C), gamma=bf16(1 + 0.1 * rng.standard_normal(C)), wq=n(C, C, scale=C ** -0.5),
                wk=n(C, C, scale=C ** -0.5), wv=n(C, C, scale=C ** -0.5), wp=n(C, C, scale=C ** -0.5), dOut=n(B, T, C), dSum=n(B, T, C))


def exact(d, H, D, window, sinks, base=10000.0):
    import torch
    t = {n: v.double().requires_grad_() for n, v in d.items()}
    B, T, C = t["x"].shape
    h = t["x"] + t["res"]
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-5) * t["gamma"]
    q, k, v = ((y @ t[w]).view(B, T, H, D) for w in ("wq", "wk", "wv"))
    a = torch.arange(T, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    c, s = torch.cos(a)[None, :, None], torch.sin(a)[None, :, None]

    def turn(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat((a * c - b * s, a * s + b * c), -1)

    q, k = turn(q), turn(k)
    i, j = torch.arange(T)[:, None], torch.arange(T)[None]
    see = (j <= i) & ((i - j < window) | (j < sinks))
    score = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(D)
    p = torch.softmax(score.masked_fill(~see, -math.inf), -1)
    o = torch.einsum("bhij,bjhd->bihd", p, v).reshape(B, T, C)
    out = o @ t["wp"]
    ((out * t["dOut"]).sum() + (h * t["dSum"]).sum()).backward()
    assert score.detach().masked_fill(~see, 0).abs().max() < 4.0 * 2
    return out.detach(), h.detach(), t["x"].grad, t["gamma"].grad, [t[w].grad for w in ("wq", "wk", "wv", "wp")]


def off(got, want):
    return float((got.detach().double().cpu() - want).norm() / want.norm())


class Half:
    """The buffers and calls of a program."""

    def __init__(self, d, H, D, window, sinks, dev):
        import torch
        import metalllm_amd as M
        self.t = {n: v.to(dev) for n, v in d.items()}
        B, T, C = d["x"].shape
        self.p = M.AttentionParams.of(B, T, H, D)
        bf = lambda: torch.empty(B, T, C, dtype=torch.bfloat16, device=dev)
        self.sum, self.y, self.o, self.out, self.dO, self.dY, self.dX = (bf() for _ in range(7))
        self.q, self.k, self.v, self.dQ, self.dK, self.dV = (bf() for _ in range(6))
        self.heads = {n: getattr(self, n).view(B, T, H, D) for n in ("q", "k", "v", "o", "dO", "dQ", "dK", "dV")}
        self.rstd, self.l = torch.empty(B * T, device=dev), torch.empty(B, H, T, device=dev)
        self.dQ32, self.dY32 = (torch.empty(B, T, C, device=dev) for _ in range(2))
        self.dgamma, self.dWq = torch.empty(C, device=dev), torch.empty(C, C, device=dev)
        self.dWk, self.dWv, self.dWp = (torch.empty(C, C, dtype=torch.bfloat16, device=dev) for _ in range(3))
        self.plan = M.rotary.RotaryPlan.of(D)
        h = self.heads
        self.wp = M.window.WindowParams.of(h["q"], h["k"], h["v"], h["o"], window, sinks)
        n = max(M.window.backward_workspace_bytes(self.wp), M.window.forward_workspace_bytes(self.wp),
                M.rmsnorm.backward_workspace_bytes(B * T, C))
        self.ws = torch.empty(n, dtype=torch.uint8, device=dev)

    def forward(self):
        import metalllm_amd as M
        t, h = self.t, self.heads
        M.rmsnorm.rmsnormForward(t["x"], t["res"], self.sum, self.y, t["gamma"], self.rstd)
        M.sublayer.computeQKV(self.y, self.q, self.k, self.v, t["wq"], t["wk"], t["wv"], self.p)
        M.rotary.rotaryForward(h["q"], h["k"], h["q"], h["k"], None, self.plan)
        M.window.windowAttentionForward(h["q"], h["k"], h["v"], h["o"], self.l, workspace=self.ws, params=self.wp)
        M.sublayer.projForward(self.o, t["wp"], self.out, self.p)

    def backward(self):
        import metalllm_amd as M
        t, h = self.t, self.heads
        for x in (self.dY32, self.dWq, self.dWk, self.dWv, self.dWp):
            x.zero_()
        M.sublayer.projBackwarddW(self.o, t["dOut"], self.dWp, self.p)
        M.sublayer.projBackwarddX(t["dOut"], t["wp"], self.dO, self.p)
        M.window.windowAttentionBackward(h["dO"], h["o"], self.l, h["q"], h["k"], h["v"], h["dQ"], h["dK"], h["dV"],
                                         workspace=self.ws, params=self.wp)
        M.rotary.rotaryBackward(h["dQ"], h["dK"], h["dQ"], h["dK"], None, self.plan)
        self.dQ32.copy_(self.dQ)  # the products take dQ in 32 bits
        M.sublayer.computeGradDx(self.dY32, t["wq"], t["wk"], t["wv"], self.dQ32, self.dK, self.dV, self.p)
        M.sublayer.computeGradDw(self.y, self.dQ32, self.dK, self.dV, self.dWq, self.dWk, self.dWv, self.p)
        M.glue.castFloatToBfloat(self.dY32, self.dY)
        M.rmsnorm.rmsnormBackward(self.dY, t["dSum"], self.sum, t["gamma"], self.rstd, self.dX, self.dgamma, self.ws)

    def results(self):
        return dict(out=self.out, sum=self.sum, dX=self.dX, dgamma=self.dgamma, dWq=self.dWq, dWk=self.dWk, dWv=self.dWv, dWp=self.dWp)


@pytest.mark.parametrize("B,T,H,D,window,sinks", [(2, 160, 4, 64, 50, 4), (1, 320, 2, 128, 100, 0)])
def test_forward_and_gradients(gpu, B, T, H, D, window, sinks):
    import torch
    print(f"case {(B, T, H, D, window, sinks)}", flush=True)
    d = inputs(B, T, H, D)
    half = Half(d, H, D, window, sinks, gpu)
    half.forward()
    half.backward()
    torch.cuda.synchronize()
    out, h, dX, dgamma, dW = exact(d, H, D, window, sinks)
    r = half.results()
    assert off(r["sum"], h) <= U and off(r["out"], out) <= 22 * U
    for n, want in (("dX", dX), ("dgamma", dgamma), *zip(("dWq", "dWk", "dWv", "dWp"), dW)):
        assert off(r[n], want) <= 44 * U, (n, off(r[n], want))


def test_captured_step_repeats(gpu):
    """The whole step in one graph, on other data each replay, equal to the eager calls bit for bit."""
    import torch
    import metalllm_amd as M
    half = Half(inputs(2, 160, 4, 64), 4, 64, 50, 4, gpu)
    M.sublayer.reserve(M.AttentionParams.of(1, 320, 4, 64))  # as many rows; the products take any T, reserve whole tiles

    def step():
        half.forward()
        half.backward()

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2, 3):
        for n, v in inputs(2, 160, 4, 64, seed).items():
            half.t[n].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = {n: v.clone() for n, v in half.results().items()}
        step()
        torch.cuda.synchronize()
        for n, v in half.results().items():
            assert torch.equal(v, got[n]), n


@pytest.mark.parametrize("D,NH,NKV,window,sinks", [(64, 4, 4, 30, 3), (128, 8, 2, 200, 0)])
def test_next_tokens_over_the_cache_of_a_prompt(gpu, D, NH, NKV, window, sinks):
    """A prompt's rows written to a cache, then one token at a time: each row as in one pass over all rows."""
    import torch
    import metalllm_amd as M
    B, T, more, room = 2, 90, 5, 128
    c = dict(B=B, TQ=T + more, TK=T + more, NH=NH, NKV=NKV, D=D, window=window, sinks=sinks)
    d = make(c)
    plan = M.rotary.RotaryPlan.of(D, interleaved=True, scaling="linear", factor=2.0)
    q, k, v = (d[n].to(gpu) for n in ("q", "k", "v"))
    tq, tk = torch.empty_like(q), torch.empty_like(k)
    M.rotary.rotaryForward(q, k, tq, tk, None, plan)
    torch.cuda.synchronize()
    whole = dict(d, q=tq.cpu(), k=tk.cpu())
    want = reference(c, whole, False)
    cache_k, cache_v = (torch.full((B, room, NKV, D), float("nan"), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    # the prompt: turned straight into the cache
    first = torch.empty(B, T, NH, D, dtype=torch.bfloat16, device=gpu)
    M.rotary.rotaryForward(q[:, :T], k[:, :T], first, cache_k[:, :T], None, plan)
    cache_v[:, :T] = v[:, :T]
    k_len = torch.full((B,), T, dtype=torch.int32, device=gpu)
    rows = [M.window.window_attention_forward(first, cache_k, cache_v, window, sinks, k_len=k_len)[0]]
    one = torch.empty(B, 1, NH, D, dtype=torch.bfloat16, device=gpu)
    for n in range(T, T + more):
        pos = torch.full((B, 1), n, dtype=torch.int32, device=gpu)
        M.rotary.rotaryForward(q[:, n:n + 1], k[:, n:n + 1], one, cache_k[:, n:n + 1], pos, plan)
        cache_v[:, n] = v[:, n]
        k_len += 1
        rows.append(M.window.window_attention_forward(one, cache_k, cache_v, window, sinks, k_len=k_len)[0])
    torch.cuda.synchronize()
    line = far(c, "out", torch.cat(rows, 1), *want["out"])
    assert line is None, line
