"""windowAttentionForward and windowAttentionBackward on the GPU against the definition in 64 bits
(tests/window_case.py, which derives the tolerances)."""
import numpy as np
import pytest

from tests.window_case import behind, far, make, reference

pytestmark = pytest.mark.gpu


def C(B, TQ, TK, NH, NKV, D, window, sinks, q_len=None, k_len=None, **more):
    return dict(B=B, TQ=TQ, TK=TK, NH=NH, NKV=NKV, D=D, window=window, sinks=sinks, q_len=q_len, k_len=k_len, **more)


def name_of(c):
    return "-".join(f"{k}{v}" for k, v in c.items() if v is not None).replace(" ", "")


TOKENS = [
    C(1, 1, 1, 1, 1, 64, 1, 0), C(1, 1, 1, 4, 1, 128, 7, 64), C(2, 1, 31, 3, 3, 64, 100, 0), C(2, 1, 33, 8, 2, 128, 100, 5),
    C(1, 1, 1000, 12, 12, 64, 512, 4), C(3, 1, 700, 8, 1, 128, 333, 33, None, [700, 1, 350]),
    C(2, 1, 500, 16, 1, 64, 64, 64, [1, 0], [499, 500]), C(2, 1, 300, 6, 2, 128, 1, 0, None, [0, 300]),
    C(1, 1, 5000, 2, 1, 128, 5000, 0), C(1, 1, 5000, 3, 1, 64, 4001, 17), C(2, 3, 400, 4, 2, 64, 100, 4),
    C(2, 5, 260, 8, 2, 128, 70, 3, [5, 2], [260, 4]), C(1, 7, 2500, 8, 1, 64, 1500, 40), C(1, 16, 300, 4, 1, 128, 9, 2),
    C(2, 4, 3, 2, 2, 64, 2, 1), C(1, 1, 90, 40, 1, 64, 50, 4), C(1, 1, 150, 72, 1, 64, 60, 4), C(2, 16, 90, 8, 2, 128, 40, 4),
    C(1, 17, 90, 2, 2, 64, 40, 4), C(1, 50, 3000, 6, 2, 64, 2900, 4), C(2, 130, 1500, 4, 1, 128, 1400, 0, [130, 40], [1500, 777]),
    C(1, 256, 4000, 3, 3, 128, 3800, 7), C(1, 384, 384, 16, 2, 64, 200, 2), C(1, 385, 385, 16, 2, 64, 200, 2), C(300, 1, 40, 2, 1, 64, 20, 2),
]
ROWS = [
    C(1, 17, 17, 1, 1, 64, 100, 0), C(1, 63, 63, 2, 2, 64, 1, 0), C(1, 64, 64, 2, 1, 128, 64, 0),
    C(2, 65, 65, 2, 2, 128, 2, 1), C(1, 128, 128, 3, 1, 64, 4096, 0), C(1, 129, 129, 1, 1, 128, 65, 64),
    C(1, 200, 200, 2, 2, 64, 63, 5), C(1, 300, 300, 2, 1, 128, 40, 33), C(1, 700, 700, 1, 1, 64, 40, 4),
    C(1, 520, 520, 3, 1, 128, 17, 64), C(1, 450, 450, 2, 2, 64, 130, 0), C(1, 400, 400, 2, 2, 128, 257, 1),
    C(2, 100, 333, 4, 2, 64, 50, 4), C(1, 130, 513, 2, 1, 128, 300, 0), C(1, 150, 90, 2, 2, 64, 30, 4),
    C(1, 200, 70, 2, 1, 128, 100, 0), C(3, 210, 210, 2, 1, 64, 70, 3, [210, 0, 131], [210, 0, 131]),
    C(4, 190, 260, 2, 2, 128, 33, 9, [190, 1, 77, 190], [260, 260, 50, 3]),
    C(2, 140, 140, 8, 1, 64, 20, 2, [999, -3], [140, 140]), C(1, 260, 260, 2, 2, 64, 100, 4, scale=4.0),
]


def packed(d, dev):
    """q, k and v as slices of one [B, T, (NH + 2 NKV) D] buffer."""
    import torch
    q, k, v = d["q"], d["k"], d["v"]
    if q.shape[1] != k.shape[1]:
        return [t.to(dev) for t in (q, k, v)]
    B, T, NH, D = q.shape
    n = k.shape[2]
    buf = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], 2).to(dev)
    return [buf[..., a * D:b * D].unflatten(2, (b - a, D)) for a, b in ((0, NH), (NH, NH + n), (NH + n, NH + 2 * n))]


def run(c, d, dev, grad=True, layout="plain", want_l=True, fill=float("nan")):
    import torch
    import metalllm_amd.window as W
    print(f"case {name_of(c)} {layout}", flush=True)
    if layout == "packed":
        q, k, v = packed(d, dev)
    elif layout == "token first":  # [T, B, heads, D] in memory
        q, k, v = (d[n].transpose(0, 1).contiguous().to(dev).transpose(0, 1) for n in ("q", "k", "v"))
    else:
        q, k, v = (d[n].to(dev) for n in ("q", "k", "v"))
    dO = d["dO"].to(dev)
    lens = [None if d[n] is None else d[n].to(dev) for n in ("q_len", "k_len")]
    out = torch.full_like(dO, fill)
    l = torch.full((c["B"], c["NH"], c["TQ"]), fill, dtype=torch.float32, device=dev) if want_l else None
    p = W.WindowParams.of(q, k, v, out, c["window"], c["sinks"])
    ws = torch.full((max(1, W.forward_workspace_bytes(p)),), 255, dtype=torch.uint8, device=dev)
    W.windowAttentionForward(q, k, v, out, l, *lens, ws, params=p)
    r = {"out": out, "l": l}
    if grad:
        g = [torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).fill_(fill) for t in (q, k, v)]
        ws = torch.full((W.backward_workspace_bytes(p),), 255, dtype=torch.uint8, device=dev)
        W.windowAttentionBackward(dO, out, l, q, k, v, *g, *lens, ws, params=p)
        r.update(dQ=g[0], dK=g[1], dV=g[2])
    torch.cuda.synchronize()
    return r


def check(c, d, got, want=None):
    want = want or reference(c, d, "dQ" in got)
    for n, x in got.items():
        if x is None:
            continue
        line = far(c, n, x, *want[n])
        assert line is None, line
        rest = x.detach().float().cpu().numpy()[behind(c, want[n][0].shape, n)]
        assert np.isnan(rest).all(), f"{n}: rows behind the lengths were written"


def crowd(c, d, want):
    """The case again with its sequences repeated to more than 8192 rows in all: other kernels than those of fewer
    rows (which split the keys in the forward, and take dS in two parts in the backward)."""
    n = 8192 // (c["B"] * c["NH"] * c["TQ"]) + 1
    c = dict(c, B=c["B"] * n, **{m: c[m] and c[m] * n for m in ("q_len", "k_len")})
    d = {m: x if x is None else x.repeat(n, *[1] * (x.ndim - 1)) for m, x in d.items()}
    return c, d, {m: tuple(np.concatenate([x] * n) for x in w) for m, w in want.items()}


def check_twice(c, d, gpu, want=None, **k):
    want = want or reference(c, d)
    check(c, d, run(c, d, gpu, **k), want)
    c, d, want = crowd(c, d, want)
    check(c, d, run(c, d, gpu, **k), want)


@pytest.mark.parametrize("c", TOKENS, ids=name_of)
def test_tokens(gpu, c):
    d = make(c)
    check(c, d, run(c, d, gpu, grad=False))


@pytest.mark.parametrize("c", ROWS, ids=name_of)
def test_rows(gpu, c):
    d = make(c)
    check_twice(c, d, gpu)


@pytest.mark.parametrize("c", [TOKENS[5], TOKENS[11]], ids=name_of)
def test_gradient_of_few_rows(gpu, c):
    d = make(c)
    check_twice(c, d, gpu)


@pytest.mark.parametrize("layout", ["packed", "token first"])
@pytest.mark.parametrize("c", [C(2, 150, 150, 4, 2, 64, 40, 5), C(3, 1, 200, 4, 1, 128, 150, 3), C(2, 3, 3, 2, 1, 128, 2, 0),
                               C(3, 1030, 1030, 4, 2, 64, 40, 5), C(2, 700, 900, 8, 2, 128, 50, 0)], ids=name_of)
def test_strides(gpu, c, layout):
    d = make(c)
    check(c, d, run(c, d, gpu, layout=layout))


def test_no_logsumexp(gpu):
    for c in (TOKENS[4], ROWS[6]):
        d = make(c)
        check(c, d, run(c, d, gpu, grad=False, want_l=False))


@pytest.mark.parametrize("c", [C(2, 90, 300, 2, 1, 64, 50, 4, [90, 61], [300, 201]), C(2, 90, 300, 2, 2, 128, 50, 0, [90, 61], [300, 201]),
                               C(2, 1, 300, 4, 1, 64, 50, 4, None, [300, 201]), C(1, 3, 300, 4, 2, 128, 50, 4)], ids=name_of)
def test_hidden_values_are_not_read(gpu, c):
    """NaN and infinities behind the lengths and in keys that no row sees change nothing."""
    d = make(c)
    want = reference(c, d)
    for b in range(c["B"]):
        lq = c["TQ"] if c["q_len"] is None else c["q_len"][b]
        lk = c["TK"] if c["k_len"] is None else c["k_len"][b]
        first = max(0, lk - lq - c["window"] + 1)
        for n, bad in (("k", float("nan")), ("v", float("inf"))):
            d[n][b, min(c["sinks"], first):first] = bad
            d[n][b, lk:] = -bad
        d["q"][b, lq:] = float("nan")
        d["dO"][b, lq:] = float("inf")
    got = run(c, d, gpu)
    for n in ("dK", "dV"):  # keys that no row sees: zero
        for b in range(c["B"]):
            lq = c["TQ"] if c["q_len"] is None else c["q_len"][b]
            lk = c["TK"] if c["k_len"] is None else c["k_len"][b]
            first = max(0, lk - lq - c["window"] + 1)
            assert (got[n][b, min(c["sinks"], first):first] == 0).all()
    check(c, d, got, want)
    c, d, want = crowd(c, d, want)
    check(c, d, run(c, d, gpu), want)


@pytest.mark.parametrize("where", ["k", "v", "q", "dO"])
@pytest.mark.parametrize("c", [C(1, 200, 200, 2, 1, 64, 40, 3), C(1, 200, 200, 2, 2, 128, 70, 0), C(1, 5, 120, 4, 2, 64, 30, 2)], ids=name_of)
def test_values_that_are_not_finite_reach_their_rows_alone(gpu, c, where):
    d = make(c)
    at = 100 if d[where].shape[1] > 5 else 3
    d[where][0, at, 0, 5] = float("nan")
    if where == "v":
        d[where][0, at + 4, 0, 9] = float("inf")
    check_twice(c, d, gpu)


def test_results_repeat(gpu):
    import torch
    c = C(2, 300, 300, 4, 2, 128, 64, 5)
    d = make(c)
    a, b = run(c, d, gpu), run(c, d, gpu)
    for n in a:
        assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize("c", [C(2, 1, 2000, 4, 1, 128, 1500, 4, None, [2000, 900]), C(2, 200, 200, 2, 1, 64, 60, 4),
                               C(2, 700, 700, 8, 2, 64, 60, 4)], ids=name_of)
def test_captured_and_replayed(gpu, c):
    """A captured forward and backward on another stream, replayed with new inputs and lengths."""
    import torch
    import metalllm_amd.window as W
    d = make(c)
    t = {n: x.to(gpu) for n, x in d.items() if x is not None}
    out, l = torch.zeros_like(t["dO"]), torch.zeros((c["B"], c["NH"], c["TQ"]), dtype=torch.float32, device=gpu)
    g = [torch.zeros_like(t[n]) for n in ("q", "k", "v")]
    p = W.WindowParams.of(t["q"], t["k"], t["v"], out, c["window"], c["sinks"])
    ws = torch.zeros(max(W.forward_workspace_bytes(p), W.backward_workspace_bytes(p)), dtype=torch.uint8, device=gpu)

    def step():
        W.windowAttentionForward(t["q"], t["k"], t["v"], out, l, t.get("q_len"), t.get("k_len"), ws, params=p)
        W.windowAttentionBackward(t["dO"], out, l, t["q"], t["k"], t["v"], *g, t.get("q_len"), t.get("k_len"), ws, params=p)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2, 3):
        e = make(c, seed)
        if c["k_len"]:
            e["k_len"] += torch.tensor([-seed, 7 * seed], dtype=torch.int32)
        for n in t:
            t[n].copy_(e[n])
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, l, *g)]
        step()
        torch.cuda.synchronize()
        for x, y in zip(got, (out, l, *g)):
            assert torch.equal(x, y)
        now = dict(c, k_len=e["k_len"].tolist() if e["k_len"] is not None else None)
        want = reference(now, e)
        for n, x in zip(("out", "l", "dQ", "dK", "dV"), got):
            if n in ("out", "l", "dQ") or not c["k_len"]:
                assert far(now, n, x, *want[n]) is None, far(now, n, x, *want[n])


def test_offsets_beyond_32_bits(gpu):
    """A cache whose last rows lie more than 2^32 bytes behind its first."""
    import torch
    c = C(1, 2, 700, 2, 1, 128, 100, 4)
    row = 1 << 21  # elements: 700 rows of 4 MiB
    d = make(c)
    buf = torch.empty(700 * row, dtype=torch.bfloat16, device=gpu)
    k = buf.as_strided((1, 700, 1, 128), (700 * row, row, 128, 1))
    v = buf.as_strided((1, 700, 1, 128), (700 * row, row, 128, 1), 128)
    k.copy_(d["k"]), v.copy_(d["v"])
    import metalllm_amd.window as W
    for TQ in (2, 20):
        c = C(1, TQ, 700, 2, 1, 128, 100, 4)
        e = make(c)
        e["k"], e["v"] = d["k"], d["v"]
        out, l = W.window_attention_forward(e["q"].to(gpu), k, v, 100, 4)
        want = reference(c, e, False)
        for n, x in (("out", out), ("l", l)):
            assert far(c, n, x, *want[n]) is None, far(c, n, x, *want[n])


def test_matches_the_full_attention(gpu):
    """With every key in the window it is the causal attention of the framework, up to that one's rounded scores."""
    import torch
    import metalllm_amd as M
    c = C(2, 256, 256, 4, 4, 64, 256, 0)
    d = make(c)
    got = run(c, d, gpu)
    out, lse = M.attention_forward(*(d[n].to(gpu) for n in ("q", "k", "v")))
    # scores rounded to bf16: each off by 2^-8 of at most 8 in magnitude here
    assert (got["l"] - lse).abs().max() <= 2.0 ** -8 * 8
    assert (got["out"].float() - out.float()).abs().max() <= 0.1
    check(c, d, got)


def test_difference_quotient(gpu):
    """The gradient of sum(out dO) along a direction against out at two near points in 64 bits."""
    c = C(1, 40, 40, 2, 1, 64, 17, 3)
    d = make(c)
    got = run(c, d, gpu)
    rng = np.random.default_rng(5)
    h = 1e-4
    for n, g in (("q", "dQ"), ("k", "dK"), ("v", "dV")):
        way = rng.standard_normal(d[n].shape)
        ends = []
        for sign in (1, -1):
            import torch
            moved = dict(d)
            moved[n] = d[n].double() + sign * h * torch.from_numpy(way)
            o = reference(c, moved, False)["out"][0]
            ends.append((o * d["dO"].double().numpy()).sum())
        slope = (ends[0] - ends[1]) / (2 * h)
        mine = (got[g].double().cpu().numpy() * way).sum()
        # every gradient element within its tolerance, and h^2 of the quotient's own error
        tol = (reference(c, d)[g][1] * np.abs(way)).sum() + 1e-4 * abs(slope)
        assert abs(mine - slope) <= tol
