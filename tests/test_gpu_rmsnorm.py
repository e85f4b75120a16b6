"""rmsnormForward, rmsnormForwardFp8 and rmsnormBackward on the GPU against the definition in 64 bits.

Tolerances. A sum of n 32-bit terms is off by at most n 2^-24 of the sum of their sizes; with e = (cols + 16)
2^-24: rstd by e of its value, out by 2^-8 (bf16) or 2^-4 of its value, at least half of e4m3's smallest step
2^-9 (times the scale), plus 2 e. dX: 2^-8 of it, and 4 e of the sizes of its terms; dgamma: (rows + 8) 2^-24
of the sizes of its terms."""
import numpy as np
import pytest

from tests.window_case import bf16

pytestmark = pytest.mark.gpu

SHAPES = [(1, 8), (3, 16), (7, 768), (5, 504), (33, 520), (64, 1024), (17, 1032), (6, 2048), (9, 2056), (130, 4096), (4, 4104),
          (3, 8192), (1000, 768), (4099, 64)]


def data(rows, cols, seed=0):
    rng = np.random.default_rng(rows * 31 + cols + seed)
    n = lambda *s: rng.standard_normal(s)
    return dict(x=bf16(n(rows, cols)), r=bf16(2 * n(rows, cols)), g=bf16(1 + 0.2 * n(cols)), dy=bf16(n(rows, cols)), ds=bf16(n(rows, cols)))


def forward64(d, eps, residual=True):
    h = d["x"].double().numpy() + (d["r"].double().numpy() if residual else 0.0)
    rstd = 1 / np.sqrt((h * h).mean(1) + eps)
    return h, rstd, h * rstd[:, None] * d["g"].double().numpy()


def near(got, want, tol):
    x = got.double().cpu().numpy()
    assert (np.abs(x - want) <= tol).all(), float((np.abs(x - want) - tol).max())


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(gpu, rows, cols):
    import torch
    import metalllm_amd.rmsnorm as M
    print(f"case {rows} {cols}", flush=True)
    d = data(rows, cols)
    t = {n: x.to(gpu) for n, x in d.items()}
    e = (cols + 16) * 2.0 ** -24
    nan = lambda x: torch.full_like(x, float("nan"))
    s, o, rstd = nan(t["x"]), nan(t["x"]), torch.full((rows,), float("nan"), device=gpu)
    M.rmsnormForward(t["x"], t["r"], s, o, t["g"], rstd, eps=1e-3)
    h, r64, y = forward64(d, 1e-3)
    near(s, h, 2.0 ** -8 * np.abs(h)), near(rstd, r64, e * r64), near(o, y, (2.0 ** -8 + 2 * e) * np.abs(y))
    # without a residual, and without what is optional
    M.rmsnormForward(t["x"], None, None, o, t["g"], None, eps=0.0)
    _, _, y = forward64(d, 0.0, False)
    near(o, y, (2.0 ** -8 + 2 * e) * np.abs(y))
    # in the residual's and x's memory
    x2, r2 = t["x"].clone(), t["r"].clone()
    M.rmsnormForward(x2, r2, r2, x2, t["g"], rstd, eps=1e-3)
    M.rmsnormForward(t["x"], t["r"], s, o, t["g"], rstd, eps=1e-3)
    assert torch.equal(r2, s) and torch.equal(x2, o)


@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_fp8(gpu, rows, cols, group):
    import torch
    import metalllm_amd.rmsnorm as M
    print(f"case {rows} {cols} {group}", flush=True)
    d = data(rows, cols, 1)
    d["r"][0] = -d["x"][0]  # a row of zeros
    t = {n: x.to(gpu) for n, x in d.items()}
    n = -(-cols // group) if group else 1
    s = torch.full_like(t["x"], float("nan"))
    o = torch.full((rows, cols), 1.0, device=gpu).to(torch.float8_e4m3fn)
    sc, rstd = (torch.full(z, float("nan"), device=gpu) for z in ((rows, n), (rows,)))
    M.rmsnormForwardFp8(t["x"], t["r"], s, o, sc, t["g"], rstd, eps=1e-5, group=group)
    e = (cols + 16) * 2.0 ** -24
    h, r64, y = forward64(d, 1e-5)
    w = group or cols
    pad = np.pad(np.abs(y), ((0, 0), (0, n * w - cols))).reshape(rows, n, w).max(2) / 448
    pad[pad == 0] = 1.0
    near(sc, pad, 3 * e * pad), near(rstd, r64, e * r64), near(s, h, 2.0 ** -8 * np.abs(h))
    each = np.repeat(pad, w, 1)[:, :cols]
    value = o.float().double().cpu().numpy() * each
    tol = np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * each) + 6 * e * np.abs(y)
    assert (np.abs(value - y) <= tol).all()


@pytest.mark.parametrize("rows,cols", SHAPES + [(2049, 104), (2100, 1024), (2048, 1040), (2055, 2040), (513, 2056), (600, 4104)])
def test_backward(gpu, rows, cols):
    import torch
    import metalllm_amd.rmsnorm as M
    print(f"case {rows} {cols}", flush=True)
    d = data(rows, cols, 2)
    t = {n: x.to(gpu) for n, x in d.items()}
    h = d["r"].double().numpy()
    rstd = torch.from_numpy((1 / np.sqrt((h * h).mean(1) + 1e-5)).astype(np.float32))
    r = rstd.double().numpy()[:, None]
    g, dy, ds = (d[n].double().numpy() for n in ("g", "dy", "ds"))
    xh = h * r
    mean = (dy * g * xh).mean(1, keepdims=True)
    e = (cols + 16) * 2.0 ** -24
    size = r * (np.abs(dy * g) + np.abs(xh) * np.abs(dy * g * xh).mean(1, keepdims=True))
    ws = torch.full((M.backward_workspace_bytes(rows, cols),), 255, dtype=torch.uint8, device=gpu)
    for have in (True, False):
        dX, dg = torch.full_like(t["dy"], float("nan")), torch.full((cols,), float("nan"), device=gpu)
        M.rmsnormBackward(t["dy"], t["ds"] if have else None, t["r"], t["g"], rstd.to(gpu), dX, dg, ws)
        want = r * (dy * g - xh * mean) + (ds if have else 0.0)
        near(dX, want, 2.0 ** -8 * np.abs(want) + 4 * e * (size + np.abs(ds)))
        near(dg, (dy * xh).sum(0), (rows + 8) * 2.0 ** -24 * np.abs(dy * xh).sum(0))
    # in the memory of each input that allows it
    for n in ("dy", "r"):
        u = {m: t[m].clone() for m in ("dy", "r")}
        dg2 = torch.empty_like(dg)
        M.rmsnormBackward(u["dy"], None, u["r"], t["g"], rstd.to(gpu), u[n], dg2, ws)
        assert torch.equal(u[n], dX) and torch.equal(dg, dg2)


def test_gradient_of_a_difference(gpu):
    """dX against out and sum at two near points in 64 bits."""
    import torch
    import metalllm_amd.rmsnorm as M
    rows, cols, eps = 5, 200, 1e-5
    d = data(rows, cols, 3)
    h = d["r"].double().numpy()
    rstd = torch.from_numpy((1 / np.sqrt((h * h).mean(1) + eps)).astype(np.float32)).to(gpu)
    t = {n: x.to(gpu) for n, x in d.items()}
    dX, dg = torch.empty_like(t["dy"]), torch.empty(cols, device=gpu)
    ws = torch.empty(M.backward_workspace_bytes(rows, cols), dtype=torch.uint8, device=gpu)
    M.rmsnormBackward(t["dy"], t["ds"], t["r"], t["g"], rstd, dX, dg, ws)
    way = np.random.default_rng(1).standard_normal((rows, cols))
    dy, ds = d["dy"].double().numpy(), d["ds"].double().numpy()

    def value(h):
        return (h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * d["g"].double().numpy() * dy + h * ds).sum()

    slope = (value(h + 1e-5 * way) - value(h - 1e-5 * way)) / 2e-5
    mine = dX.double().cpu().numpy()
    assert abs((mine * way).sum() - slope) <= (2.0 ** -8 * np.abs(mine * way)).sum() + 1e-3


def test_rows_that_are_not_finite_keep_to_themselves(gpu):
    import torch
    import metalllm_amd.rmsnorm as M
    d = data(9, 256, 4)
    clean = {n: x.to(gpu) for n, x in d.items()}
    d["x"][4, 7] = float("nan")
    d["x"][6, 9] = float("inf")
    t = {n: x.to(gpu) for n, x in d.items()}
    outs = []
    for u in (clean, t):
        s, o, rstd = torch.empty_like(u["x"]), torch.empty_like(u["x"]), torch.empty(9, device=gpu)
        M.rmsnormForward(u["x"], u["r"], s, o, u["g"], rstd)
        outs.append(o.float())
    keep = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(outs[0][keep], outs[1][keep])
    assert outs[1][4].isnan().all() and outs[1][6, 9].isnan() and (outs[1][6, :9] == 0).all()


def test_captured_and_replayed(gpu):
    import torch
    import metalllm_amd.rmsnorm as M
    t = {n: x.to(gpu) for n, x in data(300, 768, 5).items()}
    s, o, dX = (torch.empty_like(t["x"]) for _ in range(3))
    rstd, dg = torch.empty(300, device=gpu), torch.empty(768, device=gpu)
    ws = torch.empty(M.backward_workspace_bytes(300, 768), dtype=torch.uint8, device=gpu)

    def step():
        M.rmsnormForward(t["x"], t["r"], s, o, t["g"], rstd)
        M.rmsnormBackward(t["dy"], t["ds"], s, t["g"], rstd, dX, dg, ws)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (6, 7, 8):
        for n, x in data(300, 768, seed).items():
            t[n].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (s, o, rstd, dX, dg)]
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (s, o, rstd, dX, dg)):
            assert torch.equal(a, b)
