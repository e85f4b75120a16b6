"""Shared by the window attention tests: inputs, the definition in 64 bits row by row over the visible keys
alone, and how far the kernels may be from it.

Tolerances, per element, from the roundings that the kernels make. A rounding to bf16 is off by at most
u = 2^-8 of the value, a 32-bit operation by 2^-24.
  score s_ij: its product of D terms and the exponent's arithmetic are off by at most
      e_s = (D + 8) 2^-24 max_ij sum_d |q_id k_jd| / sqrt(D)  (+ 2^-22 of the largest exponent's size)
  weight P_ij: by (2 e_s + n 2^-23) P_ij =: e P_ij (n terms in the sum)
  out: u |o| (output) + sum_j P_ij |v_j| (u + e + n 2^-24)
  l: e_s + n 2^-23 + 2^-22 |l|
  dl_i = sum_d dO.O: dO times the error of out, and D 2^-24 of its terms
  dS_ij: u |dS_ij| + P_ij (error of dl_i + e (|dP_ij| + |dl_i|) + D 2^-24 sum|dO v|) / sqrt(D) =: E_ij
  dV: u |dV| + sum_i P_ij |dO_i| (u + e + n 2^-24);  dQ: u |dQ| + sum_j E_ij |k_j| (1 + n 2^-24), dK likewise
"""
import math

import numpy as np

U = 2.0 ** -8


def bf16(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16)


def make(case, seed=0):
    """q, k, v, dO as bf16 CPU tensors, and lengths (int32 tensors or None)."""
    import torch
    rng = np.random.default_rng(seed + 7 * case["TQ"] + case["TK"])
    n = lambda T, H: bf16(rng.standard_normal((case["B"], T, H, case["D"])) * case.get("scale", 1.0))
    d = dict(q=n(case["TQ"], case["NH"]), k=n(case["TK"], case["NKV"]), v=n(case["TK"], case["NKV"]), dO=n(case["TQ"], case["NH"]))
    for name in ("q_len", "k_len"):
        d[name] = None if case.get(name) is None else torch.tensor(case[name], dtype=torch.int32)
    return d


def lengths(case, b):
    lq = case["TQ"] if case.get("q_len") is None else min(max(case["q_len"][b], 0), case["TQ"])
    lk = case["TK"] if case.get("k_len") is None else min(max(case["k_len"][b], 0), case["TK"])
    return lq, lk


def visible(case, lq, lk, i):
    pos = lk - lq + i
    j = np.arange(lk)
    return np.nonzero((j <= pos) & ((pos - j < case["window"]) | (j < case["sinks"])))[0]


def reference(case, d, grad=True):
    """{name: (value, tolerance)} as float64 arrays; rows behind a sequence's length hold NaN."""
    B, TQ, TK, NH, NKV, D = (case[n] for n in ("B", "TQ", "TK", "NH", "NKV", "D"))
    f = {n: d[n].double().numpy() for n in ("q", "k", "v", "dO")}
    root = math.sqrt(D)
    none = lambda *s: np.full(s, np.nan)
    r = {"out": [none(B, TQ, NH, D), none(B, TQ, NH, D)], "l": [none(B, NH, TQ), none(B, NH, TQ)]}
    if grad:
        r["dQ"] = [none(B, TQ, NH, D), none(B, TQ, NH, D)]
        for n in ("dK", "dV"):
            r[n] = [none(B, TK, NKV, D), none(B, TK, NKV, D)]
    e32 = 2.0 ** -24
    with np.errstate(all="ignore"):
        for b in range(B):
            lq, lk = lengths(case, b)
            for n in ("dK", "dV") if grad else ():
                r[n][0][b, :lk] = 0.0
                r[n][1][b, :lk] = 0.0
            for h in range(NH):
                kh = h // (NH // NKV)
                for i in range(lq):
                    see = visible(case, lq, lk, i)
                    q, g = f["q"][b, i, h], f["dO"][b, i, h]
                    k, v = f["k"][b, see, kh], f["v"][b, see, kh]
                    if not len(see):
                        r["out"][0][b, i, h] = r["out"][1][b, i, h] = 0.0
                        r["l"][0][b, h, i], r["l"][1][b, h, i] = -np.inf, 0.0
                        if grad:
                            r["dQ"][0][b, i, h] = r["dQ"][1][b, i, h] = 0.0
                        continue
                    n = len(see)
                    s = k @ q / root
                    m = s.max()
                    p = np.exp(s - m)
                    l = m + np.log(p.sum())
                    p = p / p.sum()
                    es = (D + 8) * e32 * (np.abs(k) @ np.abs(q)).max() / root + 2.0 ** -22 * np.abs(s).max()
                    e = 2 * es + n * 2 * e32
                    o = p @ v
                    to = U * np.abs(o) + (p @ np.abs(v)) * (U + e + n * e32) * (1 + U)
                    r["out"][0][b, i, h], r["out"][1][b, i, h] = o, to
                    r["l"][0][b, h, i], r["l"][1][b, h, i] = l, es + n * 2 * e32 + 2.0 ** -22 * abs(l)
                    if not grad:
                        continue
                    dP, terms = v @ g, np.abs(v) @ np.abs(g)
                    dl = g @ o
                    tdl = np.abs(g) @ to + D * e32 * (np.abs(g) @ np.abs(o))
                    dS = p * (dP - dl) / root
                    E = U * np.abs(dS) + p * (1 + U) * (tdl + (e + 8 * e32) * (np.abs(dP) + abs(dl)) + D * e32 * terms) / root
                    dQ = dS @ k
                    r["dQ"][0][b, i, h] = dQ
                    r["dQ"][1][b, i, h] = U * np.abs(dQ) + (E @ np.abs(k) + n * e32 * (np.abs(dS) @ np.abs(k))) * (1 + U)
                    m_ = TQ * (NH // NKV)
                    r["dK"][0][b, see, kh] += dS[:, None] * q
                    r["dK"][1][b, see, kh] += (E + m_ * e32 * np.abs(dS))[:, None] * np.abs(q) * (1 + U)
                    r["dV"][0][b, see, kh] += p[:, None] * g
                    r["dV"][1][b, see, kh] += (p * (U + e + m_ * e32))[:, None] * np.abs(g) * (1 + U)
    for n in ("dK", "dV") if grad else ():
        r[n][1] += U * np.abs(r[n][0])
    return {n: tuple(x) for n, x in r.items()}


def far(case, name, got, want, tol):
    """A line on the worst element beyond its tolerance, or None; NaN and infinities have to be in the same
    places. Rows behind a sequence's length are not looked at."""
    live = ~behind(case, want.shape, name)
    x, w, t = got.detach().double().cpu().numpy()[live], want[live], tol[live]
    if not np.array_equal(np.isnan(w), np.isnan(x)):
        return f"{name}: NaN in {np.sum(np.isnan(x))} places, wanted in {np.sum(np.isnan(w))}"
    fine = np.isfinite(w)
    if not np.array_equal(x[~fine & ~np.isnan(w)], w[~fine & ~np.isnan(w)]):
        return f"{name}: infinities differ"
    x, w, t = x[fine], w[fine], t[fine]
    bad = np.nonzero(~(np.abs(x - w) <= t))[0]
    if len(bad):
        k = bad[np.argmax(np.abs(x - w)[bad])]
        return f"{name}: {x[k]} against {w[k]}, tolerance {t[k]} ({len(bad)} of {len(x)})"
    return None


def behind(case, shape, name):
    """Which rows of an output lie behind the lengths."""
    mask = np.zeros(shape, dtype=bool)
    for b in range(case["B"]):
        lq, lk = lengths(case, b)
        if name == "l":
            mask[b, :, lq:] = True
        else:
            mask[b, (lk if name in ("dK", "dV") else lq):] = True
    return mask
