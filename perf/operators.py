"""The operators around the attention core as cases that can be timed and checked: attention over a
window of keys with a few first keys that stay visible, rotary positions, and the root-mean-square
norm with the residual's addition.

Kinds of case, each one pass:
  window        attention forward: a prompt or a part of one behind an existing cache, or single
                tokens (TQ = 1) over a cache
  window_train  attention forward, then backward
  rotary        rotation of q and k
  rotary_back   its gradient
  norm          h = x + residual, the norm of h in bf16
  norm8         the same with the norm in 8 bits (e4m3) and scales
  norm_back     the gradient of the norm and the residual

`own` says whether run() computes a pass in plain torch operations or by the package's entry points.
listed() holds the cases, draw(rng) gives another one of the same ranges, prepare(case, seed) a
program's state, run(state) one pass, work(case) the bytes and operations a pass cannot do without,
and exact(case, seed) the same outputs in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-5
FP8_MAX = 448.0


def listed():
    return [
        # one user's next token: 12 heads of 64, a short cache, latency of a call
        {"name": "token, one sequence", "kind": "window", "B": 1, "TQ": 1, "TK": 1000, "NH": 12, "NKV": 12, "D": 64,
         "window": 512, "sinks": 4, "step": 0},
        # a serving batch of next tokens over long caches, four query heads to a key head
        {"name": "tokens, batch", "kind": "window", "B": 64, "TQ": 1, "TK": 8192, "NH": 16, "NKV": 4, "D": 128,
         "window": 4096, "sinks": 4, "step": 61},
        # prompts of several lengths behind caches of several lengths, nothing a multiple of a tile
        {"name": "prompts, ragged", "kind": "window", "B": 5, "TQ": 777, "TK": 1501, "NH": 12, "NKV": 4, "D": 64,
         "window": 300, "sinks": 5, "step": 131},
        # prefill of two long prompts, 128-wide heads
        {"name": "prompts, long", "kind": "window", "B": 2, "TQ": 8192, "TK": 8192, "NH": 16, "NKV": 16, "D": 128,
         "window": 2048, "sinks": 4, "step": 0},
        # a training step at the benchmark's sublayer shape
        {"name": "training", "kind": "window_train", "B": 8, "TQ": 2048, "TK": 2048, "NH": 12, "NKV": 12, "D": 64,
         "window": 512, "sinks": 4, "step": 0},
        # a training step on long documents, 128-wide heads, four query heads to a key head
        {"name": "training, wide", "kind": "window_train", "B": 2, "TQ": 4096, "TK": 4096, "NH": 16, "NKV": 4, "D": 128,
         "window": 1024, "sinks": 4, "step": 0},
        # rotary positions of a serving batch's next tokens, far into long contexts
        {"name": "rotary, tokens", "kind": "rotary", "B": 32, "T": 1, "NH": 16, "NKV": 4, "D": 128, "R": 128,
         "interleaved": False, "scaling": "parts", "start": 100000},
        # a training batch, a quarter of each head left unrotated, neighbours paired
        {"name": "rotary, part of the head", "kind": "rotary", "B": 8, "T": 2048, "NH": 12, "NKV": 12, "D": 64, "R": 48,
         "interleaved": True, "scaling": "none", "start": 0},
        # the gradient at the benchmark's long-context shape
        {"name": "rotary, gradient", "kind": "rotary_back", "B": 16, "T": 4096, "NH": 16, "NKV": 16, "D": 128, "R": 128,
         "interleaved": False, "scaling": "linear", "start": 0},
        # the norm before a sublayer, next tokens of seven sequences
        {"name": "norm, tokens", "kind": "norm", "rows": 7, "cols": 768},
        # a large prefill whose next product takes 8 bits
        {"name": "norm, 8 bits", "kind": "norm8", "rows": 16383, "cols": 4096, "group": 128},
        # the gradient at the benchmark's activation size
        {"name": "norm, gradient", "kind": "norm_back", "rows": 16384, "cols": 768},
    ]


MAX_FLOPS = 2.4e11                         # of the largest listed case
MAX_TRAIN = 2 * 16 * 4096 * 4096 * 128     # B * NH * T * T * D of the largest listed training step
MAX_CACHE = 64 * 8192 * 4 * 128            # elements of the largest listed cache
MAX_ROTARY = 16 * 4096 * 32 * 128
MAX_NORM = 16383 * 4096


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "window", "window_train", "window_train", "rotary", "rotary_back", "norm",
                       "norm8", "norm_back"])
    if kind in ("window", "window_train"):
        D = rng.choice([64, 128])
        NKV = rng.choice([1, 2, 3, 4, 8])
        NH = NKV * rng.choice([1, 2, 3, 4, 8])
        sinks = rng.choice([0, 1, 4, 5, 17, 33, 64])
        window = _log_int(rng, 16 if kind == "window_train" else 1, 4096)
        if kind == "window" and rng.random() < 0.4:
            TQ, TK = 1, _log_int(rng, 1, 8192)
            B = max(1, min(_log_int(rng, 1, 64), MAX_CACHE // (TK * NKV * D)))
        else:
            TK = _log_int(rng, 32 if kind == "window_train" else 1, 4096)
            TQ = TK if kind == "window_train" or rng.random() < 0.5 else rng.randint(1, TK)
            most = MAX_TRAIN if kind == "window_train" else 2 * MAX_TRAIN
            B = max(1, min(_log_int(rng, 1, 16), most // (NH * TK * TK * D)))
            while B == 1 and NH > NKV and NH * TK * TK * D > most:
                NH -= NKV
        step = rng.choice([0, 1, 63, 64, 129]) if B > 1 else 0
        case = {"kind": kind, "B": B, "TQ": TQ, "TK": TK, "NH": NH, "NKV": NKV, "D": D, "window": window, "sinks": sinks,
                "step": step}
        while work(case)["flops"] > MAX_FLOPS:
            case["window"] //= 2
        return case
    if kind in ("rotary", "rotary_back"):
        D = rng.choice([64, 128])
        NKV = rng.choice([1, 2, 3, 4, 8, 12])
        NH = NKV * rng.choice([1, 2, 4])
        T = _log_int(rng, 1, 8192)
        B = max(1, min(_log_int(rng, 1, 64), MAX_ROTARY // (T * (NH + NKV) * D)))
        R = 2 * rng.randint(1, D // 2) if rng.random() < 0.3 else 16 * rng.randint(1, D // 16)
        return {"kind": kind, "B": B, "T": T, "NH": NH, "NKV": NKV, "D": D, "R": R,
                "interleaved": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "parts"]),
                "start": rng.choice([0, _log_int(rng, 1, 1000000)])}
    cols = 8 * _log_int(rng, 1, 1024)
    rows = _log_int(rng, 1, max(2, min(65536, MAX_NORM // cols)))
    case = {"kind": kind, "rows": rows, "cols": cols}
    if kind == "norm8":
        case["group"] = rng.choice([0, 32, 64, 128])
    return case


# ---- what a pass cannot do without -------------------------------------------------------------

def _key_lengths(c):
    """Keys of each sequence: the capacity, less by `step` from one sequence to the next."""
    return [max(1, c["TK"] - b * c["step"]) for b in range(c["B"])]


def _query_lengths(c):
    """Query rows of each sequence; the first keeps all, where the keys run short so do the rows."""
    return [min(c["TQ"], n) for n in _key_lengths(c)]


def _pairs(c):
    """Visible (row, key) pairs of one head over all sequences, and the keys that some row sees."""
    pairs = keys = 0
    for lq, lk in zip(_query_lengths(c), _key_lengths(c)):
        pos = torch.arange(lk - lq, lk, dtype=torch.int64)
        inside = (pos + 1).clamp(max=c["window"])
        pairs += int((inside + (pos + 1 - inside).clamp(max=c["sinks"])).sum())
        first = max(0, lk - lq - c["window"] + 1)
        keys += lk - first + min(c["sinks"], first)
    return pairs, keys


def work(c):
    kind = c["kind"]
    if kind in ("window", "window_train"):
        pairs, keys = _pairs(c)
        rows = sum(_query_lengths(c))
        q = 2 * rows * c["NH"] * c["D"]
        kv = 2 * keys * c["NKV"] * c["D"]
        l = 4 * rows * c["NH"]
        if kind == "window":
            return {"bytes": 2 * q + 2 * kv + l, "flops": 4 * c["D"] * pairs * c["NH"]}
        # q, k, v, dO in; out, l, dQ, dK, dV out
        return {"bytes": 4 * q + 4 * kv + l, "flops": 14 * c["D"] * pairs * c["NH"]}
    if kind in ("rotary", "rotary_back"):
        n = c["B"] * c["T"] * (c["NH"] + c["NKV"])
        return {"bytes": 4 * n * c["D"] + 4 * c["B"] * c["T"], "flops": 3 * n * c["R"]}
    n = c["rows"] * c["cols"]
    if kind == "norm":
        return {"bytes": 8 * n + 2 * c["cols"] + 4 * c["rows"], "flops": 5 * n}
    if kind == "norm8":
        groups = -(-c["cols"] // c["group"]) if c["group"] else 1
        return {"bytes": 7 * n + 2 * c["cols"] + 4 * c["rows"] * (1 + groups), "flops": 8 * n}
    return {"bytes": 8 * n + 6 * c["cols"] + 4 * c["rows"], "flops": 9 * n}


# ---- a program's state -------------------------------------------------------------------------

def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(torch.bfloat16)

    def like(t, dtype=None):
        return torch.zeros_like(t, dtype=dtype or t.dtype)

    s = {"case": c}
    if c["kind"] in ("window", "window_train"):
        B, TQ, TK, D = c["B"], c["TQ"], c["TK"], c["D"]
        s["q"] = normal(B, TQ, c["NH"], D)
        s["k"] = normal(B, TK, c["NKV"], D)
        s["v"] = normal(B, TK, c["NKV"], D)
        s["q_len"] = torch.tensor(_query_lengths(c), dtype=torch.int32, device=dev)
        s["k_len"] = torch.tensor(_key_lengths(c), dtype=torch.int32, device=dev)
        s["out"] = like(s["q"])
        s["l"] = torch.zeros(B, c["NH"], TQ, dtype=torch.float32, device=dev)
        if c["kind"] == "window_train":
            s["dO"] = normal(B, TQ, c["NH"], D)
            s["dQ"], s["dK"], s["dV"] = like(s["q"]), like(s["k"]), like(s["v"])
    elif c["kind"] in ("rotary", "rotary_back"):
        B, T, D = c["B"], c["T"], c["D"]
        s["q"], s["k"] = normal(B, T, c["NH"], D), normal(B, T, c["NKV"], D)
        s["q_out"], s["k_out"] = like(s["q"]), like(s["k"])
        first = torch.randint(0, c["start"] + 1, (B, 1), generator=g, device=dev, dtype=torch.int32)
        s["positions"] = (first + torch.arange(T, device=dev, dtype=torch.int32)).contiguous()
    else:
        R, C = c["rows"], c["cols"]
        s["gamma"] = (1.0 + 0.1 * torch.randn(C, generator=g, device=dev)).to(torch.bfloat16)
        s["rstd"] = torch.zeros(R, dtype=torch.float32, device=dev)
        if c["kind"] == "norm_back":
            s["h"], s["dOut"], s["dSum"] = normal(R, C, scale=2.0), normal(R, C), normal(R, C)
            s["rstd"] = torch.rsqrt(s["h"].float().square().mean(-1) + EPS)
            s["dX"] = like(s["h"])
            s["dgamma"] = torch.zeros(C, dtype=torch.float32, device=dev)
        else:
            s["x"], s["residual"] = normal(R, C), normal(R, C, scale=2.0)
            s["sum"] = like(s["x"])
            s["out"] = like(s["x"])
            if c["kind"] == "norm8":
                s["out"] = torch.zeros(R, C, dtype=torch.float8_e4m3fn, device=dev)
                groups = -(-C // c["group"]) if c["group"] else 1
                s["scales"] = torch.zeros(R, groups, dtype=torch.float32, device=dev)
    return s


# ---- the plain form ----------------------------------------------------------------------------

def _visible(s):
    """[B, 1, 1, TQ, TK]: whether a row sees a key; [B, TQ]: whether it is a row of its sequence."""
    c = s["case"]
    i = torch.arange(c["TQ"], device="cuda")
    j = torch.arange(c["TK"], device="cuda")
    pos = (s["k_len"] - s["q_len"])[:, None] + i  # [B, TQ]
    row = i < s["q_len"][:, None]
    back = pos[:, :, None] - j
    see = (back >= 0) & ((back < c["window"]) | (j < c["sinks"])) & row[:, :, None]
    return see[:, None, None], row


def _heads(t, NKV):
    """[B, T, NH, D] -> fp32 [B, NKV, group, T, D]"""
    B, T, NH, D = t.shape
    return t.float().view(B, T, NKV, NH // NKV, D).permute(0, 2, 3, 1, 4).contiguous()


def _rows(t):
    """[B, NKV, group, T, D] -> [B, T, NH, D]"""
    B, NKV, G, T, D = t.shape
    return t.permute(0, 3, 1, 2, 4).reshape(B, T, NKV * G, D)


def _shared(a, b):
    """a [B, NKV, group, T, X] times b [B, NKV, X, Y] -> [B, NKV, group, T, Y]"""
    B, N, G, T, X = a.shape
    return torch.matmul(a.reshape(B, N, G * T, X), b).view(B, N, G, T, b.shape[-1])


def _grouped(a, b):
    """sum over the group and its rows: a, b [B, NKV, group, T, X / Y] -> [B, NKV, X, Y]"""
    B, N, G, T, X = a.shape
    return torch.matmul(a.reshape(B, N, G * T, X).transpose(-1, -2).contiguous(), b.reshape(B, N, G * T, b.shape[-1]))


def _plain_window(s):
    c = s["case"]
    NKV, scale = c["NKV"], 1.0 / math.sqrt(c["D"])
    see, row = _visible(s)
    q = _heads(s["q"], NKV)
    k, v = (s[n].float().permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))  # [B, NKV, TK, D]
    kt = k.transpose(-1, -2).contiguous()
    score = (_shared(q, kt) * scale).masked_fill(~see, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    some = total > 0
    p = torch.where(some, p / total, torch.zeros_like(p))
    out = _shared(p, v)
    l = torch.where(some, top + torch.log(total), torch.full_like(top, -math.inf)).squeeze(-1).flatten(1, 2)
    l = torch.where(row[:, None], l, torch.zeros_like(l))
    result = {"out": _rows(out).to(torch.bfloat16), "l": l}
    if c["kind"] == "window":
        return result
    dO = _heads(s["dO"], NKV)
    dO = torch.where(row[:, None, None, :, None], dO, torch.zeros_like(dO))
    dP = _shared(dO, v.transpose(-1, -2).contiguous())
    dS = p * (dP - (dO * out).sum(-1, keepdim=True)) * scale
    result["dQ"] = _rows(_shared(dS, k)).to(torch.bfloat16)
    result["dK"] = _grouped(dS, q).permute(0, 2, 1, 3).to(torch.bfloat16).contiguous()
    result["dV"] = _grouped(p, dO).permute(0, 2, 1, 3).to(torch.bfloat16).contiguous()
    return result


SCALING = {"none": {}, "linear": {"factor": 8.0},
           "parts": {"factor": 16.0, "original": 4096, "low": 1.0, "high": 32.0, "magnitude": 1.2}}
BASE = 10000.0


def _frequencies(c):
    """Radians per position of each pair, and the factor on the rotated values, in 64 bits."""
    f = BASE ** (-torch.arange(0, c["R"], 2, device="cuda", dtype=torch.float64) / c["R"])
    k = SCALING[c["scaling"]]
    if c["scaling"] == "linear":
        f = f / k["factor"]
    elif c["scaling"] == "parts":
        turns = k["original"] * f / (2 * math.pi)
        keep = ((turns - k["low"]) / (k["high"] - k["low"])).clamp(0, 1)
        f = f * keep + f / k["factor"] * (1 - keep)
    return f, k.get("magnitude", 1.0)


def _plain_rotary(s):
    c = s["case"]
    R = c["R"]
    f, m = _frequencies(c)
    angle = s["positions"].double()[..., None] * f
    cos, sin = ((t * m).float()[:, :, None] for t in (angle.cos(), angle.sin()))  # [B, T, 1, R/2]
    if c["kind"] == "rotary_back":
        sin = -sin

    def turned(x):
        y = x.float()
        if c["interleaved"]:
            a, b = y[..., 0:R:2], y[..., 1:R:2]
            z = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        else:
            a, b = y[..., :R // 2], y[..., R // 2:R]
            z = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        return torch.cat((z, y[..., R:]), -1).to(torch.bfloat16)

    return {"q": turned(s["q"]), "k": turned(s["k"])}


def _plain_norm(s):
    c = s["case"]
    gamma = s["gamma"].float()
    if c["kind"] == "norm_back":
        rstd = s["rstd"][:, None]
        x = s["h"].float() * rstd
        dy = s["dOut"].float()
        d = dy * gamma
        dX = s["dSum"].float() + rstd * (d - x * (d * x).mean(-1, keepdim=True))
        return {"dX": dX.to(torch.bfloat16), "dgamma": (dy * x).double().sum(0).float()}
    h = s["x"].float() + s["residual"].float()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    y = h * rstd * gamma
    result = {"sum": h.to(torch.bfloat16), "rstd": rstd[:, 0]}
    if c["kind"] == "norm":
        result["out"] = y.to(torch.bfloat16)
        return result
    group = c["group"] or c["cols"]
    R, C = y.shape
    parts = torch.nn.functional.pad(y, (0, -C % group)).view(R, -1, group)
    scale = parts.abs().amax(-1, keepdim=True) / FP8_MAX
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    q = (parts / scale).clamp(-FP8_MAX, FP8_MAX).view(R, -1)[:, :C]
    result["out"] = q.to(torch.float8_e4m3fn)
    result["scales"] = scale[..., 0].contiguous()
    return result


# ---- the package's entry points ----------------------------------------------------------------

def _own_window(s):
    import metalllm_amd.window as W
    c = s["case"]
    if "params" not in s:  # what a program sets up once for its buffers
        s["params"] = W.WindowParams.of(s["q"], s["k"], s["v"], s["out"], window=c["window"], sinks=c["sinks"])
        n = W.forward_workspace_bytes(s["params"])
        if c["kind"] == "window_train":
            n = max(n, W.backward_workspace_bytes(s["params"]))
        s["workspace"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    p, ws = s["params"], s["workspace"]
    W.windowAttentionForward(s["q"], s["k"], s["v"], s["out"], s["l"], s["q_len"], s["k_len"], ws, params=p)
    result = {"out": s["out"], "l": s["l"]}
    if c["kind"] == "window_train":
        W.windowAttentionBackward(s["dO"], s["out"], s["l"], s["q"], s["k"], s["v"], s["dQ"], s["dK"], s["dV"], s["q_len"],
                                  s["k_len"], ws, params=p)
        result.update(dQ=s["dQ"], dK=s["dK"], dV=s["dV"])
    return result


def _own_rotary(s):
    import metalllm_amd.rotary as R
    c = s["case"]
    if "plan" not in s:
        s["plan"] = R.RotaryPlan.of(c["R"], base=BASE, interleaved=c["interleaved"], scaling=c["scaling"],
                                    **SCALING[c["scaling"]])
    call = R.rotaryForward if c["kind"] == "rotary" else R.rotaryBackward
    call(s["q"], s["k"], s["q_out"], s["k_out"], s["positions"], s["plan"])
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_norm(s):
    import metalllm_amd.rmsnorm as N
    c = s["case"]
    if c["kind"] == "norm_back":
        if "workspace" not in s:
            s["workspace"] = torch.empty(N.backward_workspace_bytes(c["rows"], c["cols"]), dtype=torch.uint8, device="cuda")
        N.rmsnormBackward(s["dOut"], s["dSum"], s["h"], s["gamma"], s["rstd"], s["dX"], s["dgamma"], s["workspace"])
        return {"dX": s["dX"], "dgamma": s["dgamma"]}
    if c["kind"] == "norm":
        N.rmsnormForward(s["x"], s["residual"], s["sum"], s["out"], s["gamma"], s["rstd"], eps=EPS)
        return {"sum": s["sum"], "rstd": s["rstd"], "out": s["out"]}
    N.rmsnormForwardFp8(s["x"], s["residual"], s["sum"], s["out"], s["scales"], s["gamma"], s["rstd"], eps=EPS,
                        group=c["group"])
    return {"sum": s["sum"], "rstd": s["rstd"], "out": s["out"], "scales": s["scales"]}


def run(s):
    kind = s["case"]["kind"]
    if kind in ("window", "window_train"):
        return _own_window(s) if own else _plain_window(s)
    if kind in ("rotary", "rotary_back"):
        return _own_rotary(s) if own else _plain_rotary(s)
    return _own_norm(s) if own else _plain_norm(s)


# ---- 64 bits -----------------------------------------------------------------------------------

def _exact_window(c, s):
    B, TQ, TK, NH, NKV, D = (c[n] for n in ("B", "TQ", "TK", "NH", "NKV", "D"))
    train = c["kind"] == "window_train"
    opts = dict(dtype=torch.float64, device="cuda")
    r = {"out": torch.zeros(B, TQ, NH, D, **opts), "l": torch.zeros(B, NH, TQ, **opts)}
    if train:
        r.update(dQ=torch.zeros(B, TQ, NH, D, **opts), dK=torch.zeros(B, TK, NKV, D, **opts),
                 dV=torch.zeros(B, TK, NKV, D, **opts))
    root = math.sqrt(D)
    for b, (lq, lk) in enumerate(zip(_query_lengths(c), _key_lengths(c))):
        pos = torch.arange(lk - lq, lk, device="cuda").view(-1, 1)
        key = torch.arange(lk, device="cuda").view(1, -1)
        hidden = (key > pos) | ((key <= pos - c["window"]) & (key >= c["sinks"]))
        for h in range(NH):
            n = h // (NH // NKV)
            q, k, v = s["q"][b, :lq, h].double(), s["k"][b, :lk, n].double(), s["v"][b, :lk, n].double()
            x = torch.mm(q, k.t()) / root
            x[hidden] = -math.inf
            l = torch.logsumexp(x, 1)
            p = torch.exp(x - l[:, None])
            o = torch.mm(p, v)
            r["out"][b, :lq, h], r["l"][b, h, :lq] = o, l
            if train:
                g = s["dO"][b, :lq, h].double()
                r["dV"][b, :lk, n] += torch.mm(p.t(), g)
                d = torch.mm(g, v.t())
                d = p * (d - (p * d).sum(1, keepdim=True)) / root
                r["dQ"][b, :lq, h] = torch.mm(d, k)
                r["dK"][b, :lk, n] += torch.mm(d.t(), q)
    return r


def _exact_rotary(c, s):
    f, m = _frequencies(c)
    turn = torch.polar(torch.full_like(f, m).expand(*s["positions"].shape, -1).contiguous(),
                       s["positions"].double().unsqueeze(-1) * f)
    if c["kind"] == "rotary_back":
        turn = turn.conj()
    R, found = c["R"], {}
    for n in ("q", "k"):
        x = s[n].double()
        y = x.clone()
        first = slice(0, R, 2) if c["interleaved"] else slice(0, R // 2)
        second = slice(1, R, 2) if c["interleaved"] else slice(R // 2, R)
        z = torch.complex(x[..., first], x[..., second]) * turn[:, :, None]
        y[..., first], y[..., second] = z.real, z.imag
        found[n] = y
    return found


def _exact_norm(c, s):
    gamma = s["gamma"].double()
    if c["kind"] == "norm_back":
        h, dy, r = s["h"].double(), s["dOut"].double(), s["rstd"].double().unsqueeze(1)
        dh = dy * gamma * r - h * r ** 3 * (dy * gamma * h).sum(1, keepdim=True) / c["cols"]
        return {"dX": s["dSum"].double() + dh, "dgamma": (dy * h * r).sum(0)}
    h = s["x"].double() + s["residual"].double()
    r = 1 / torch.sqrt((h * h).sum(1) / c["cols"] + EPS)
    y = gamma * (h * r[:, None])
    found = {"sum": h, "rstd": r, "out": y}
    if c["kind"] == "norm8":
        group = c["group"] or c["cols"]
        scales = torch.stack([p.abs().max(1).values / FP8_MAX for p in y.split(group, 1)], 1)
        scales[scales == 0] = 1.0
        found["scales"] = scales
        found["out"] = y / scales.repeat_interleave(group, 1)[:, :c["cols"]]
    return found


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("window", "window_train"):
        return _exact_window(case, s)
    if case["kind"] in ("rotary", "rotary_back"):
        return _exact_rotary(case, s)
    return _exact_norm(case, s)
