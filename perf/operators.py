"""The operators of a mixture layer, and how they are timed: the router (``route``), the products grouped by expert
(``gmm``, with its gradients) and the microscaled 4-bit format (``mx4_quantize``, ``mm_mx4``).

Every case is a dict of plain values; ``kind`` names the operator.  Letters: T rows in E groups ("experts") of ragged
sizes, K contracted, N columns, k experts chosen per row.  ``tail`` rows stand behind the last group (a padded batch).
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 32  # values that share a scale in the 4-bit format
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- cases -----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of a serving call that went to two experts: latency, and two of the eight weight matrices
        {"name": "gmm one token", "kind": "gmm", "type": "bf16", "T": 2, "E": 8, "K": 1024, "N": 4096, "tail": 0, "layout": "kn"},
        # a decoding batch over many experts, a few rows each: every weight matrix once
        {"name": "gmm decode", "kind": "gmm", "type": "bf16", "T": 256, "E": 64, "K": 2048, "N": 1024, "tail": 0, "layout": "nk"},
        # prompts: thousands of rows per expert
        {"name": "gmm prompt", "kind": "gmm", "type": "bf16", "T": 16384, "E": 8, "K": 4096, "N": 4096, "tail": 0, "layout": "kn"},
        # odd sizes, and a batch padded behind its last group
        {"name": "gmm odd padded", "kind": "gmm", "type": "fp16", "T": 5001, "E": 5, "K": 1033, "N": 777, "tail": 130, "layout": "kn"},
        # fp32, the type of the framework's own products
        {"name": "gmm fp32", "kind": "gmm", "type": "fp32", "T": 4096, "E": 16, "K": 512, "N": 512, "tail": 0, "layout": "kn"},
        # a training step's two gradients
        {"name": "gmm_grad train", "kind": "gmm_grad", "type": "bf16", "T": 16384, "E": 16, "K": 2048, "N": 1024, "tail": 0, "layout": "kn"},
        # the same over few, odd and small matrices
        {"name": "gmm_grad odd", "kind": "gmm_grad", "type": "fp16", "T": 1000, "E": 3, "K": 257, "N": 130, "tail": 9, "layout": "nk"},
        # weights quantised when a model is loaded, and read back
        {"name": "mx4 weights", "kind": "mx4", "type": "bf16", "T": 16384, "K": 4096},
        # one token through 4-bit weights
        {"name": "mm_mx4 one token", "kind": "mm_mx4", "type": "bf16", "T": 1, "E": 0, "K": 4096, "N": 8192, "tail": 0},
        # prompts through 4-bit experts, their rows quantised on the way
        {"name": "mm_mx4 prompt", "kind": "mm_mx4", "type": "bf16", "T": 16384, "E": 8, "K": 4096, "N": 4096, "tail": 0},
        # the router of a decoding batch
        {"name": "route decode", "kind": "route", "type": "fp32", "T": 64, "E": 64, "k": 2, "normalize": True, "masked": 0.0, "grad": False},
        # the router of a training step, with its gradient
        {"name": "route train", "kind": "route", "type": "fp32", "T": 65536, "E": 128, "k": 8, "normalize": True, "masked": 0.05, "grad": True},
    ]


MOST_FLOPS = 2.0 * 16384 * 4096 * 4096  # of a drawn product
MOST_BYTES = 768e6


def _between(rng, lo, hi, multiple=1):
    """A whole number spread over [lo, hi] by its logarithm; a multiple of `multiple` where that is more than one."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v // multiple * multiple))


def draw(rng):
    kind = rng.choice(["gmm", "gmm", "gmm_grad", "mx4", "mm_mx4", "mm_mx4", "route"])
    if kind == "route":
        E = _between(rng, 4, 512)
        return {"kind": kind, "type": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "T": _between(rng, 1, 65536 * 128 // max(E, 128)), "E": E,
                "k": _between(rng, 1, min(E, 16)), "normalize": rng.random() < 0.6, "masked": rng.choice([0.0, 0.0, 0.1]), "grad": rng.random() < 0.5}
    if kind == "mx4":
        K = _between(rng, 16, 16384)
        return {"kind": kind, "type": rng.choice(["bf16", "fp16", "fp32"]), "T": _between(rng, 1, 16384 * 4096 // K), "K": K}
    multiple = rng.choice([1, 8, 64, 64])  # odd sizes, and those of models
    K, N = _between(rng, 64, 4096, multiple), _between(rng, 64, 8192, multiple)
    if kind == "mm_mx4":
        E = rng.choice([0, 0, _between(rng, 1, 32)])
        T = _between(rng, 1, 16384)
        while 2.0 * T * K * N > MOST_FLOPS or max(E, 1) * K * N > MOST_BYTES / 4:
            T, N = max(1, T // 2), max(32, N // 2)
        tail = rng.choice([0, 0, T // 9]) if E else 0
        return {"kind": kind, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "T": T, "E": E, "K": K, "N": N, "tail": tail}
    name = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    E, T = _between(rng, 1, 128), _between(rng, 1, 16384)
    cost = (3 if kind == "gmm_grad" else 1) * (8 if name == "fp32" else 1)
    while 2.0 * T * K * N * cost > MOST_FLOPS or E * K * N * SIZE[name] * (3 if kind == "gmm_grad" else 1) > MOST_BYTES:
        T, E, N = max(1, T * 2 // 3), max(1, E * 2 // 3), max(32, N * 2 // 3 // multiple * multiple)
    return {"kind": kind, "type": name, "T": T, "E": E, "K": K, "N": N, "tail": rng.choice([0, 0, T // 9]), "layout": rng.choice(["kn", "nk"])}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _counts(case, seed):
    """Rows of each expert: every row picks one, some experts more often than others."""
    g = torch.Generator().manual_seed(1000003 * seed + 17)
    p = torch.softmax(0.7 * torch.randn(case["E"], generator=g), dim=0)
    rows = case["T"] - case["tail"]
    if rows == 0:
        return [0] * case["E"]
    return torch.bincount(torch.multinomial(p, rows, replacement=True, generator=g), minlength=case["E"]).tolist()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device=dev, generator=g)  # noqa: E731
    dtype = TYPES[case["type"]]
    kind, state = case["kind"], dict(case)
    if kind == "route":
        x = 1.5 * normal(case["T"], case["E"])
        if case["masked"]:  # experts that a row may not choose; now and then (a padded row) all of them
            x[torch.rand(x.shape, device=dev, generator=g) < case["masked"]] = -math.inf
            x[torch.rand(case["T"], device=dev, generator=g) < case["masked"] / 4] = -math.inf
        state["x"], state["g"] = x.to(dtype), normal(case["T"], case["k"])
        return state
    if kind == "mx4":
        state["x"] = (normal(case["T"], case["K"]) * torch.exp(normal(case["T"], 1))).to(dtype)
        return state
    T, E, K, N = case["T"], case["E"], case["K"], case["N"]
    state["a"] = normal(T, K).to(dtype)
    if E:
        state["counts"] = _counts(case, seed)
        state["sizes"] = torch.tensor(state["counts"], dtype=torch.int32, device=dev)
    if kind == "mm_mx4":
        state["codes"], state["scales"] = _pack(normal(*((E,) if E else ()), N, K) * K ** -0.5)
        return state
    b = normal(E, K, N) if case["layout"] == "kn" else normal(E, N, K)
    b = (b * K ** -0.5).to(dtype)
    state["b"] = b if case["layout"] == "kn" else b.transpose(1, 2)
    if kind == "gmm_grad":
        state["g"] = normal(T, N).to(dtype)
    return state


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _power(e):
    """2^e in 64 bits, exactly: the exponent's bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantize(x):
    """(codes, exponents): E2M1 codes of the rows of x in blocks of 32, padded with zeros, and each block's scale 2^exponent."""
    K = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    e = (torch.frexp(x.abs().amax(-1))[1] - 3).clamp(-127, 127)  # the largest lies in [4, 8) then
    v = x.double() * _power(-e).unsqueeze(-1)
    u = v.abs()  # to the nearest value, ties to the even code
    code = (u > 0.25).to(torch.uint8) + (u >= 0.75) + (u > 1.25) + (u >= 1.75) + (u > 2.5) + (u >= 3.5) + (u > 5.0)
    return (code + 8 * torch.signbit(v)).to(torch.uint8), e


def _pack(x):
    """The stored form: two codes a byte, the even one in the low bits; exponents biased by 127."""
    codes, e = _quantize(x)
    codes = codes.flatten(-2).unflatten(-1, (-1, 2))
    return codes[..., 0] + 16 * codes[..., 1], (e + 127).to(torch.uint8)


def _unpack(codes, scales, K):
    both = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).unflatten(-1, (-1, BLOCK))
    return _value(both, scales.int() - 127)[..., :K]


def _value(code, e):
    """fp32 values of codes in blocks, each block under its own exponent."""
    v = torch.tensor(E2M1, device=code.device)[(code & 7).long()]
    return (torch.where(code >= 8, -v, v) * _power(e).float().unsqueeze(-1)).flatten(-2)


def _products(a, b, counts):
    """Rows of a in consecutive groups, each times its own matrix; zeros behind the last group."""
    behind = a.shape[0] - sum(counts)
    c = torch.cat([x @ w for x, w in zip(a.split(counts + [behind]), b)])
    return torch.nn.functional.pad(c, (0, 0, 0, behind))


def _route(s):
    x = s["x"].float()
    top, at = torch.sort(x, dim=1, descending=True, stable=True)
    top, at = top[:, :s["k"]], at[:, :s["k"]]
    e = torch.exp(top - top[:, :1]).where(top > -math.inf, 0.0)
    total = e if s["normalize"] else torch.exp(x - top[:, :1]).where(x > -math.inf, 0.0)
    total = total.sum(1, keepdim=True)
    weights = torch.where(total > 0, e / total, 0.0)
    experts = torch.where(top > -math.inf, at, -1)
    # places of the chosen pairs, by expert and then by row
    key = torch.where(experts < 0, s["E"], experts).flatten()
    order = torch.sort(key, stable=True)[1]
    chosen = key < s["E"]
    rows = torch.where(chosen[order], order // s["k"], 0)
    slots = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=x.device)).where(chosen, -1)
    sizes = torch.zeros(s["E"] + 1, dtype=torch.int32, device=x.device).index_add_(0, key, torch.ones_like(key, dtype=torch.int32))
    out = {"weights": weights, "experts": experts.int(), "rows": rows.int(), "slots": slots.view_as(experts).int(), "sizes": sizes[:-1]}
    if s["grad"]:
        inner = (s["g"] * weights).sum(1, keepdim=True)
        if s["normalize"]:
            d = torch.zeros_like(x).scatter_(1, at, weights * (s["g"] - inner))
        else:
            p = torch.where(total > 0, torch.exp(x - top[:, :1]) / total, 0.0).where(x > -math.inf, 0.0)
            d = (-p * inner).scatter_add_(1, at, weights * s["g"])
        out["grad"] = d.to(s["x"].dtype)
    return out


def _plain(s):
    kind = s["kind"]
    if kind == "route":
        return _route(s)
    if kind == "mx4":
        return _value(*_quantize(s["x"]))[..., :s["K"]].to(s["x"].dtype)
    a = s["a"].float()
    if kind == "mm_mx4":
        a = _value(*_quantize(a))[..., :s["K"]]
        b = _unpack(s["codes"], s["scales"], s["K"]).mT
        c = _products(a, b, s["counts"]) if s["E"] else a @ b
        return c.to(s["a"].dtype)
    if kind == "gmm":
        return _products(a, s["b"].float(), s["counts"]).to(s["a"].dtype)
    g = s["g"].float()
    da = _products(g, s["b"].float().mT, s["counts"])
    db = torch.stack([x.mT @ y for x, y in zip(a.split(s["counts"] + [s["T"] - sum(s["counts"])])[:-1], g.split(s["counts"] + [s["T"] - sum(s["counts"])]))])
    return da.to(s["a"].dtype), db.to(s["a"].dtype)


def run(state):
    if not own:
        return _plain(state)
    s, kind = state, state["kind"]
    if kind == "route":
        from triturus_amd.route import route, route_grad

        r = route(s["x"], s["k"], normalize=s["normalize"])
        out = {"weights": r.weights, "experts": r.experts, "rows": r.rows, "slots": r.slots, "sizes": r.sizes}
        if s["grad"]:
            out["grad"] = route_grad(s["g"], s["x"], r, normalize=s["normalize"])
        return out
    if kind == "gmm":
        from triturus_amd.gmm import gmm

        return gmm(s["a"], s["b"], s["sizes"])
    if kind == "gmm_grad":
        from triturus_amd.gmm import gmm_grad

        return gmm_grad(s["g"], s["a"], s["b"], s["sizes"])
    from triturus_amd.mx4 import MX4, mm_mx4, mx4_dequantize, mx4_quantize

    if kind == "mx4":
        return mx4_dequantize(mx4_quantize(s["x"]), dtype=s["x"].dtype)
    b = MX4(s["codes"], s["scales"], s["K"])
    return mm_mx4(s["a"], b, s["sizes"]) if s["E"] else mm_mx4(s["a"], b)


def work(case):
    T, size = case["T"], SIZE[case["type"]]
    if case["kind"] == "route":
        k, E = case["k"], case["E"]
        b = T * E * size + T * k * (4 + 4 + 4 + 4) + 4 * E
        return {"bytes": b + (T * k * 4 + T * E * size if case["grad"] else 0), "flops": 0}
    K = case["K"]
    if case["kind"] == "mx4":  # in, the 4-bit form out and in again, out
        return {"bytes": 2 * T * K * size + 2 * T * math.ceil(K / BLOCK) * 17, "flops": 0}
    N, rows = case["N"], T - case["tail"]
    used = min(case["E"], rows) if case["E"] else 1  # matrices that some row meets
    if case["kind"] == "mm_mx4":
        return {"bytes": (rows * K + T * N) * size + used * N * math.ceil(K / BLOCK) * 17, "flops": 2 * rows * K * N}
    if case["kind"] == "gmm":
        return {"bytes": (rows * K + T * N + used * K * N) * size, "flops": 2 * rows * K * N}
    return {"bytes": (rows * (K + N) + T * K + (used + case["E"]) * K * N) * size, "flops": 4 * rows * K * N}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def _exact_mx4(x):
    """Values of the 4-bit form of x: in each block of 32, multiples of a step that follows the value's own binade."""
    x, K = x.double(), x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    binades = torch.tensor([2.0 ** e for e in range(-125, 129)], dtype=torch.float64, device=x.device)  # exact, unlike log2 and exp2
    at = (torch.searchsorted(binades, x.abs().amax(-1, keepdim=True).contiguous(), right=True) - 1).clamp(min=0)
    scale = binades[at] / 4
    v = x / scale
    step = 0.5 + 0.5 * (v.abs() >= 2) + (v.abs() >= 4)
    return (scale * (torch.round(v / step) * step).clamp(-6.0, 6.0)).flatten(-2)[..., :K]


def _exact_route(s):
    x, T, E, k = s["x"].double(), s["T"], s["E"], s["k"]
    before = torch.arange(E, device=x.device)[:, None] < torch.arange(E, device=x.device)  # [j, i]: j stands before i
    at = torch.empty(T, k, dtype=torch.long, device=x.device)
    chunk = max(1, (1 << 27) // (E * E))
    for t in range(0, T, chunk):
        y = x[t:t + chunk]
        rank = ((y[:, :, None] > y[:, None, :]) | ((y[:, :, None] == y[:, None, :]) & before)).sum(1)
        at[t:t + chunk] = rank.argsort(1)[:, :k]
    top = x.gather(1, at)
    live = torch.isfinite(top)
    p = torch.zeros_like(x)
    among = torch.full_like(x, -math.inf).scatter(1, at, top) if s["normalize"] else x
    some = live[:, 0]
    p[some] = torch.softmax(among[some], dim=1)
    weights = p.gather(1, at) * live
    out = {"weights": weights, "experts": at.where(live, -1), "rows": None, "slots": None, "sizes": None}
    if s["grad"]:
        g = torch.zeros_like(x).scatter(1, at, s["g"].double() * live)
        out["grad"] = p * (g - (p * g).sum(1, keepdim=True))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(s)
    if case["kind"] == "mx4":
        return _exact_mx4(s["x"])
    if case["kind"] == "mm_mx4":
        a = _exact_mx4(s["a"])
        low, high = s["codes"] & 15, s["codes"] >> 4
        code = torch.stack((low, high), -1).flatten(-2).long()
        mantissa, e = (code & 1).double(), (code >> 1) & 3
        v = torch.where(e > 0, (1 + mantissa / 2) * torch.exp2(e.double() - 1), mantissa / 2) * (1 - 2 * (code >> 3)).double()
        b = (v * torch.pow(2.0, s["scales"].double() - 127).repeat_interleave(BLOCK, -1))[..., :case["K"]].transpose(-1, -2)
        if not case["E"]:
            return a @ b
    else:
        a, b = s["a"].double(), s["b"].double()
    group = torch.repeat_interleave(torch.arange(case["E"], device=a.device), s["sizes"].long())
    here = [group == e for e in range(case["E"])]
    n = group.numel()
    if case["kind"] != "gmm_grad":
        c = torch.zeros(case["T"], case["N"], dtype=torch.float64, device=a.device)
        for e, rows in enumerate(here):
            c[:n][rows] = a[:n][rows] @ b[e]
        return c
    g, da, db = s["g"].double(), torch.zeros_like(a), torch.zeros(b.shape, dtype=torch.float64, device=a.device)
    for e, rows in enumerate(here):
        da[:n][rows] = g[:n][rows] @ b[e].T
        db[e] = a[:n][rows].T @ g[:n][rows]
    return da, db
