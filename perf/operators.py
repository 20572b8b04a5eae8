"""The operators an engine runs beside the streamed units, as they are measured: the matrix product with its epilogue
(`linear`), the router's selection (`route`) and the gated feed-forward block of the units in their slots (`ffn`), each
with its backward pass. `own` False: elementary torch operations in 32 bits; True: the framework's calls."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the router's logits of one decoded token: the smallest product, all latency
        {"name": "linear_logits_1", "op": "linear", "rows": 1, "n": 128, "k": 4096, "type": "bf16", "act": "none",
         "bias": False, "residual": False},
        # a streamed dense layer's projection for a handful of decoded rows, everything in the epilogue
        {"name": "linear_dense_5", "op": "linear", "rows": 5, "n": 8192, "k": 8192, "type": "bf16", "act": "gelu",
         "bias": True, "residual": True},
        # the same for a prompt of odd length in the other type
        {"name": "linear_prompt_2047", "op": "linear", "rows": 2047, "n": 7168, "k": 4096, "type": "fp16",
         "act": "silu", "bias": True, "residual": True},
        # a training step's gradients of such a product
        {"name": "linear_back_4096", "op": "linear_back", "rows": 4096, "n": 4096, "k": 4096, "type": "bf16",
         "act": "gelu", "bias": True, "residual": False},
        # one decoded token's routing among 8 experts
        {"name": "route_1", "op": "route", "rows": 1, "experts": 8, "top": 2, "type": "fp32", "norm": True,
         "masked": 0.0},
        # a long prompt's routing among 256 experts, some of them closed to some tokens
        {"name": "route_8191", "op": "route", "rows": 8191, "experts": 256, "top": 8, "type": "fp32", "norm": True,
         "masked": 0.1},
        # the routing weights' gradient, softmax over all experts
        {"name": "route_back_4096", "op": "route_back", "rows": 4096, "experts": 128, "top": 8, "type": "bf16",
         "norm": False, "masked": 0.0},
        # one decoded token of the 8-expert top-2 model: the weights' bytes
        {"name": "ffn_decode_1", "op": "ffn", "rows": 1, "hidden": 4096, "ffn": 14336, "experts": 8, "top": 2,
         "type": "bf16", "act": "silu", "residual": True, "pad": 0},
        # a batch of decode streams of the 128-expert top-8 model, the last rows empty
        {"name": "ffn_decode_24", "op": "ffn", "rows": 24, "hidden": 4096, "ffn": 1536, "experts": 128, "top": 8,
         "type": "bf16", "act": "silu", "residual": True, "pad": 3},
        # its prompt of odd length: ragged groups of about a hundred rows
        {"name": "ffn_prompt_2047", "op": "ffn", "rows": 2047, "hidden": 4096, "ffn": 1536, "experts": 128, "top": 8,
         "type": "bf16", "act": "silu", "residual": False, "pad": 0},
        # gradients through frozen streamed units (adapters below them): no weight gradients
        {"name": "ffn_back_frozen_515", "op": "ffn_back", "rows": 515, "hidden": 2048, "ffn": 1408, "experts": 32,
         "top": 4, "type": "fp16", "act": "gelu", "units": False, "pad": 5},
        # a training step of the 8-expert top-2 model's layer, weight gradients included
        {"name": "ffn_back_1023", "op": "ffn_back", "rows": 1023, "hidden": 4096, "ffn": 14336, "experts": 8, "top": 2,
         "type": "bf16", "act": "silu", "units": True, "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_back", "route", "route_back", "ffn", "ffn", "ffn", "ffn_back"])
    act = rng.choice(["silu", "gelu", "gelu_tanh", "relu"])
    half = rng.choice(["bf16", "fp16"])
    if op in ("linear", "linear_back"):
        step = rng.choice([1, 8, 8, 64])  # rows of any length, of whole 16 bytes, of whole tiles
        return {"op": op, "rows": _log(rng, 1, 4096), "n": step * _log(rng, 8 / step + 1, 8192 // step),
                "k": step * _log(rng, 64 // step, 4096 // step), "type": half,
                "act": rng.choice(["none", act]), "bias": rng.random() < 0.5, "residual": op == "linear" and rng.random() < 0.5}
    if op in ("route", "route_back"):
        experts = _log(rng, 4, 512)
        return {"op": op, "rows": _log(rng, 1, 8192), "experts": experts, "top": rng.randint(1, min(16, experts)),
                "type": rng.choice(["fp32", "bf16", "fp16"]), "norm": rng.random() < 0.5,
                "masked": rng.choice([0.0, 0.2])}
    experts = _log(rng, 2, 64)
    case = {"op": op, "rows": _log(rng, 1, 2048), "hidden": 8 * _log(rng, 16, 512), "ffn": 8 * _log(rng, 16, 512),
            "experts": experts, "top": rng.randint(1, min(8, experts)), "type": half, "act": act}
    case.update({"residual": rng.random() < 0.5} if op == "ffn" else {"units": rng.random() < 0.5})
    case["pad"] = rng.randint(0, case["rows"] // 8)
    return case


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype) * scale


def _logits(g, case):
    """Logits whose experts differ in popularity, as trained routers' do; a masked expert is -inf."""
    rows, experts = case["rows"], case["experts"]
    x = _randn(g, rows, experts) + _randn(g, 1, experts, scale=0.7)
    if case.get("masked"):
        x.masked_fill_(torch.rand((rows, experts), generator=g, device="cuda") < case["masked"], -math.inf)
    return x


def prepare(case, seed):
    g = _gen(seed)
    rows, op = case["rows"], case["op"]
    t = TYPES[case["type"]]
    s = {"case": case}
    if op in ("linear", "linear_back"):
        n, k = case["n"], case["k"]
        s["x"] = _randn(g, rows, k, dtype=t)
        s["w"] = _randn(g, n, k, scale=k ** -0.5, dtype=t)
        s["bias"] = _randn(g, n, scale=0.1, dtype=t) if case["bias"] else None
        s["residual"] = _randn(g, rows, n, dtype=t) if case["residual"] else None
        if op == "linear_back":
            s["dy"] = _randn(g, rows, n, dtype=t)
            s["pre"] = None  # what the forward pass kept
            if case["act"] != "none":
                z = s["x"].float() @ s["w"].float().T
                s["pre"] = (z if s["bias"] is None else z + s["bias"].float()).to(t)
    elif op in ("route", "route_back"):
        s["logits"] = _logits(g, case).to(t)
        if op == "route_back":
            s["ids"], s["weights"] = _route(s["logits"], case["top"], case["norm"])
            s["dweights"] = _randn(g, rows, case["top"])
    else:
        d, f, e = case["hidden"], case["ffn"], case["experts"]
        slots = e + 3  # spare slots, and units in no order
        s["gate"] = _randn(g, slots, f, d, scale=d ** -0.5, dtype=t)
        s["up"] = _randn(g, slots, f, d, scale=d ** -0.5, dtype=t)
        s["down"] = _randn(g, slots, d, f, scale=f ** -0.5, dtype=t)
        s["slot_of"] = torch.randperm(slots, generator=g, device="cuda")[:e].to(torch.int32)
        s["x"] = _randn(g, rows, d, dtype=t)
        s["ids"], s["weights"] = _route(_logits(g, case), case["top"], True)
        if case["pad"]:
            s["ids"][rows - case["pad"]:] = -1
        if op == "ffn":
            s["residual"] = _randn(g, rows, d, dtype=t) if case["residual"] else None
        else:
            s["dy"] = _randn(g, rows, d, dtype=t)
    return s


# ---- the plain forms ----
def _act(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return torch.clamp(z, min=0) if act == "relu" else z


def _dact(z, act):
    if act == "silu":
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        p = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + p) + 0.5 * z * (1 - p * p) * c * (1 + 3 * 0.044715 * z * z)
    return (z > 0).to(z.dtype) if act == "relu" else torch.ones_like(z)


def _linear(s):
    c = s["case"]
    z = s["x"].float() @ s["w"].float().T
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _linear_back(s):
    c, t = s["case"], s["x"].dtype
    dz = s["dy"].float()
    if c["act"] != "none":
        dz = dz * _dact(s["pre"].float(), c["act"])
    out = {"dx": (dz @ s["w"].float()).to(t), "dw": (dz.T @ s["x"].float()).to(t)}
    if s["bias"] is not None:
        out["db"] = dz.sum(0).to(t)
    return out


def _route(logits, top, norm):
    z = logits.float()
    v, i = torch.sort(z, dim=1, descending=True, stable=True)  # equal logits: the lowest id first
    v, i = v[:, :top], i[:, :top]
    p = torch.exp(v - v[:, :1])
    p = p / (p if norm else torch.exp(z - v[:, :1])).sum(1, keepdim=True)
    shut = torch.isinf(v)
    return torch.where(shut, -1, i).to(torch.int32), torch.where(shut, 0, p)


def _route_back(s):
    z, ids, dw = s["logits"].float(), s["ids"].long(), s["dweights"]
    there = ids >= 0
    at = ids.clamp(min=0)
    if s["case"]["norm"]:
        p = s["weights"]
        d = torch.where(there, p * (dw - (p * dw).sum(1, keepdim=True)), 0)
        out = torch.zeros_like(z).scatter_add_(1, at, d)
    else:
        p = torch.exp(z - z.max(1, keepdim=True).values)
        p = p / p.sum(1, keepdim=True)
        full = torch.zeros_like(z).scatter_add_(1, at, torch.where(there, dw, 0))
        out = p * (full - (p * full).sum(1, keepdim=True))
    return out.to(s["logits"].dtype)


def _groups(s):
    """The (token, choice) pairs by expert: the experts met, and per pair its expert's place and its place in the group."""
    ids = s["ids"].reshape(-1).long()
    pair = torch.nonzero(ids >= 0).reshape(-1)
    e = ids[pair]
    order = torch.argsort(e, stable=True)
    pair, e = pair[order], e[order]
    met, place, count = torch.unique_consecutive(e, return_inverse=True, return_counts=True)
    first = torch.cumsum(count, 0) - count
    inside = torch.arange(pair.numel(), device=pair.device) - first[place]
    return met, place, inside, pair, int(count.max()) if pair.numel() else 0


def _ffn(s):
    c, x = s["case"], s["x"]
    met, place, inside, pair, most = _groups(s)
    y = torch.zeros_like(x, dtype=torch.float32) if s["residual"] is None else s["residual"].float()
    if most:
        token = pair // c["top"]
        slot = s["slot_of"].long()[met]
        a = x.new_zeros((met.numel(), most, c["hidden"]), dtype=torch.float32)
        a[place, inside] = x.float()[token]
        h = _act(a @ s["gate"][slot].float().mT, c["act"]) * (a @ s["up"][slot].float().mT)
        o = (h @ s["down"][slot].float().mT)[place, inside] * s["weights"].reshape(-1)[pair, None]
        rows = x.new_zeros((c["rows"] * c["top"], c["hidden"]), dtype=torch.float32)
        rows[pair] = o
        y = y + rows.view(c["rows"], c["top"], c["hidden"]).sum(1)
    return y.to(x.dtype)


def _ffn_back(s):
    c, x, t = s["case"], s["x"], s["x"].dtype
    met, place, inside, pair, most = _groups(s)
    pairs = c["rows"] * c["top"]
    dx_rows = x.new_zeros((pairs, c["hidden"]), dtype=torch.float32)
    dweights = x.new_zeros(pairs, dtype=torch.float32)
    out = {}
    if c["units"]:
        out = {"dgate": x.new_zeros((c["experts"], c["ffn"], c["hidden"])),
               "dup": x.new_zeros((c["experts"], c["ffn"], c["hidden"])),
               "ddown": x.new_zeros((c["experts"], c["hidden"], c["ffn"]))}
    if most:
        token = pair // c["top"]
        slot = s["slot_of"].long()[met]
        gate, up, down = (s[n][slot].float() for n in ("gate", "up", "down"))
        a = x.new_zeros((met.numel(), most, c["hidden"]), dtype=torch.float32)
        b, w = torch.zeros_like(a), a.new_zeros((met.numel(), most, 1))
        a[place, inside] = x.float()[token]
        b[place, inside] = s["dy"].float()[token]
        w[place, inside, 0] = s["weights"].reshape(-1)[pair]
        g, u = a @ gate.mT, a @ up.mT
        k = _act(g, c["act"])
        h, dh = k * u, b @ down
        dweights[pair] = (h * dh).sum(2)[place, inside]
        dg, du = w * dh * u * _dact(g, c["act"]), w * dh * k
        dx_rows[pair] = (dg @ gate + du @ up)[place, inside]
        if c["units"]:
            out["dgate"][met] = (dg.mT @ a).to(t)
            out["dup"][met] = (du.mT @ a).to(t)
            out["ddown"][met] = (b.mT @ (w * h)).to(t)
    out["dx"] = dx_rows.view(c["rows"], c["top"], c["hidden"]).sum(1).to(t)
    out["dweights"] = dweights.view(c["rows"], c["top"]).to(t)
    return out


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        if op == "linear":
            return _linear(s)
        if op == "linear_back":
            return _linear_back(s)
        if op == "route":
            ids, weights = _route(s["logits"], c["top"], c["norm"])
            return {"ids": ids, "weights": weights}
        return _route_back(s) if op == "route_back" else _ffn(s) if op == "ffn" else _ffn_back(s)
    from tierstream_b200 import ops
    if op == "linear":
        return ops.linear(s["x"], s["w"], bias=s["bias"], residual=s["residual"], act=c["act"])
    if op == "linear_back":
        dx, dw, db = ops.linear_backward(s["dy"], s["x"], s["w"], act=c["act"], pre=s["pre"],
                                         need=("x", "w", "bias") if c["bias"] else ("x", "w"))
        return {"dx": dx, "dw": dw, "db": db} if c["bias"] else {"dx": dx, "dw": dw}
    if op == "route":
        ids, weights = ops.route(s["logits"], c["top"], norm=c["norm"])
        return {"ids": ids, "weights": weights}
    if op == "route_back":
        return ops.route_backward(s["dweights"], s["logits"], s["ids"], s["weights"], norm=c["norm"])
    units = ops.Units(s["gate"], s["up"], s["down"], s["slot_of"])
    if op == "ffn":
        return ops.ffn(s["x"], s["ids"], s["weights"], units, act=c["act"], residual=s["residual"])
    g = ops.ffn_backward(s["dy"], s["x"], s["ids"], s["weights"], units, act=c["act"],
                         need=("x", "weights", "units") if c["units"] else ("x", "weights"))
    return {n: v for n, v in g.items() if v is not None}


def work(case):
    rows, op = case["rows"], case["op"]
    size = 4 if case["type"] == "fp32" else 2
    if op in ("linear", "linear_back"):
        n, k = case["n"], case["k"]
        extra = n * case["bias"] + rows * n * case["residual"]
        if op == "linear":
            return {"bytes": 2 * (rows * k + n * k + rows * n + extra), "flops": 2 * rows * n * k}
        pre = rows * n * (case["act"] != "none")
        return {"bytes": 2 * (2 * rows * k + 2 * n * k + rows * n + pre + extra), "flops": 4 * rows * n * k}
    if op in ("route", "route_back"):
        e, top = case["experts"], case["top"]
        if op == "route":
            return {"bytes": rows * (e * size + top * 8), "flops": 4 * rows * e}
        return {"bytes": rows * (2 * e * size + top * 12), "flops": 6 * rows * e}
    d, f, e, top = case["hidden"], case["ffn"], case["experts"], case["top"]
    live = rows - case["pad"]
    pairs = live * top
    met = e * (1 - (1 - top / e) ** live)  # experts met by that many tokens of uniform routes
    weights = 3 * met * d * f
    if op == "ffn":
        return {"bytes": 2 * (weights + rows * d * (2 + case["residual"])) + rows * top * 8, "flops": 6 * pairs * d * f}
    grads = 3 * e * d * f * case["units"]
    return {"bytes": 2 * (weights + grads + 3 * rows * d) + rows * top * 10,
            "flops": (16 if case["units"] else 10) * pairs * d * f}


# ---- from the definitions, in 64 bits ----
def _slope(z, act):
    """f(z) and f'(z) in 64 bits, through the normal distribution and tanh's own derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.relu(), (z > 0).double()
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p + z * p * (1 - p)
    if act == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    q = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    p = 1 / (1 + torch.exp(-2 * q))  # (1 + tanh q) / 2
    return z * p, p + z * 2 * p * (1 - p) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)


def exact(case, seed):
    s = prepare(dict(case), seed)
    op = case["op"]
    if op == "linear":
        z = torch.einsum("tk,nk->tn", s["x"].double(), s["w"].double())
        z = z if s["bias"] is None else z + s["bias"].double()
        y = _slope(z, case["act"])[0]
        return y if s["residual"] is None else y + s["residual"].double()
    if op == "linear_back":
        dz = s["dy"].double()
        if case["act"] != "none":
            dz = dz * _slope(s["pre"].double(), case["act"])[1]
        out = {"dx": torch.einsum("tn,nk->tk", dz, s["w"].double()), "dw": torch.einsum("tn,tk->nk", dz, s["x"].double())}
        if case["bias"]:
            out["db"] = dz.sum(0)
        return out
    if op == "route":
        z = s["logits"].double()
        ids, weights = [], []
        left = z.clone()
        for _ in range(case["top"]):
            best = left.max(1, keepdim=True).values
            at = torch.argmax((left == best).int(), 1, keepdim=True)  # the first of the equal ones
            shut = torch.isinf(best)
            ids.append(torch.where(shut, -1, at))
            weights.append(torch.where(shut, -math.inf, z.gather(1, at)))
            left.scatter_(1, at, -math.inf)
        v = torch.cat(weights, 1)
        over = torch.logsumexp(v if case["norm"] else z, 1, keepdim=True)
        return {"ids": torch.cat(ids, 1).to(torch.int32), "weights": torch.exp(v - over)}
    if op == "route_back":
        z = s["logits"].double().requires_grad_(True)
        there = s["ids"] >= 0
        v = torch.where(there, z.gather(1, s["ids"].long().clamp(min=0)), -math.inf)
        over = torch.logsumexp(v if case["norm"] else z, 1, keepdim=True)
        w = torch.where(there, torch.exp(v - over), 0)
        return torch.autograd.grad((w * s["dweights"].double()).sum(), z)[0]
    rows, top = case["rows"], case["top"]
    x, ids, w = s["x"].double(), s["ids"].long(), s["weights"].double()
    back = op == "ffn_back"
    if back:
        dy, dx, dw = s["dy"].double(), torch.zeros_like(x), torch.zeros_like(w)
        grads = {n: torch.zeros((case["experts"],) + s[n].shape[1:], dtype=torch.float64, device="cuda")
                 for n in (("gate", "up", "down") if case["units"] else ())}
    else:
        y = torch.zeros_like(x) if s["residual"] is None else s["residual"].double()
    for e in range(case["experts"]):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        if not t.numel():
            continue
        gate, up, down = (s[n][int(s["slot_of"][e])].double() for n in ("gate", "up", "down"))
        g, u = x[t] @ gate.T, x[t] @ up.T
        f, df = _slope(g, case["act"])
        if not back:
            y.index_add_(0, t, w[t, k, None] * ((f * u) @ down.T))
            continue
        dh = dy[t] @ down
        dw[t, k] = (dh * f * u).sum(1)
        dh = dh * w[t, k, None]
        dx.index_add_(0, t, (dh * u * df) @ gate + (dh * f) @ up)
        if grads:
            grads["gate"][e], grads["up"][e] = (dh * u * df).T @ x[t], (dh * f).T @ x[t]
            grads["down"][e] = dy[t].T @ (w[t, k, None] * f * u)
    if not back:
        return y
    return {"dx": dx, "dweights": dw, **{"d" + n: v for n, v in grads.items()}}
