"""The operators of a mixture-of-experts feed-forward layer, as measured.

Three operators and their gradients: `dense` (matrix product with bias,
activation and residual: the projections and the shared expert), `moe_route`
(scores to chosen experts and weights) and `moe_combine` (the experts' rows
back to one row per token). `run` computes them from elementary torch
operations, or, where `own` is true, by the calls of `cutile_b200.ops`.

Layouts are those of `cutile_b200.ops`: a weight is the torch tensor
`A_t` (K, M), activations are `B_t` (N, K), one row per token, and the product
is (N, M).
"""
import math
import os
import sys

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_INF = float("inf")


# ---- cases --------------------------------------------------------------------
def _dense(name, n, m, k, dtype, act, bias=True, residual=False, preact=False):
    return {"name": name, "op": "dense", "n": n, "m": m, "k": k, "dtype": dtype, "act": act,
            "bias": bias, "residual": residual, "preact": preact}


def _route(name, t, e, topk, dtype, score, bias, groups, topk_groups, group_top, renorm, scale, pad):
    return {"name": name, "op": "route", "t": t, "e": e, "topk": topk, "dtype": dtype,
            "score": score, "bias": bias, "groups": groups, "topk_groups": topk_groups,
            "group_top": group_top, "renorm": renorm, "scale": scale, "pad": pad}


def listed():
    return [
        # one token of one request through a projection: the weight is read once, latency counts
        _dense("dense one token", 1, 4096, 4096, "f16", "silu"),
        # one token each of 37 requests through the wide projection of a feed-forward layer
        _dense("dense batch of tokens", 37, 14336, 4096, "bf16", "gelu_tanh"),
        # a ragged layer: no stride is a multiple of 16 bytes
        _dense("dense ragged", 777, 1001, 1003, "f16", "relu", residual=True),
        # a prompt through the narrow projection, added to the residual stream
        _dense("dense prompt", 2049, 4096, 14336, "f16", "none", residual=True),
        # training: the wide projection, its value before the activation kept for the gradient
        _dense("dense training", 8192, 14336, 4096, "bf16", "gelu", preact=True),
        # the gradients of a square layer
        {"name": "dense gradients", "op": "dense_bwd", "n": 8192, "m": 4096, "k": 4096,
         "dtype": "bf16", "act": "gelu", "bias": True},
        # one token to 2 of 8 experts
        _route("route one token", 1, 8, 2, "bf16", "softmax", False, 1, 1, 2, True, 1.0, 0),
        # a long prompt to 8 of 256 experts in 4 of 8 groups, balanced by a bias; a padded tail
        _route("route prompt", 16384, 256, 8, "f32", "sigmoid", True, 8, 4, 2, True, 2.5, 100),
        # the gradient of the scores of a training batch
        {"name": "route gradients", "op": "route_bwd", "t": 16384, "e": 64, "topk": 6,
         "dtype": "f32", "score": "softmax", "renorm": False, "scale": 1.0},
        # one token's 8 expert rows back to one
        {"name": "combine one token", "op": "combine", "t": 1, "topk": 8, "n": 4096,
         "dtype": "f16", "weights": True, "residual": True, "drop": 0.0},
        # a training batch, top 2 of 8 experts, with the residual stream; some slots dropped
        {"name": "combine batch", "op": "combine", "t": 16384, "topk": 2, "n": 4096,
         "dtype": "f16", "weights": True, "residual": True, "drop": 0.01},
        # the gradients of the experts' rows and of the weights of an odd batch
        {"name": "combine gradients", "op": "combine_bwd", "t": 4099, "topk": 8, "n": 2048,
         "dtype": "bf16", "weights": True, "drop": 0.01},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: mostly whole 16-byte rows, one in six any number."""
    w = _log_int(rng, lo, hi)
    return w if rng.random() < 1 / 6 else max(8, w // 8 * 8)


def draw(rng):
    op = rng.choice(["dense", "dense", "dense", "dense_bwd", "dense_bwd", "route", "route",
                     "route_bwd", "combine", "combine_bwd"])
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    dtype = rng.choice(["f16", "bf16"])
    if op in ("dense", "dense_bwd"):
        n = _log_int(rng, 1, 8192) if op == "dense" else _log_int(rng, 16, 8192)
        m, k = _width(rng, 64, 14336), _width(rng, 64, 8192)
        if op == "dense":
            c = _dense(None, n, m, k, dtype, act, rng.random() < 0.7, rng.random() < 0.5,
                       rng.random() < 0.3)
            del c["name"]
            return c
        return {"op": op, "n": n, "m": min(m, 8192), "k": min(k, 4096), "dtype": dtype,
                "act": act, "bias": rng.random() < 0.7}
    if op in ("route", "route_bwd"):
        t = _log_int(rng, 1, 16384)
        groups = rng.choice([1, 1, 2, 4, 8])
        e = groups * _log_int(rng, 4, 256 // groups)
        topk = rng.randint(1, min(8, e // groups))
        dt = rng.choice(["f16", "bf16", "f32"])
        score = rng.choice(["softmax", "sigmoid"])
        renorm = rng.random() < 0.6
        scale = rng.choice([1.0, 2.5])
        if op == "route_bwd":
            return {"op": op, "t": t, "e": e, "topk": topk, "dtype": dt, "score": score,
                    "renorm": renorm, "scale": scale}
        c = _route(None, t, e, topk, dt, score, rng.random() < 0.5, groups,
                   rng.randint(1, groups), rng.choice([1, 2]), renorm, scale,
                   t // 50 if rng.random() < 0.5 else 0)
        del c["name"]
        return c
    topk = rng.randint(1, 8)
    c = {"op": op, "t": _log_int(rng, 1, 32768 // topk), "topk": topk, "n": _width(rng, 64, 4096),
         "dtype": dtype, "weights": rng.random() < 0.8, "drop": rng.choice([0.0, 0.01])}
    if op == "combine":
        c["residual"] = rng.random() < 0.5
    return c


# ---- inputs -------------------------------------------------------------------
def _normal(g, shape, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _some_ids(g, t, e, topk):
    """Distinct experts per row, best first, as a router gives them."""
    return torch.rand((t, e), generator=g, device="cuda").argsort(-1)[:, :topk].to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    dt = _DT[case["dtype"]]
    if op in ("dense", "dense_bwd"):
        n, m, k = case["n"], case["m"], case["k"]
        s["A"] = _normal(g, (k, m), dt, 1 / math.sqrt(k))
        s["B"] = _normal(g, (n, k), dt)
        if op == "dense":
            s["b"] = _normal(g, (m,), torch.float32, 0.5) if case["bias"] else None
            s["R"] = _normal(g, (n, m), dt) if case["residual"] else None
        else:
            s["dC"] = _normal(g, (n, m), dt, 0.1)
            s["Z"] = _normal(g, (n, m), dt) if case["act"] != "none" else None
    elif op == "route":
        x = _normal(g, (case["t"], case["e"]), torch.float32, 1.5)
        if case["pad"]:
            x[-case["pad"]:] = -_INF  # tokens of the padding: no expert
        s["x"] = x.to(dt)
        s["rb"] = _normal(g, (case["e"],), torch.float32, 0.1) if case["bias"] else None
    elif op == "route_bwd":
        s["x"] = _normal(g, (case["t"], case["e"]), dt, 1.5)
        s["ids"] = _some_ids(g, case["t"], case["e"], case["topk"])
        s["dw"] = _normal(g, (case["t"], case["topk"]))
    else:
        t, topk, n = case["t"], case["topk"], case["n"]
        s["e"] = 64
        s["ids"] = _some_ids(g, t, 64, topk)
        s["y"] = _normal(g, (t * topk, n), dt)
        if case["drop"]:  # slots that no expert took: their rows were never written
            lost = torch.rand((t, topk), generator=g, device="cuda") < case["drop"]
            s["ids"][lost] = -1
            s["y"][lost.reshape(-1)] = float("nan")
        s["w"] = torch.rand((t, topk), generator=g, device="cuda") if case["weights"] else None
        if op == "combine":
            s["R"] = _normal(g, (t, n), dt) if case["residual"] else None
        else:
            s["dout"] = _normal(g, (t, n), dt)
    return s


# ---- plain forms --------------------------------------------------------------
def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    if act == "gelu_tanh":
        u = math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)
        return 0.5 * z * (1 + torch.tanh(u))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        pdf = torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
        return 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * pdf
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_dense(s):
    z = s["B"].float() @ s["A"].float()
    if s["b"] is not None:
        z = z + s["b"]
    y = _act(z, s["act"])
    if s["R"] is not None:
        y = y + s["R"].float()
    dt = s["B"].dtype
    return (y.to(dt), z.to(dt)) if s["preact"] else y.to(dt)


def _plain_dense_bwd(s):
    dz = s["dC"].float()
    if s["Z"] is not None:
        dz = dz * _act_slope(s["Z"].float(), s["act"])
    dt = s["B"].dtype
    dA = (s["B"].float().t() @ dz).to(dt)
    dB = (dz @ s["A"].float().t()).to(dt)
    return (dA, dB, dz.sum(0)) if s["bias"] else (dA, dB)


def _plain_route(s):
    """Choice scores in 64 bits: two that differ by less than 32 bits resolve
    must still be told apart; equal ones go to the lowest index."""
    x = s["x"].double()
    t, e = x.shape
    x = torch.where(x == x, x, -_INF)
    live = x > -_INF
    top = x.amax(-1, keepdim=True)
    top = torch.where(top > -_INF, top, torch.zeros_like(top))
    if s["score"] == "softmax":
        p = torch.exp(x - top)
        total = p.sum(-1, keepdim=True)
        score = p / torch.where(total > 0, total, torch.ones_like(total))
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = score if s["rb"] is None else score + s["rb"].double()
    live = live & (choice > -_INF)
    order = x if s["rb"] is None else choice  # scores rise with their logits
    order = torch.where(live, order, -_INF)
    g = s["groups"]
    if s["topk_groups"] < g:
        c = torch.where(live, choice, -_INF).reshape(t, g, e // g)
        best = torch.sort(c, dim=-1, descending=True).values[..., :min(s["group_top"], e // g)]
        of_group = torch.where(best[..., :1] > -_INF,
                               torch.where(best > -_INF, best, torch.zeros_like(best)).sum(-1, keepdim=True),
                               -_INF).squeeze(-1)
        chosen = torch.sort(of_group, dim=-1, descending=True, stable=True).indices[:, :s["topk_groups"]]
        in_group = torch.zeros((t, g), dtype=torch.bool, device=x.device).scatter_(1, chosen, True)
        order = torch.where(in_group.repeat_interleave(e // g, 1), order, -_INF)
    best, ids = torch.sort(order, dim=-1, descending=True, stable=True)
    best, ids = best[:, :s["topk"]], ids[:, :s["topk"]]
    taken = best > -_INF
    if s["renorm"]:
        xs = torch.where(taken, torch.gather(x, 1, ids), -_INF)
        m = xs.amax(-1, keepdim=True)
        m = torch.where(m > -_INF, m, torch.zeros_like(m))
        if s["score"] == "softmax":
            v = torch.exp(xs - m)
        else:  # sigmoid(x) * exp(-min(m, 0)): the common factor drops out of the shares
            v = torch.exp(xs - m.clamp(max=0) - xs.clamp(min=0)) / (1 + torch.exp(-xs.abs()))
        total = v.sum(-1, keepdim=True)
        w = v / torch.where(total > 0, total, torch.ones_like(total))
    else:
        w = torch.gather(score, 1, ids)
    w = torch.where(taken, w * s["scale"], torch.zeros_like(w))
    return w.float(), torch.where(taken, ids, -1).to(torch.int32)


def _plain_route_bwd(s):
    x = s["x"].float()
    ids = s["ids"].long()
    xs = torch.gather(x, 1, ids)
    g = s["dw"] * s["scale"]
    if s["renorm"]:
        if s["score"] == "softmax":
            v = torch.exp(xs - xs.amax(-1, keepdim=True))
            p = v / v.sum(-1, keepdim=True)
            d = p * (g - (g * p).sum(-1, keepdim=True))
        else:
            v = 1 / (1 + torch.exp(-xs))
            p = v / v.sum(-1, keepdim=True)
            d = p * (g - (g * p).sum(-1, keepdim=True)) / (1 + torch.exp(xs))
        return torch.zeros_like(x).scatter_add_(1, ids, d).to(s["x"].dtype)
    if s["score"] == "sigmoid":
        v = 1 / (1 + torch.exp(-xs))
        return torch.zeros_like(x).scatter_add_(1, ids, g * v * (1 - v)).to(s["x"].dtype)
    v = torch.exp(x - x.amax(-1, keepdim=True))
    p = v / v.sum(-1, keepdim=True)
    ps = torch.gather(p, 1, ids)
    dx = -p * (g * ps).sum(-1, keepdim=True)
    return dx.scatter_add_(1, ids, g * ps).to(s["x"].dtype)


def _plain_combine(s):
    t, topk = s["ids"].shape
    y = s["y"].float().reshape(t, topk, -1)
    used = ((s["ids"] >= 0) & (s["ids"] < s["e"])).unsqueeze(-1)
    if s["w"] is not None:
        y = y * s["w"].unsqueeze(-1)
    out = torch.where(used, y, torch.zeros_like(y)).sum(1)
    if s["R"] is not None:
        out = out + s["R"].float()
    return out.to(s["y"].dtype)


def _plain_combine_bwd(s):
    t, topk = s["ids"].shape
    used = ((s["ids"] >= 0) & (s["ids"] < s["e"])).unsqueeze(-1)
    d = s["dout"].float().unsqueeze(1)
    y = s["y"].float().reshape(t, topk, -1)
    if s["w"] is None:
        dy = torch.where(used, d, torch.zeros_like(y))
        return dy.to(s["y"].dtype).reshape(t * topk, -1)
    dy = torch.where(used, d * s["w"].unsqueeze(-1), torch.zeros_like(y))
    dw = torch.where(used, d * y, torch.zeros_like(y)).sum(-1)
    return dy.to(s["y"].dtype).reshape(t * topk, -1), dw


_PLAIN = {"dense": _plain_dense, "dense_bwd": _plain_dense_bwd, "route": _plain_route,
          "route_bwd": _plain_route_bwd, "combine": _plain_combine,
          "combine_bwd": _plain_combine_bwd}

_ops = None


def _own_ops():
    global _ops
    if _ops is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "cutile-triton_b200"))
        from cutile_b200 import ops

        _ops = ops
    return _ops


def run(s):
    op = s["op"]
    if not own:
        return _PLAIN[op](s)
    ops = _own_ops()
    if op == "dense":
        if s["preact"]:
            z = torch.empty((s["n"], s["m"]), dtype=s["B"].dtype, device="cuda")
            return ops.dense(s["A"], s["B"], bias=s["b"], act=s["act"], residual=s["R"], preact=z), z
        return ops.dense(s["A"], s["B"], bias=s["b"], act=s["act"], residual=s["R"])
    if op == "dense_bwd":
        dA, dB, db = ops.dense_bwd(s["dC"], s["A"], s["B"], act=s["act"], preact=s["Z"],
                                   need_dbias=s["bias"])
        return (dA, dB, db) if s["bias"] else (dA, dB)
    if op == "route":
        return ops.moe_route(s["x"], s["topk"], score=s["score"], bias=s["rb"],
                             groups=s["groups"], topk_groups=s["topk_groups"],
                             group_top=s["group_top"], renorm=s["renorm"], scale=s["scale"])
    if op == "route_bwd":
        return ops.moe_route_bwd(s["dw"], s["x"], s["ids"], score=s["score"], renorm=s["renorm"],
                                 scale=s["scale"])
    if op == "combine":
        return ops.moe_combine(s["y"], s["topk"], weights=s["w"], ids=s["ids"],
                               num_experts=s["e"], residual=s["R"])
    dy, dw = ops.moe_combine_bwd(s["dout"], s["y"], s["topk"], weights=s["w"], ids=s["ids"],
                                 num_experts=s["e"])
    return dy if s["w"] is None else (dy, dw)


# ---- what a pass cannot do without ------------------------------------------------
def work(case):
    op, es = case["op"], {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]]
    if op == "dense":
        n, m, k = case["n"], case["m"], case["k"]
        outs = 1 + case["residual"] + case["preact"]
        return {"bytes": es * (m * k + n * k + outs * n * m) + 4 * m * case["bias"],
                "flops": 2 * n * m * k}
    if op == "dense_bwd":
        n, m, k = case["n"], case["m"], case["k"]
        ins = 1 if case["act"] == "none" else 2
        return {"bytes": es * (2 * m * k + 2 * n * k + ins * n * m) + 4 * m * case["bias"],
                "flops": 4 * n * m * k}
    if op in ("route", "route_bwd"):
        t, e, k = case["t"], case["e"], case["topk"]
        if op == "route":
            return {"bytes": es * t * e + 8 * t * k + 4 * e * case["bias"], "flops": 8 * t * e}
        whole = case["score"] == "softmax" and not case["renorm"]
        return {"bytes": es * t * (e + (e if whole else k)) + 8 * t * k, "flops": 8 * t * e}
    t, k, n = case["t"], case["topk"], case["n"]
    if op == "combine":
        return {"bytes": es * t * n * (k + 1 + case["residual"]) + t * k * (4 + 4 * case["weights"]),
                "flops": 2 * t * k * n}
    reads = (k if case["weights"] else 0) + 1
    return {"bytes": es * t * n * (k + reads) + t * k * (4 + 8 * case["weights"]),
            "flops": (4 if case["weights"] else 1) * t * k * n}


# ---- the definitions in 64 bits -----------------------------------------------------
def _cdf(z):
    return torch.special.ndtr(z)


def _exact_act(z, act):
    """(value, slope) of an activation."""
    if act == "relu":
        return z.clamp(min=0), torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
    if act == "silu":
        sg = torch.sigmoid(z)
        return z * sg, sg + z * sg * torch.sigmoid(-z)
    if act == "gelu":
        return z * _cdf(z), _cdf(z) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":  # 0.5 (1 + tanh(u)) is the logistic function of 2 u
        a = 2 * math.sqrt(2 / math.pi)
        sg = torch.sigmoid(a * (z + 0.044715 * z.pow(3)))
        return z * sg, sg + z * sg * (1 - sg) * a * (1 + 0.134145 * z.square())
    return z, torch.ones_like(z)


def _exact_route(s):
    x = s["x"].double().nan_to_num(nan=-_INF, posinf=_INF, neginf=-_INF)
    t, e = x.shape
    logp = torch.log_softmax(x, -1) if s["score"] == "softmax" else torch.nn.functional.logsigmoid(x)
    logp = logp.nan_to_num(nan=-_INF, posinf=_INF, neginf=-_INF)
    choice = logp.exp()
    if s["rb"] is not None:
        choice = choice + s["rb"].double()
    rank = (x if s["rb"] is None else choice).masked_fill(x == -_INF, -_INF)
    if s["topk_groups"] < s["groups"]:
        size = e // s["groups"]
        best = choice.masked_fill(x == -_INF, 0.0).view(t, s["groups"], size)
        best = best.topk(min(s["group_top"], size), -1).values.sum(-1)
        cut = best.topk(s["topk_groups"], -1).values[:, -1:]
        rank = rank.masked_fill((best < cut).repeat_interleave(size, 1), -_INF)
    top = rank.topk(s["topk"], -1)
    lw = logp.gather(1, top.indices).masked_fill(top.values == -_INF, -_INF)
    if s["renorm"]:
        lw = torch.log_softmax(lw, -1).nan_to_num(nan=-_INF, neginf=-_INF)
    return lw.exp() * s["scale"], None


def _exact_route_bwd(s):
    x = s["x"].double().requires_grad_(True)
    logp = torch.log_softmax(x, -1) if s["score"] == "softmax" else torch.nn.functional.logsigmoid(x)
    lw = logp.gather(1, s["ids"].long())
    if s["renorm"]:
        lw = torch.log_softmax(lw, -1)
    return torch.autograd.grad(lw.exp() * s["scale"], x, s["dw"].double())[0]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "dense":
        z = torch.mm(s["B"].double(), s["A"].double())
        if s["b"] is not None:
            z += s["b"].double()
        y = _exact_act(z, case["act"])[0]
        if s["R"] is not None:
            y = y + s["R"].double()
        return (y, z) if case["preact"] else y
    if op == "dense_bwd":
        dz = s["dC"].double()
        if s["Z"] is not None:
            dz = dz * _exact_act(s["Z"].double(), case["act"])[1]
        dA = torch.mm(s["B"].double().t(), dz)
        dB = torch.mm(dz, s["A"].double().t())
        return (dA, dB, dz.sum(0)) if case["bias"] else (dA, dB)
    if op == "route":
        return _exact_route(s)
    if op == "route_bwd":
        return _exact_route_bwd(s)
    t, topk = s["ids"].shape
    y = s["y"].double().nan_to_num(nan=0.0).view(t, topk, -1)
    w = torch.ones((t, topk), dtype=torch.float64, device="cuda") if s["w"] is None else s["w"].double()
    w = w * (s["ids"] >= 0)
    if op == "combine":
        out = torch.einsum("tk,tkn->tn", w, y)
        return out if s["R"] is None else out + s["R"].double()
    d = s["dout"].double()
    dy = torch.einsum("tk,tn->tkn", w, d).reshape(t * topk, -1)
    return dy if s["w"] is None else (dy, torch.einsum("tkn,tn->tk", y, d))
