"""Workloads of the dense operators in ``flyvec_b200.ops``: layer norm, the matrix product with its
epilogue, and the log probabilities of given tokens, each with its backward pass.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes the inputs
of one on the GPU and ``run`` makes one pass: with ``own`` false from elementary torch operations in
32 bits, with ``own`` true through the framework's calls.  ``exact`` is the definition in 64 bits and
``work`` what a pass cannot do without.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
EPS = 1e-5


def listed():
    return [
        # one word's dense embedding (400 units) standardised before it is compared with others
        {"name": "norm one row", "op": "norm", "rows": 1, "cols": 400, "dtype": "float32", "affine": True, "pad": 0},
        # a training batch of wide hidden states
        {"name": "norm batch", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bfloat16", "affine": True, "pad": 0},
        # gradients of a small ragged batch of 1000-unit embeddings beside one more feature
        {"name": "norm grad odd", "op": "norm_grad", "rows": 1237, "cols": 1001, "dtype": "float32", "affine": True, "pad": 0},
        # gradients of a training batch of wide hidden states
        {"name": "norm grad batch", "op": "norm_grad", "rows": 16384, "cols": 4096, "dtype": "bfloat16", "affine": True, "pad": 0},
        # one word against the whole vocabulary of 20000: the product that answers a single query
        {"name": "linear one row", "op": "linear", "rows": 1, "inner": 400, "outer": 20000, "dtype": "bfloat16", "out": "float32",
         "act": "none", "bias": True, "residual": False, "keep": False, "pad": 0, "flip": False},
        # a wide hidden layer over a training batch, everything in the epilogue, pre-activation kept
        {"name": "linear batch", "op": "linear", "rows": 8192, "inner": 2048, "outer": 8192, "dtype": "bfloat16", "out": "bfloat16",
         "act": "gelu", "bias": True, "residual": True, "keep": True, "pad": 0, "flip": False},
        # gradients at odd sizes: no row starts on a 16-byte boundary
        {"name": "linear grad odd", "op": "linear_grad", "rows": 777, "inner": 501, "outer": 1003, "dtype": "float16", "act": "silu",
         "pad": 0, "flip": False},
        # gradients of a hidden layer over a training batch
        {"name": "linear grad batch", "op": "linear_grad", "rows": 16384, "inner": 1024, "outer": 4096, "dtype": "bfloat16", "act": "gelu",
         "pad": 0, "flip": False},
        # one query answered: the vocabulary's scores, the 20 best words
        {"name": "log probs one row", "op": "log_probs", "rows": 1, "vocab": 20000, "dtype": "float32", "beta": 1.0, "top": 20,
         "masked": 0.0, "pad": 0},
        # a step's 10000 windows scored over 20000 words, a twentieth of the words masked, 10 best
        {"name": "log probs batch", "op": "log_probs", "rows": 10000, "vocab": 20000, "dtype": "bfloat16", "beta": 1.0, "top": 10,
         "masked": 0.05, "pad": 0},
        # gradient of a few rows over a vocabulary of odd size
        {"name": "log probs grad odd", "op": "log_probs_grad", "rows": 37, "vocab": 50001, "dtype": "float32", "beta": 0.7,
         "masked": 0.05, "entropy": True, "pad": 0},
        # gradient of a training batch over 50000 words
        {"name": "log probs grad batch", "op": "log_probs_grad", "rows": 4096, "vocab": 50000, "dtype": "bfloat16", "beta": 1.0,
         "masked": 0.0, "entropy": True, "pad": 0},
    ]


def _span(rng, low, high):
    """A whole number spread evenly over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "linear", "linear_grad", "log_probs", "log_probs_grad"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    pad = rng.choice([0, 0, 0, 8, 3])  # rows that lie this many elements further apart than they are long
    if op in ("norm", "norm_grad"):
        cols = _span(rng, 1 if op == "norm" else 8, 16384)
        rows = _span(rng, 1, min(65536, max(1, (32 << 20) // cols)))
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "affine": rng.random() < 0.8, "pad": pad}
    if op in ("linear", "linear_grad"):
        dtype = rng.choice(["bfloat16", "float16"])
        rows, inner, outer = _span(rng, 1, 16384), _span(rng, 16, 4096), _span(rng, 16, 20000)
        if rng.random() < 0.5:  # half the cases at the multiples of 8 that models are built with
            inner, outer = -(-inner // 8) * 8, -(-outer // 8) * 8
        most = (100 << 30) // (2 if op == "linear" else 4)
        rows = max(1, min(rows, most // (inner * outer), (160 << 20) // max(inner, outer)))
        case = {"op": op, "rows": rows, "inner": inner, "outer": outer, "dtype": dtype,
                "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "pad": pad, "flip": rng.random() < 0.2}
        if op == "linear":
            case.update(out=rng.choice([dtype, dtype, "float32"]), bias=rng.random() < 0.7, residual=rng.random() < 0.4,
                        keep=rng.random() < 0.3)
        return case
    vocab = _span(rng, 2, 131072)
    rows = _span(rng, 1, min(32768, max(1, (128 << 20) // (vocab * SIZE[dtype]))))
    case = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "beta": rng.choice([1.0, 1.0, 0.7, 2.5]),
            "masked": rng.choice([0.0, 0.0, 0.05, 0.9]), "pad": pad}
    if op == "log_probs":
        case["top"] = min(vocab, rng.choice([0, 1, 5, 20, 64]))
    else:
        case["entropy"] = rng.random() < 0.5
    return case


def _made(gen, shape, dtype, pad=0, scale=1.0, shift=0.0):
    """Normal values; with ``pad`` a view whose rows lie further apart than they are long."""
    wide = torch.randn(*shape[:-1], shape[-1] + pad, generator=gen, device="cuda")
    return wide.mul_(scale).add_(shift).to(TYPES[dtype])[..., : shape[-1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, dtype, rows, pad = case["op"], case["dtype"], case["rows"], case["pad"]
    state = {"case": case}
    if op in ("norm", "norm_grad"):
        cols = case["cols"]
        state["x"] = _made(gen, (rows, cols), dtype, pad, 1.5, 0.3)
        state["weight"] = _made(gen, (cols,), dtype, 0, 0.2, 1.0) if case["affine"] else None
        state["bias"] = _made(gen, (cols,), dtype, 0, 0.2) if case["affine"] else None
        if op == "norm_grad":  # what the forward pass left, and the gradient that comes back
            state["dy"] = _made(gen, (rows, cols), dtype, pad)
            x = state["x"].double()
            state["mean"] = x.mean(1).float()
            state["rstd"] = (x.var(1, unbiased=False) + EPS).rsqrt().float()
    elif op in ("linear", "linear_grad"):
        inner, outer = case["inner"], case["outer"]
        state["x"] = _made(gen, (rows, inner), dtype, pad)
        w = _made(gen, (inner, outer) if case["flip"] else (outer, inner), dtype, 0, inner ** -0.5)
        state["w"] = w.t() if case["flip"] else w  # [outer][inner], stored either way round
        if op == "linear":
            state["bias"] = _made(gen, (outer,), dtype, 0, 0.5) if case["bias"] else None
            state["residual"] = _made(gen, (rows, outer), dtype, pad) if case["residual"] else None
        else:
            state["z"] = _made(gen, (rows, outer), dtype) if case["act"] != "none" else None
            state["dy"] = _made(gen, (rows, outer), dtype, pad)
    else:
        vocab = case["vocab"]
        logits = _made(gen, (rows, vocab), dtype, pad, 2.0)
        if case["masked"]:
            out = torch.rand(rows, vocab, generator=gen, device="cuda") < case["masked"]
            out[5::97] = True  # now and then a row in which nothing is left
            logits.masked_fill_(out, -math.inf)
        state["logits"] = logits
        targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        targets[3::31] = -1  # padding
        state["targets"] = targets
        if op == "log_probs_grad":
            _, log_z, entropy = _row_values(logits.double(), case["beta"])
            state["row_max"], state["log_z"], state["entropy"] = logits.amax(1).float(), log_z.float(), entropy.float()
            state["g"] = torch.randn(rows, generator=gen, device="cuda") / rows
            state["gh"] = 0.01 * torch.randn(rows, generator=gen, device="cuda") / rows if case["entropy"] else None
    return state


# ---- elementary forms ------------------------------------------------------------------------------
def _act(z, kind):
    if kind == "relu":
        return z.clamp_min(0)
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _row_values(s, beta):
    """(beta * (s - max), log of the sum of their exp, entropy) of each row; a row in which nothing is
    left has log 0 and no entropy.  The largest element's own 1 stays out of the sum, so that a row
    that is nearly certain keeps its digits."""
    top, at = s.max(1, keepdim=True)
    none = top.eq(-math.inf)
    d = beta * (s - top.masked_fill(none, 0.0))
    e = torch.exp(d)
    rest = e.scatter(1, at, 0.0).sum(1)
    log_z = torch.log1p(rest)
    entropy = log_z - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1) / (1 + rest)
    none = none[:, 0]
    return d, log_z.masked_fill(none, -math.inf), entropy.masked_fill(none, 0.0)


def _norm(x, weight, bias):
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    y = c * rstd
    if weight is not None:
        y = y * weight + bias
    return y, mean[:, 0], rstd[:, 0]


def _norm_grad(dy, x, mean, rstd, weight):
    xhat = (x - mean[:, None]) * rstd[:, None]
    g = dy * weight if weight is not None else dy
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if weight is None:
        return dx, None, None
    return dx, (dy * xhat).sum(0), dy.sum(0)


def _plain(state):
    case = state["case"]
    op, kind = case["op"], TYPES[case["dtype"]]
    wide = {k: v.float() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in state.items()}
    if op == "norm":
        y, mean, rstd = _norm(wide["x"], wide["weight"], wide["bias"])
        return {"y": y.to(kind), "mean": mean, "rstd": rstd}
    if op == "norm_grad":
        dx, dw, db = _norm_grad(wide["dy"], wide["x"], wide["mean"], wide["rstd"], wide["weight"])
        return {"dx": dx.to(kind)} if dw is None else {"dx": dx.to(kind), "dw": dw.to(kind), "db": db.to(kind)}
    if op == "linear":
        z = wide["x"] @ wide["w"].t()
        if wide["bias"] is not None:
            z = z + wide["bias"]
        y = _act(z, case["act"])
        if wide["residual"] is not None:
            y = y + wide["residual"]
        y = y.to(TYPES[case["out"]])
        return {"y": y, "z": z.to(kind)} if case["keep"] else {"y": y}
    if op == "linear_grad":
        dz = wide["dy"] * _act_slope(wide["z"], case["act"]) if wide["z"] is not None else wide["dy"]
        return {"dx": (dz @ wide["w"]).to(kind), "dw": (dz.t() @ wide["x"]).to(kind), "db": dz.sum(0).to(kind)}
    targets = state["targets"]
    at = targets.clamp_min(0)[:, None]
    if op == "log_probs":
        d, log_z, entropy = _row_values(wide["logits"], case["beta"])
        none = log_z.eq(-math.inf)[:, None]
        logp = (d - log_z.masked_fill(none[:, 0], 0.0)[:, None])
        out = {"log_prob": logp.gather(1, at)[:, 0].masked_fill(targets < 0, 0.0), "entropy": entropy,
               "row_max": wide["logits"].amax(1), "log_z": log_z}
        if case["top"]:
            ids = torch.sort(wide["logits"], dim=1, descending=True, stable=True)[1][:, : case["top"]]
            out["top_ids"], out["top_log_prob"] = ids.to(torch.int32), logp.gather(1, ids)
        return out
    logits, log_z, beta = wide["logits"], wide["log_z"], case["beta"]
    none = log_z.eq(-math.inf)[:, None]
    logp = beta * (logits - wide["row_max"][:, None].masked_fill(none, 0.0)) - log_z[:, None].masked_fill(none, 0.0)
    p = torch.exp(logp)
    g = state["g"].masked_fill((targets < 0) | none[:, 0], 0.0)[:, None]
    ds = -g * p
    ds.scatter_(1, at, -g * torch.expm1(logp.gather(1, at)))
    if state["gh"] is not None:
        ds = ds - state["gh"][:, None] * torch.where(p > 0, p * (logp + wide["entropy"][:, None]), torch.zeros_like(p))
    return {"dlogits": (beta * ds).to(kind)}


# ---- the framework's calls -------------------------------------------------------------------------
def _ours(state):
    from flyvec_b200 import ops

    case = state["case"]
    op = case["op"]
    if op == "norm":
        y, mean, rstd = ops.layer_norm(state["x"], state["weight"], state["bias"], eps=EPS, return_stats=True)
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "norm_grad":
        dx, dw, db = ops.layer_norm_backward(state["dy"], state["x"], state["mean"], state["rstd"], state["weight"])
        return {"dx": dx} if dw is None else {"dx": dx, "dw": dw, "db": db}
    if op == "linear":
        out = ops.linear(state["x"], state["w"], state["bias"], activation=case["act"], residual=state["residual"],
                         out_dtype=case["out"], return_preactivation=case["keep"])
        return {"y": out[0], "z": out[1]} if case["keep"] else {"y": out}
    if op == "linear_grad":
        dx, dw, db = ops.linear_backward(state["dy"], state["x"], state["w"], preactivation=state["z"], activation=case["act"])
        return {"dx": dx, "dw": dw, "db": db}
    if op == "log_probs":
        r = ops.token_log_probs(state["logits"], state["targets"], beta=case["beta"], top=case["top"])
        out = {"log_prob": r.log_prob, "entropy": r.entropy, "row_max": r.row_max, "log_z": r.log_z}
        if case["top"]:
            out["top_ids"], out["top_log_prob"] = r.top_ids, r.top_log_prob
        return out
    return {"dlogits": ops.token_log_probs_backward(state["g"], state["logits"], state["targets"], state["row_max"], state["log_z"],
                                                    state["entropy"], grad_entropy=state["gh"], beta=case["beta"])}


def run(state):
    return _ours(state) if own else _plain(state)


def work(case):
    op, b, n = case["op"], SIZE[case["dtype"]], case["rows"]
    if op in ("norm", "norm_grad"):
        d = case["cols"]
        big = (2 if op == "norm" else 3) * n * d * b
        vectors = (2 if op == "norm" else 3) * d * b if case["affine"] else 0
        return {"bytes": big + vectors + 8 * n, "flops": (8 if op == "norm" else 14) * n * d}
    if op == "linear":
        k, m = case["inner"], case["outer"]
        out = n * m * (SIZE[case["out"]] + b * (case["residual"] + case["keep"]))
        return {"bytes": b * (n * k + m * k + m * case["bias"]) + out, "flops": 2 * n * m * k}
    if op == "linear_grad":
        k, m = case["inner"], case["outer"]
        return {"bytes": b * (2 * n * k + 2 * m * k + m + n * m * (1 + (case["act"] != "none"))), "flops": 4 * n * m * k}
    v = case["vocab"]
    if op == "log_probs":
        return {"bytes": n * (v * b + 16 + 8 * case["top"]), "flops": 5 * n * v}
    return {"bytes": n * (2 * v * b + 28), "flops": 8 * n * v}


# ---- the definition in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    v = {k: t.double() if torch.is_tensor(t) and t.is_floating_point() else t for k, t in state.items()}
    op, kind = case["op"], case.get("act", "none")
    if op == "norm":
        x = v["x"]
        n = x.shape[1]
        mean = x.sum(1) / n
        var = ((x - mean[:, None]) ** 2).sum(1) / n
        rstd = (var + EPS) ** -0.5
        y = torch.einsum("rc,r->rc", x - mean[:, None], rstd)
        if v["weight"] is not None:
            y = torch.addcmul(v["bias"], y, v["weight"])
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "norm_grad":
        n = v["x"].shape[1]
        h = torch.einsum("rc,r->rc", v["x"] - v["mean"][:, None], v["rstd"])
        u = v["dy"] if v["weight"] is None else torch.einsum("rc,c->rc", v["dy"], v["weight"])
        a, b = u.sum(1) / n, torch.einsum("rc,rc->r", u, h) / n
        dx = torch.einsum("rc,r->rc", u - a[:, None] - torch.einsum("rc,r->rc", h, b), v["rstd"])
        if v["weight"] is None:
            return {"dx": dx}
        return {"dx": dx, "dw": torch.einsum("rc,rc->c", v["dy"], h), "db": v["dy"].sum(0)}
    normal = lambda t: 0.5 * torch.erfc(-t / math.sqrt(2))  # noqa: E731  the normal distribution function
    if op == "linear":
        z = torch.einsum("ri,oi->ro", v["x"], v["w"])
        if v["bias"] is not None:
            z += v["bias"]
        if kind == "relu":
            y = torch.where(z > 0, z, torch.zeros_like(z))
        elif kind == "gelu":
            y = z * normal(z)
        elif kind == "gelu_tanh":
            y = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        elif kind == "silu":
            y = z * torch.sigmoid(z)
        else:
            y = z.clone()
        if v["residual"] is not None:
            y += v["residual"]
        return {"y": y, "z": z} if case["keep"] else {"y": y}
    if op == "linear_grad":
        dz = v["dy"]
        if kind != "none":
            z = v["z"].detach().requires_grad_()
            y = {"relu": torch.relu, "gelu": lambda t: t * normal(t), "silu": lambda t: t * torch.sigmoid(t),
                 "gelu_tanh": lambda t: t * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3))}[kind](z)
            dz, = torch.autograd.grad(y, z, dz)
        return {"dx": torch.einsum("ro,oi->ri", dz, v["w"]), "dw": torch.einsum("ro,ri->oi", dz, v["x"]), "db": dz.sum(0)}
    s, t = case["beta"] * v["logits"], state["targets"]
    lse = torch.logsumexp(s, 1)
    empty = lse == -math.inf
    logp = torch.where(empty[:, None], s, s - lse[:, None])
    p = torch.where(empty[:, None], torch.zeros_like(s), torch.exp(logp))
    entropy = -torch.xlogy(p, p).sum(1)
    rows = torch.arange(len(t), device=t.device)
    if op == "log_probs":
        out = {"log_prob": torch.where(t < 0, torch.zeros_like(lse), logp[rows, t.clamp_min(0)]), "entropy": entropy}
        out["row_max"] = v["logits"].max(1)[0]
        out["log_z"] = torch.where(empty, lse, lse - case["beta"] * out["row_max"])
        if case["top"]:
            _, ids = torch.sort(v["logits"], dim=1, descending=True, stable=True)
            ids = ids[:, : case["top"]]
            out["top_ids"], out["top_log_prob"] = ids.to(torch.int32), torch.take_along_dim(logp, ids, 1)
        return out
    one = torch.zeros_like(p)
    one[rows, t.clamp_min(0)] = 1.0
    g = torch.where((t < 0) | empty, torch.zeros_like(v["g"]), v["g"])
    ds = g[:, None] * (one - p)
    if v["gh"] is not None:
        ds -= v["gh"][:, None] * (torch.xlogy(p, p) + p * entropy[:, None])
    return {"dlogits": case["beta"] * ds}
