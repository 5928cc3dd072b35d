"""Measured cases of the training and projection operators next to the KNN search.

The rows that are searched come out of a projection of features (``linear``),
and such a projection is trained by a softmax over the inner products with a
large set of class or base rows (``softmax_xent``); both have their gradients.

``own`` False computes the operators with elementary torch operations in 32
bits, rounded once to the outputs' type; ``own`` True calls the package.
Feature widths 128, 300, 784, 960 and 1024 and set sizes of 10,000, 100,000 and
1,000,000 rows are those of the KNN workloads and tests of this repository.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def listed():
    return [
        # Serving: one query's features projected before a search.
        dict(name="linear one row", op="linear", m=1, k=960, n=1024, dtype="bf16", act="gelu", bias=True,
             residual=False, save=False, out="same", pad=0),
        # A small ragged batch out of a wider feature table, with a skip connection.
        dict(name="linear ragged batch", op="linear", m=33, k=785, n=300, dtype="f16", act="relu", bias=True,
             residual=True, save=False, out="same", pad=3),
        # Projecting a float data set to the width that is searched.
        dict(name="linear f32 rows", op="linear", m=10000, k=960, n=128, dtype="f32", act="none", bias=True,
             residual=False, save=False, out="same", pad=0),
        # The hidden layer of a training step over a whole 100,000 x 784 feature set.
        dict(name="linear hidden layer", op="linear", m=100000, k=784, n=1024, dtype="bf16", act="gelu", bias=True,
             residual=False, save=True, out="same", pad=0),
        # Gradients of that layer for a mini-batch, and for the whole set.
        dict(name="linear grad mini-batch", op="linear_backward", m=1537, k=960, n=300, dtype="f16", act="silu",
             bias=True, pad=0),
        dict(name="linear grad hidden layer", op="linear_backward", m=100000, k=784, n=1024, dtype="bf16",
             act="gelu", bias=True, pad=0),
        # Scoring one query's label against 100,000 rows.
        dict(name="xent one row", op="xent", m=1, k=128, n=100000, dtype="bf16", scale=20.0, ignored=0.0, pad=0),
        # Evaluation against a million rows at width 128: the softmax itself bounds it.
        dict(name="xent million rows", op="xent", m=2048, k=128, n=1000000, dtype="bf16", scale=20.0, ignored=0.0,
             pad=0),
        # A training batch against 100,000 rows at width 960: the product bounds it.
        dict(name="xent wide rows", op="xent", m=8192, k=960, n=100000, dtype="bf16", scale=16.0, ignored=0.1, pad=0),
        # A step of a small data set in fp16 with unlabelled rows.
        dict(name="xent grad small set", op="xent_backward", m=1000, k=128, n=10000, dtype="f16", scale=10.0,
             ignored=0.25, pad=8),
        # The gradient in 32 bits, odd sizes.
        dict(name="xent grad f32", op="xent_backward", m=2000, k=300, n=30011, dtype="f32", scale=8.0, ignored=0.1,
             pad=0),
        # The gradient of the large training batch.
        dict(name="xent grad wide rows", op="xent_backward", m=8192, k=960, n=100000, dtype="bf16", scale=16.0,
             ignored=0.1, pad=0),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    while True:
        op = rng.choice(("linear", "linear_backward", "xent", "xent_backward"))
        case = dict(op=op, dtype=rng.choice(("bf16", "bf16", "f16", "f32")), pad=rng.choice((0, 0, 3, 8)))
        if op.startswith("linear"):
            case.update(m=_spread(rng, 1 if op == "linear" else 32, 100000), k=_spread(rng, 17, 1024),
                        n=_spread(rng, 32, 1024), act=rng.choice(ACTIVATIONS), bias=rng.random() < 0.7)
            if op == "linear":
                case.update(residual=rng.random() < 0.4, save=rng.random() < 0.4,
                            out=rng.choice(("same", "same", "f32")))
        else:
            case.update(m=_spread(rng, 1 if op == "xent" else 16, 8192), k=_spread(rng, 17, 960),
                        n=_spread(rng, 1000, 1000000), scale=rng.choice((1.0, 8.0, 20.0)),
                        ignored=rng.choice((0.0, 0.1, 0.5)))
        # No dearer than the dearest listed case; the plain form keeps m x n values.
        if case["m"] * case["n"] <= 1000000000 and work(case)["flops"] <= work(listed()[-1])["flops"]:
            return case


def work(case):
    m, k, n, e = case["m"], case["k"], case["n"], SIZES[case["dtype"]]
    if case["op"] == "linear":
        out = 4 if case["out"] == "f32" else e
        moved = e * (m * k + n * k + m * n * (int(case["residual"]) + int(case["save"])) + n * int(case["bias"]))
        return {"bytes": moved + out * m * n, "flops": 2 * m * n * k}
    if case["op"] == "linear_backward":
        pre = 0 if case["act"] == "none" else 1
        return {"bytes": e * (m * n * (1 + pre) + 2 * (m * k + n * k) + n * int(case["bias"])), "flops": 4 * m * n * k}
    if case["op"] == "xent":
        return {"bytes": e * (m * k + n * k) + 16 * m, "flops": 2 * m * n * k}
    return {"bytes": 2 * e * (m * k + n * k) + 16 * m, "flops": 6 * m * n * k}


def _rows(gen, rows, width, pad, dtype, scale=1.0):
    """Rows of a table that is `pad` values wider than they are."""
    t = torch.randn((rows, width + pad), generator=gen, device="cuda") * scale
    return t.to(dtype)[:, :width]


def _unit(t):
    return t / t.norm(dim=1, keepdim=True).clamp_min(1e-12)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, m, k, n = DTYPES[case["dtype"]], case["m"], case["k"], case["n"]
    state = dict(case=case)
    if case["op"].startswith("linear"):
        # Standardised features, weights as a layer starts with them.
        state["x"] = _rows(gen, m, k, case["pad"], dtype)
        state["w"] = _rows(gen, n, k, 0, dtype, k ** -0.5)
        bias = (torch.randn(n, generator=gen, device="cuda") * 0.1).to(dtype) if case["bias"] else None
        if case["op"] == "linear":
            state["bias"] = bias
            state["residual"] = _rows(gen, m, n, case["pad"], dtype) if case["residual"] else None
        else:
            state["dy"] = _rows(gen, m, n, case["pad"], dtype, 0.05)
            state["pre"] = None
            if case["act"] != "none":
                z = state["x"].float() @ state["w"].float().t()
                state["pre"] = (z if bias is None else z + bias.float()).to(dtype)
        return state
    # Class rows of unit length; a row's embedding lies near its class's.
    w = _unit(torch.randn((n, k), generator=gen, device="cuda"))
    labels = torch.randint(0, n, (m,), generator=gen, device="cuda")
    x = _unit(w[labels] + torch.randn((m, k), generator=gen, device="cuda") * k ** -0.5)
    wide = torch.zeros((m, k + case["pad"]), device="cuda", dtype=dtype)
    wide[:, :k] = x.to(dtype)
    state.update(x=wide[:, :k], w=w.to(dtype))
    out = torch.rand(m, generator=gen, device="cuda") < case["ignored"]
    state["labels"] = torch.where(out, torch.full_like(labels, -1), labels)
    if case["op"] == "xent_backward":
        # The mean over the rows; fp16 steps run under a loss scale.
        state["dloss"] = torch.full((m,), (1024.0 if case["dtype"] == "f16" else 1.0) / m, device="cuda")
        state["lse"] = torch.cat([torch.logsumexp((xs.float() @ state["w"].float().t()) * case["scale"], dim=1)
                                  for xs in state["x"].split(1024)])
    return state


def _activate(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain(state):
    case = state["case"]
    x, w, dtype = state["x"].float(), state["w"].float(), state["x"].dtype
    if case["op"] == "linear":
        z = x @ w.t()
        if state["bias"] is not None:
            z = z + state["bias"].float()
        y = _activate(z, case["act"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        out = y.to(torch.float32 if case["out"] == "f32" else dtype)
        return {"out": out, "pre": z.to(dtype)} if case["save"] else {"out": out}
    if case["op"] == "linear_backward":
        dz = state["dy"].float()
        if state["pre"] is not None:
            dz = dz * _slope(state["pre"].float(), case["act"])
        got = {"dx": (dz @ w).to(dtype), "dw": (dz.t() @ x).to(dtype)}
        if case["bias"]:
            got["db"] = dz.sum(dim=0).to(dtype)
        return got
    labels = state["labels"]
    kept = (labels >= 0) & (labels < w.shape[0])
    at = torch.where(kept, labels, torch.zeros_like(labels))[:, None]
    z = (x @ w.t()) * case["scale"]
    if case["op"] == "xent":
        top = z.max(dim=1, keepdim=True).values
        lse = (torch.log(torch.exp(z - top).sum(dim=1, keepdim=True)) + top)[:, 0]
        return {"loss": torch.where(kept, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse)), "lse": lse}
    g = torch.exp(z - state["lse"][:, None])
    g.scatter_add_(1, at, torch.full_like(g[:, :1], -1.0))
    g = g * torch.where(kept, state["dloss"] * case["scale"], torch.zeros_like(state["dloss"]))[:, None]
    return {"dx": (g @ w).to(dtype), "dw": (g.t() @ x).to(dtype)}


def _own(state):
    import knng_gpu_b200 as kg

    case = state["case"]
    if case["op"] == "linear":
        got = kg.linear(state["x"], state["w"], bias=state["bias"], residual=state["residual"],
                        activation=case["act"], out_dtype=torch.float32 if case["out"] == "f32" else None,
                        save_pre=case["save"])
        return {"out": got[0], "pre": got[1]} if case["save"] else {"out": got}
    if case["op"] == "linear_backward":
        dx, dw, db = kg.linear_backward(state["dy"], state["x"], state["w"], pre=state["pre"],
                                        activation=case["act"], need_db=case["bias"])
        return {"dx": dx, "dw": dw, "db": db} if case["bias"] else {"dx": dx, "dw": dw}
    if case["op"] == "xent":
        loss, lse = kg.softmax_xent(state["x"], state["w"], state["labels"], scale=case["scale"])
        return {"loss": loss, "lse": lse}
    dx, dw = kg.softmax_xent_backward(state["dloss"], state["x"], state["w"], state["labels"], state["lse"],
                                      scale=case["scale"])
    return {"dx": dx, "dw": dw}


def run(state):
    return _own(state) if own else _plain(state)


def exact(case, seed):
    """The definitions in 64 bits, a block of rows at a time."""
    s = prepare(case, seed)
    x, w = s["x"].double(), s["w"].double()
    m, n = case["m"], case["n"]
    block = max(1, min(m, 250000000 // n))
    parts = [slice(i, min(i + block, m)) for i in range(0, m, block)]
    normal = torch.distributions.Normal(torch.zeros((), device="cuda", dtype=torch.float64), 1.0)
    c = (2.0 / math.pi) ** 0.5

    def both(z):
        """act(z) and its derivative."""
        if case["act"] == "none":
            return z, torch.ones_like(z)
        if case["act"] == "relu":
            return torch.relu(z), torch.heaviside(z, torch.zeros_like(z))
        if case["act"] == "gelu":
            return z * normal.cdf(z), normal.cdf(z) + z * torch.exp(normal.log_prob(z))
        # x sigmoid(u(x)): silu has u = x, the tanh form u = 2c(x + 0.044715 x^3).
        tanh_form = case["act"] == "gelu_tanh"
        u = 2 * c * (z + 0.044715 * z ** 3) if tanh_form else z
        du = 2 * c * (1 + 0.134145 * z ** 2) if tanh_form else torch.ones_like(z)
        p, q = torch.special.expit(u), torch.special.expit(-u)
        return z * p, p + z * p * q * du

    if case["op"] == "linear":
        bias = torch.zeros(n, device="cuda", dtype=torch.float64) if s["bias"] is None else s["bias"].double()
        pre = torch.cat([torch.addmm(bias, x[r], w.t()) for r in parts])
        y = torch.cat([both(pre[r])[0] for r in parts])
        if s["residual"] is not None:
            y = y + s["residual"].double()
        return {"out": y, "pre": pre} if case["save"] else {"out": y}
    if case["op"] == "linear_backward":
        dx, dw = torch.empty_like(x), torch.zeros_like(w)
        db = torch.zeros(n, device="cuda", dtype=torch.float64)
        for r in parts:
            dz = s["dy"][r].double()
            if s["pre"] is not None:
                dz = dz * both(s["pre"][r].double())[1]
            dx[r] = dz @ w
            dw += dz.t() @ x[r]
            db += dz.sum(0)
        return {"dx": dx, "dw": dw, "db": db} if case["bias"] else {"dx": dx, "dw": dw}
    y = s["labels"]
    kept = (0 <= y) & (y < n)
    if case["op"] == "xent":
        lse, loss = [], []
        for r in parts:
            z = case["scale"] * (x[r] @ w.t())
            lse.append(torch.logsumexp(z, dim=1))
            own_z = case["scale"] * (x[r] * w[y[r].clamp(0, n - 1)]).sum(1)
            loss.append((lse[-1] - own_z) * kept[r])
        return {"loss": torch.cat(loss), "lse": torch.cat(lse)}
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for r in parts:
        g = torch.exp(case["scale"] * (x[r] @ w.t()) - s["lse"][r].double()[:, None])
        hit = kept[r].nonzero()[:, 0]
        g[hit, y[r][hit]] -= 1.0
        g *= (case["scale"] * s["dloss"][r].double() * kept[r])[:, None]
        dx[r] = g @ w
        dw += g.t() @ x[r]
    return {"dx": dx, "dw": dw}
