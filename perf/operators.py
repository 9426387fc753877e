"""The node-feature operators of gpu_eigsh.features, as cases to be timed.

Three operators, forward alone or with their backward pass:

  lookup   rows of a table by id, scaled, and the table's gradient
  norm     layer norm over the last dimension, and the gradients of x, weight and bias
  edges    squared distances along the edges of a graph, and the features' gradient

``own`` chooses between the plain form (elementary torch operations) and the
framework's calls.  A case is a dict of plain values; see listed().
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f64": torch.float64, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f64": 8, "f16": 2, "bf16": 2}
_ops = None


def _features():
    global _ops
    if _ops is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lanczos-gpu_b200")
        if pkg not in sys.path:
            sys.path.insert(1, pkg)
        import gpu_eigsh.features as f

        _ops = f
    return _ops


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _lookup(name, rows, dim, tokens, dtype, ids, scale, pad, back, wide=True):
    return {"name": name, "op": "lookup", "rows": rows, "dim": dim, "tokens": tokens, "dtype": dtype, "ids": ids,
            "scale": scale, "pad": pad, "back": back, "wide": wide}


def _norm(name, rows, dim, dtype, affine, back):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "affine": affine, "back": back}


def _edges(name, n, edges, dim, dtype, hubs, back):
    return {"name": name, "op": "edges", "n": n, "edges": edges, "dim": dim, "dtype": dtype, "hubs": hubs,
            "back": back}


def listed():
    return [
        # one new token of a sequence: latency
        _lookup("lookup one token", 32768, 1024, 1, "bf16", "zipf", "number", False, False),
        # the 64 fp32 probes of a log-det over a million vertices, renumbered: a lookup by a permutation
        _lookup("lookup probe rows", 1000000, 64, 1000000, "f32", "permutation", "none", False, False),
        # a training step's token embeddings: frequent and rare ids, one token in 16 is padding
        _lookup("lookup train bf16", 131072, 2048, 16384, "bf16", "zipf", "number", True, True),
        # a mini-batch of vertices of a spectral embedding: k = 20 eigenvectors, each column with its own scale
        _lookup("lookup spectral f64", 100000, 20, 8192, "f64", "uniform", "column", False, True),
        # odd row length and count, narrow ids
        _lookup("lookup odd f16", 50001, 333, 7777, "f16", "zipf", "none", False, True, wide=False),
        # one token's features: latency
        _norm("norm one token", 1, 1024, "bf16", True, False),
        # a training step's activations
        _norm("norm train bf16", 16384, 4096, "bf16", True, True),
        # the points of a kNN graph (a million points of 10 coordinates), normalised before the neighbour search
        _norm("norm points f64", 1000000, 10, "f64", False, False),
        # odd rows
        _norm("norm odd f32", 5003, 1537, "f32", True, True),
        # the graph of the smoke check: latency of a small training step
        _edges("edges small f64", 600, 3000, 3, "f64", False, True),
        # the graph of the million-vertex log-det (5 edges a vertex), 10 features
        _edges("edges large f32", 1000000, 5000000, 10, "f32", False, True),
        # wide learned features on a graph with hubs
        _edges("edges wide bf16", 20000, 200000, 256, "bf16", True, True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    limit = 5.0e8   # bytes of a drawn case: below the largest listed one
    while True:
        op = rng.choice(["lookup", "norm", "edges"])
        dtype = rng.choice(["f32", "f64", "f16", "bf16", "bf16"])
        if op == "lookup":
            ids = rng.choice(["zipf", "zipf", "uniform", "permutation"])
            rows, dim = _log_int(rng, 10, 1000000), _log_int(rng, 1, 8192)
            tokens = rows if ids == "permutation" else _log_int(rng, 1, 200000)
            c = _lookup("", rows, dim, tokens, dtype, ids, rng.choice(["none", "number", "column"]),
                        ids != "permutation" and rng.random() < 0.4, rng.random() < 0.7, rng.random() < 0.7)
            size = rows * dim + 3 * tokens * dim
        elif op == "norm":
            c = _norm("", _log_int(rng, 1, 500000), _log_int(rng, 4, 32768), dtype, rng.random() < 0.7,
                      rng.random() < 0.7)
            size = 4 * c["rows"] * c["dim"]
        else:
            n = _log_int(rng, 10, 1000000)
            c = _edges("", n, _log_int(rng, n, 8 * n), _log_int(rng, 1, 1024), dtype, rng.random() < 0.3,
                       rng.random() < 0.7)
            size = 2 * c["edges"] * c["dim"]
            if c["edges"] > 5000000:
                continue
        del c["name"]
        if size * 4 <= limit and work(c)["bytes"] <= limit:
            return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _zipf(count, rows, gen):
    """Ids whose frequency falls as 1 / rank."""
    u = torch.rand(count, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(rows + 1.0)).long() - 1).clamp_(0, rows - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    wide = torch.float64 if dt == torch.float64 else torch.float32

    def normal(*shape, dtype=dt, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=wide) * std + mean).to(dtype)

    back = case["back"]
    s = {"op": case["op"], "back": back}
    if case["op"] == "lookup":
        rows, dim, tokens = case["rows"], case["dim"], case["tokens"]
        if case["ids"] == "permutation":
            ids = torch.randperm(rows, generator=gen, device="cuda")
        elif case["ids"] == "zipf":
            ids = _zipf(tokens, rows, gen)
        else:
            ids = torch.randint(0, rows, (tokens,), generator=gen, device="cuda")
        s["pad"] = None
        if case["pad"]:
            s["pad"] = rows - 1
            ids[torch.rand(tokens, generator=gen, device="cuda") < 1.0 / 16.0] = rows - 1
        s["ids"] = ids if case["wide"] else ids.to(torch.int32)
        s["table"] = normal(rows, dim, std=dim ** -0.5).requires_grad_(back)
        s["scale"] = None
        if case["scale"] == "number":
            s["scale"] = math.sqrt(dim)
        elif case["scale"] == "column":
            s["scale"] = torch.rand(dim, generator=gen, device="cuda", dtype=wide).add_(0.5).requires_grad_(back)
        if back:
            s["g"] = normal(tokens, dim)
    elif case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        s["x"] = normal(rows, dim, std=1.5, mean=0.25).requires_grad_(back)
        s["w"] = normal(dim, std=0.2, mean=1.0).requires_grad_(back) if case["affine"] else None
        s["b"] = normal(dim, std=0.2).requires_grad_(back) if case["affine"] else None
        if back:
            s["g"] = normal(rows, dim)
    else:
        n, m, dim = case["n"], case["edges"], case["dim"]
        i = torch.arange(m, device="cuda") * n // m
        j = _zipf(m, n, gen) if case["hubs"] else torch.randint(0, n, (m,), generator=gen, device="cuda")
        lo, hi = torch.minimum(i, j), torch.maximum(i, j)
        key = torch.sort(lo * n + hi).values
        s["idx"] = torch.stack([key // n, key % n])
        s["x"] = normal(n, dim).requires_grad_(back)
        if back:
            s["g"] = normal(m, dtype=wide)
        if own:
            s["graph"] = _features().EdgeDistances(s["idx"], n)   # kept by a program that trains on one graph
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _plain_lookup(s):
    W, ids, scale = s["table"].detach(), s["ids"].long(), s["scale"]
    wide = torch.float64 if W.dtype == torch.float64 else torch.float32
    column = torch.is_tensor(scale)
    f = scale.detach() if column else 1.0 if scale is None else scale
    rows = W[ids].to(wide)
    keep = None if s["pad"] is None else (ids != s["pad"]).to(wide)[:, None]
    y = rows * f if keep is None else rows * f * keep
    out = [y.to(W.dtype)]
    if s["back"]:
        g = s["g"].to(wide) if keep is None else s["g"].to(wide) * keep
        out.append(torch.zeros(W.shape, dtype=wide, device=W.device).index_add_(0, ids, g * f).to(W.dtype))
        if column:
            out.append((rows * g).sum(0).to(scale.dtype))
    return out


def _plain_norm(s):
    x, w, b = (None if t is None else t.detach() for t in (s["x"], s["w"], s["b"]))
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    xf = x.to(wide)
    c = xf - xf.mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-5)
    h = c * r
    y = h if w is None else h * w.to(wide) + b.to(wide)
    out = [y.to(x.dtype)]
    if s["back"]:
        g = s["g"].to(wide)
        wg = g if w is None else g * w.to(wide)
        out.append((r * (wg - wg.mean(-1, keepdim=True) - h * (wg * h).mean(-1, keepdim=True))).to(x.dtype))
        if w is not None:
            out += [(g * h).sum(0).to(w.dtype), g.sum(0).to(b.dtype)]
    return out


def _plain_edges(s):
    x, (i, j) = s["x"].detach(), s["idx"]
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    xf = x.to(wide)
    d = xf[i] - xf[j]
    out = [(d * d).sum(-1)]
    if s["back"]:
        c = 2.0 * s["g"][:, None] * d
        out.append(torch.zeros_like(xf).index_add_(0, i, c).index_add_(0, j, -c).to(x.dtype))
    return out


def run(s):
    if not own:
        return {"lookup": _plain_lookup, "norm": _plain_norm, "edges": _plain_edges}[s["op"]](s)
    f = _features()
    if s["op"] == "lookup":
        y = f.embedding_lookup(s["table"], s["ids"], s["scale"], s["pad"])
        leaves = [s["table"]] + ([s["scale"]] if torch.is_tensor(s["scale"]) else [])
    elif s["op"] == "norm":
        y = f.layer_norm(s["x"], s["w"], s["b"], 1e-5)
        leaves = [s["x"]] + ([s["w"], s["b"]] if s["w"] is not None else [])
    else:
        y = s["graph"](s["x"])
        leaves = [s["x"]]
    if not s["back"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["g"])]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _distinct(case):
    """Expected number of different rows named by the ids."""
    rows, tokens = case["rows"], case["tokens"]
    if case["ids"] == "permutation":
        return rows
    if case["ids"] == "uniform":
        return rows * -math.expm1(tokens * math.log1p(-1.0 / rows)) if rows > 1 else 1
    p = np.diff(np.log(np.arange(1, rows + 2))) / math.log(rows + 1.0)
    return float(-np.expm1(tokens * np.log1p(-p)).sum()) if rows > 1 else 1


def work(case):
    e, back = _SIZE[case["dtype"]], case["back"]
    wide = max(4, e)
    if case["op"] == "lookup":
        rows, dim, tokens = case["rows"], case["dim"], case["tokens"]
        scale = {"none": 0, "number": 0, "column": dim * wide}[case["scale"]]
        b = tokens * (8 if case["wide"] else 4) + (_distinct(case) + tokens) * dim * e + scale
        f = tokens * dim * (0 if case["scale"] == "none" else 1)
        if back:
            b += tokens * dim * e + rows * dim * e + scale
            f += tokens * dim * 2 + (2 * tokens * dim if case["scale"] == "column" else 0)
    elif case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        par = 2 * dim * e if case["affine"] else 0
        b = (4 if back else 2) * rows * dim * e + (2 if back else 1) * par
        f = (18 if back else 7) * rows * dim
    else:
        n, m, dim = case["n"], case["edges"], case["dim"]
        b = m * 16 + n * dim * e + m * wide + (m * wide + n * dim * e if back else 0)
        f = (9 if back else 3) * m * dim
    return {"bytes": float(b), "flops": float(f)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    leaf = lambda t: t.detach().to(f64).requires_grad_(case["back"])  # noqa: E731
    if case["op"] == "lookup":
        W = leaf(s["table"])
        leaves = [W]
        if torch.is_tensor(s["scale"]):
            f = leaf(s["scale"])
            leaves.append(f)
        else:
            f = torch.tensor(1.0 if s["scale"] is None else s["scale"], dtype=f64, device="cuda")
        y = torch.index_select(W, 0, s["ids"].long()) * f
        if s["pad"] is not None:
            y = torch.where((s["ids"] == s["pad"])[:, None], torch.zeros((), dtype=f64, device="cuda"), y)
    elif case["op"] == "norm":
        x = leaf(s["x"])
        leaves = [x]
        var, mean = torch.var_mean(x, dim=-1, unbiased=False, keepdim=True)
        y = (x - mean) / torch.sqrt(var + 1e-5)
        if s["w"] is not None:
            w, b = leaf(s["w"]), leaf(s["b"])
            leaves += [w, b]
            y = y * w + b
    else:
        x = leaf(s["x"])
        leaves = [x]
        d = torch.index_select(x, 0, s["idx"][0]) - torch.index_select(x, 0, s["idx"][1])
        y = torch.linalg.vector_norm(d, dim=-1) ** 2 if not case["back"] else (d ** 2).sum(dim=-1)
    if not case["back"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["g"].to(f64))]
