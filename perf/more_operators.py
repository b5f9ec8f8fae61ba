"""The operators of leaves that are more than linear, as cases to be timed and checked.

A leaf may hold a layer: a linear map with an activation, or a gated one, whose outputs are
added to what a row has already.  Such leaves are trained by gradients, which are clipped
by their global norm before a step.  The operators:

  layer     y[n] = r[n] + sum over trees of f(W[t, leaf] x[n] + b[t, leaf]) (`leaf_layer`);
            f is an activation, or gated: the map's first half goes through the activation
            and multiplies the second
  train     the layer and its gradients: y, dx, dW, db (`leaf_layer`, `leaf_layer_grad`)
  norm      the 2-norm over all elements of many tensors (`grad_norm`)
  clip      the same, and the tensors scaled to a largest norm (`clip_grads`)

A case is a dict of plain values.  `listed()` names the fixed ones and `draw()` gives more
of the same ranges; `prepare()` makes what a program holds before the call, `run()` is one
pass: the plain form in elementary torch operations, or the package's entry points where
`own` is set; `exact()` is the same in 64 bits and `work()` the bytes and operations that
a pass cannot do without.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "mixed": 3}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid")

LAYER = dict(op="layer", rows=64, cols=28, outputs=1, trees=1, leaves=31, type="f32", act="relu",
             gated=False, residual=True, bias=True, lost=0.0, pad=0)
TRAIN = dict(LAYER, op="train")
CLIP = dict(op="clip", tensors=2, total=1000, type="f32", flat=False, limit=0.5)


def listed():
    return [
        # an online request to a forest of small leaves: one output, added to a start score
        dict(LAYER, name="layer_request", trees=100, act="sigmoid"),
        # batch scoring of ten classes by the leaves of one tree, added to the earlier trees'
        dict(LAYER, name="layer_table", rows=2000000, outputs=10, leaves=127, act="silu"),
        # a batch of single rows through one wide layer: its weights
        dict(LAYER, name="layer_batch", cols=4096, outputs=4096, leaves=1, type="bf16", act="gelu"),
        # a long batch through one wide layer and back onto the stream
        dict(LAYER, name="layer_dense", rows=16389, cols=4096, outputs=2048, leaves=1, type="bf16",
             act="gelu_tanh"),
        # a step of one tree's hidden leaves over a table
        dict(TRAIN, name="train_hidden", rows=200003, cols=100, outputs=64, act="gelu"),
        # one row through a wide gated layer
        dict(LAYER, name="gated_token", rows=1, cols=4096, outputs=4096, leaves=7, type="bf16",
             act="silu", gated=True, residual=False, bias=False),
        # a few rows through wide gated experts: the weights of the experts that are hit
        dict(LAYER, name="gated_few", rows=16, cols=4096, outputs=2048, type="f16", act="silu",
             gated=True, residual=False),
        # a batch through wide gated experts: matrix products of ragged sizes
        dict(LAYER, name="gated_experts", rows=40007, cols=2000, outputs=2048, type="bf16",
             act="silu", gated=True, residual=False),
        # a step of wide gated experts
        dict(TRAIN, name="gated_train", rows=16389, cols=2048, outputs=2048, leaves=15,
             type="bf16", act="silu", gated=True, residual=False, bias=False),
        # the gradients of one tree's small leaves: maps and biases
        dict(CLIP, name="norm_leaves", op="norm", total=31 * 10 * 101),
        # the gradients of many layers, in one buffer end to end
        dict(CLIP, name="clip_layers", tensors=1000, total=100000007, type="bf16", flat=True),
        # a few large gradients of both widths, over their limit
        dict(CLIP, name="clip_large", tensors=16, total=400000000, type="mixed"),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("layer", "layer", "train", "norm", "clip"))
    if op in ("norm", "clip"):
        flat = rng.choice((True, False))
        tensors = _between(rng, 1, 1500) if flat else _between(rng, 1, 48)
        return dict(CLIP, op=op, flat=flat, tensors=tensors,
                    total=_between(rng, max(100, tensors), 400000000),
                    type=rng.choice(("f32", "bf16", "f16") if flat else ("f32", "bf16", "mixed")),
                    limit=rng.choice((0.1, 0.5, 2.0)))
    trees = rng.choice((1, 1, 1, 1, 2, 20))
    case = dict(LAYER, op=op, trees=trees, leaves=rng.choice((1, 2, 7, 15, 31, 127)),
                type=rng.choice(("f32", "bf16", "bf16", "f16")), act=rng.choice(ACTIVATIONS),
                gated=rng.choice((True, False)), residual=rng.choice((True, False)),
                bias=rng.choice((True, False)), lost=rng.choice((0.0, 0.0, 0.1)),
                pad=rng.choice((0, 0, 1, 8)))
    case["cols"] = _between(rng, 1, 4096)
    case["outputs"] = rng.choice((1, _between(rng, 2, 32), _between(rng, 33, 4096)))
    size = case["cols"] * case["outputs"] * (2 if case["gated"] else 1)
    if trees * case["leaves"] * size > 300000000:
        case["trees"], case["leaves"] = 1, min(case["leaves"], 7)
    # no more rows than 150 GFLOP or a table of 800 MB give
    wide = max(case["cols"], case["outputs"] * (2 if case["gated"] else 1))
    most = min(75e9 / (size * case["trees"]) / (3 if op == "train" else 1),
               2e8 / (wide * case["trees"]), 2e6)
    case["rows"] = _between(rng, 1, max(1, int(most)))
    return case


# ---- inputs -----------------------------------------------------------------------------

def _matrix(case, gen, rows, cols, scale=1.0, pad=0):
    """N(0, 1) * scale; `pad` columns more in memory than in the matrix."""
    out = torch.empty((rows, cols + pad), device=DEVICE, dtype=TYPES[case["type"]])
    step = max(1, 50000000 // max(1, cols + pad))
    for r in range(0, rows, step):
        b = out[r:r + step]
        b.copy_(torch.randn(b.shape, generator=gen, device=DEVICE) * scale)
    return out[:, :cols]


def _groups(case, gen):
    """order int32 [trees, rows], begin and count int32 [trees, leaves]: the rows of a tree by
    their leaf, those of one leaf ascending, those in no leaf last.  Leaf sizes spread as
    exp(N(0, 1)), one leaf in ten without rows; the share `lost` of the rows is in none."""
    N, T, L = case["rows"], case["trees"], case["leaves"]
    order, begin, count = [], [], []
    # sizes from the host, whose sums do not depend on a schedule
    host = torch.Generator().manual_seed(gen.initial_seed())
    for t in range(T):
        size = torch.randn(L, generator=host).exp()
        size[torch.rand(L, generator=host) < 0.1] = 0
        size[int(torch.randint(L, (1,), generator=host))] += 0.5
        edges = (size.cumsum(0) / size.sum()).to(DEVICE)
        u = torch.rand(N, generator=gen, device=DEVICE)
        leaf = torch.bucketize(u, edges, right=True).clamp_(max=L - 1)
        if case["lost"]:
            leaf[torch.rand(N, generator=gen, device=DEVICE) < case["lost"]] = L
        order.append(torch.sort(leaf, stable=True).indices)
        c = torch.bincount(leaf, minlength=L + 1)[:L]
        count.append(c)
        begin.append(c.cumsum(0) - c)
    return tuple(torch.stack(v).int() for v in (order, begin, count))


def _tensors(case, gen):
    """The tensors of a list, each of its own memory or views of one buffer end to end: sizes
    spread as exp(N(0, 1)), those of a model, whatever the seed."""
    n, total = case["tensors"], case["total"]
    share = torch.randn(n, generator=torch.Generator().manual_seed(n)).exp().double()
    edges = ((share.cumsum(0) / share.sum()) * total).long().tolist()
    edges = [0] + edges[:-1] + [total]
    sizes = [b - a for a, b in zip(edges, edges[1:])]
    if case["flat"]:
        flat = _matrix(case, gen, 1, total, scale=0.01)[0]
        return flat, list(flat.split(sizes))
    types = ("f32", "bf16") if case["type"] == "mixed" else (case["type"],)
    return None, [_matrix(dict(type=types[i % len(types)]), gen, 1, k, scale=0.01)[0]
                  for i, k in enumerate(sizes)]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    state = {"case": case}
    if own:
        from lightgbm_rs_amd import HipBackend
        state["be"] = HipBackend(0)
    if case["op"] in ("norm", "clip"):
        state["flat"], state["grads"] = _tensors(case, gen)
        # of the norm that such gradients have
        state["limit"] = case["limit"] * 0.01 * math.sqrt(case["total"])
        if case["op"] == "clip":  # where the clipped gradients go
            state["flat_out"] = None if state["flat"] is None else torch.empty_like(state["flat"])
            state["out"] = ([torch.empty_like(g) for g in state["grads"]] if state["flat"] is None
                            else list(state["flat_out"].split([len(g) for g in state["grads"]])))
        return state
    N, K, H, G = case["rows"], case["cols"], case["outputs"], case["trees"] * case["leaves"]
    W = 2 * H if case["gated"] else H
    state["x"] = _matrix(case, gen, N, K, pad=case["pad"])
    state["w"] = _matrix(case, gen, G * W, K, scale=K ** -0.5).view(G, W, K)
    state["b"] = _matrix(case, gen, G, W, scale=0.5) if case["bias"] else None
    state["r"] = _matrix(case, gen, N, H, pad=case["pad"]) if case["residual"] else None
    state["groups"] = _groups(case, gen)
    if case["op"] == "train":
        state["dy"] = _matrix(case, gen, N, H, pad=case["pad"])
    return state


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    case, be = s["case"], s["be"]
    if case["op"] == "norm":
        return be.grad_norm(s["grads"])
    if case["op"] == "clip":
        norm = be.clip_grads(s["grads"], s["limit"], out=s["out"])
        return norm, (s["out"] if s["flat"] is None else s["flat_out"])
    form = dict(activation=case["act"], gated=case["gated"])
    if case["op"] == "layer":
        return be.leaf_layer(s["x"], s["w"], s["groups"], bias=s["b"], residual=s["r"], **form)
    y, z = be.leaf_layer(s["x"], s["w"], s["groups"], bias=s["b"], residual=s["r"], keep=True, **form)
    dx, dw, db = be.leaf_layer_grad(s["dy"], z, s["x"], s["w"], s["groups"], bias=case["bias"], **form)
    return (y, dx, dw, db) if case["bias"] else (y, dx, dw)


def _run_plain(s):
    if s["case"]["op"] in ("norm", "clip"):
        return _plain_clip(s)
    return _plain_layer(s)


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).double().sum().sqrt()
    if s["case"]["op"] == "norm":
        return norm.float()
    scale = (s["limit"] / norm).clamp(max=1.0).float()
    clipped = [(g.float() * scale).to(g.dtype) for g in s["grads"]]
    return norm.float(), (clipped if s["flat"] is None else torch.cat(clipped))


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z / (1 + (-z).exp())
    if act == "sigmoid":
        return 1 / (1 + (-z).exp())
    if act == "gelu":
        return 0.5 * z * (1 + (z * math.sqrt(0.5)).erf())
    u = math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)
    return 0.5 * z * (1 + u.tanh())


def _slope(z, act):
    """The activation's derivative."""
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).float()
    if act in ("silu", "sigmoid"):
        p = 1 / (1 + (-z).exp())
        return p * (1 - p) if act == "sigmoid" else p * (1 + z * (1 - p))
    if act == "gelu":
        return (0.5 * (1 + (z * math.sqrt(0.5)).erf())
                + z * (-0.5 * z * z).exp() * (1 / math.sqrt(2 * math.pi)))
    c = math.sqrt(2 / math.pi)
    t = (c * (z + 0.044715 * z * z * z)).tanh()
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain_layer(s):
    """Rows taken in the order of their leaves; products by leaf, or for small work by a copy
    of its weights for every row."""
    case, x, w, b = s["case"], s["x"], s["w"], s["b"]
    N, K, T, L, act = case["rows"], case["cols"], case["trees"], case["leaves"], case["act"]
    order, begin, count = s["groups"]
    H, W = case["outputs"], w.shape[1]
    small = N * T * K * W <= 20000000
    if small:
        # the leaf of every place in the order; L: in none
        ends = (begin + count).contiguous()  # leaves stand in the order of their numbers
        place = torch.arange(N, device=x.device, dtype=torch.int32).expand(T, N).contiguous()
        at = torch.searchsorted(ends, place, right=True)
        there = (at < L).flatten()[:, None]
        at = (at.clamp(max=L - 1) + torch.arange(T, device=x.device)[:, None] * L).flatten()
        rows = order.flatten().long()
        wr = w[at].float()
        xr = x[rows].float()
        z = (wr * xr[:, None, :]).sum(2)
        if b is not None:
            z = z + b[at].float()
    else:
        sizes = count.flatten().tolist()
        hit = [g for g in range(T * L) if sizes[g]]
        starts = (begin + torch.arange(T, device=x.device)[:, None] * N).flatten().tolist()
        of = order.flatten().long()
        rows = [of[starts[g]:starts[g] + sizes[g]] for g in hit]
        there = None
        xs = [x[r].float() for r in rows]
        z = torch.cat([v @ w[g].float().t() if b is None else v @ w[g].float().t() + b[g].float()
                       for v, g in zip(xs, hit)])
        rows = torch.cat(rows)
    if case["gated"]:
        zg, zu = z[:, :H], z[:, H:]
        f = _act(zg, act) * zu
    else:
        f = _act(z, act)
    if there is not None:
        f = torch.where(there, f, 0.0)
    y = torch.zeros((N, H), device=x.device) if s["r"] is None else s["r"].float()
    y = y.index_add(0, rows, f).to(x.dtype)
    if case["op"] == "layer":
        return y
    d = s["dy"][rows].float()
    if there is not None:
        d = torch.where(there, d, 0.0)
    dz = torch.cat([d * zu * _slope(zg, act), d * _act(zg, act)], 1) if case["gated"] else d * _slope(z, act)
    dx = torch.zeros((N, K), device=x.device)
    dw = torch.zeros(w.shape, device=x.device)
    db = torch.zeros(w.shape[:2], device=x.device)
    if small:
        dx.index_add_(0, rows, (wr * dz[:, :, None]).sum(1))
        dw.index_add_(0, at, dz[:, :, None] * xr[:, None, :])
        db.index_add_(0, at, dz)
    else:
        parts = dz.split([sizes[g] for g in hit])
        dx.index_add_(0, rows, torch.cat([p @ w[g].float() for p, g in zip(parts, hit)]))
        dw[hit] = torch.stack([p.t() @ v for p, v in zip(parts, xs)])
        db[hit] = torch.stack([p.sum(0) for p in parts])
    dx, dw, db = dx.to(x.dtype), dw.to(x.dtype), db.to(x.dtype)
    return (y, dx, dw, db) if case["bias"] else (y, dx, dw)


# ---- the same in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] in ("norm", "clip"):
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["grads"]))
        norm64 = torch.tensor(norm, dtype=torch.float64, device=DEVICE)
        if case["op"] == "norm":
            return norm64
        if norm > s["limit"]:
            clipped = [g.double() / (norm / s["limit"]) for g in s["grads"]]
        else:
            clipped = [g.double() for g in s["grads"]]
        return norm64, (clipped if s["flat"] is None else torch.cat(clipped))
    F = torch.nn.functional
    fn = {"none": lambda v: v * 1.0, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "sigmoid": torch.sigmoid,
          "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}[case["act"]]
    H, train = case["outputs"], case["op"] == "train"
    order, begin, count = (v.cpu() for v in s["groups"])
    y = torch.zeros((case["rows"], H), device=DEVICE, dtype=torch.float64)
    if s["r"] is not None:
        y += s["r"]
    if train:
        dx = torch.zeros((case["rows"], case["cols"]), device=DEVICE, dtype=torch.float64)
        dw = torch.zeros(s["w"].shape, device=DEVICE, dtype=torch.float64)
        db = torch.zeros(s["w"].shape[:2], device=DEVICE, dtype=torch.float64)
    for g in range(case["trees"] * case["leaves"]):
        t, leaf = divmod(g, case["leaves"])
        b0, c = int(begin[t, leaf]), int(count[t, leaf])
        if not c:
            continue
        n = order[t, b0:b0 + c].to(DEVICE).long()
        x, w = s["x"][n].double(), s["w"][g].double()
        z = torch.mm(x, w.t().contiguous())
        if s["b"] is not None:
            z += s["b"][g].double()
        z.requires_grad_(train)
        f = fn(z[:, :H]) * z[:, H:] if case["gated"] else fn(z)
        y.index_add_(0, n, f.detach())
        if train:
            dz, = torch.autograd.grad(f, z, s["dy"][n].double())
            dx.index_add_(0, n, torch.mm(dz, w))
            dw[g] = torch.mm(dz.t().contiguous(), x)
            db[g] = dz.sum(0)
    if not train:
        return y
    return (y, dx, dw, db) if case["bias"] else (y, dx, dw)


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    e = SIZES[case["type"]]
    if case["op"] in ("norm", "clip"):
        n = case["total"]
        return {"bytes": e * n if case["op"] == "norm" else 2 * e * n, "flops": 2 * n}
    N, K, H, T = case["rows"], case["cols"], case["outputs"], case["trees"]
    W = 2 * H if case["gated"] else H
    hit = min(T * case["leaves"], N * T)  # leaves that can have rows
    maps = e * hit * W * (K + (1 if case["bias"] else 0))
    flops = 2 * N * T * W * K + 8 * N * T * W
    forward = e * N * (K + H + (H if case["residual"] else 0)) + maps + 4 * N * T
    if case["op"] == "layer":
        return {"bytes": forward, "flops": flops}
    # the gradients: dy and dx once, dW and db of every leaf
    return {"bytes": forward + e * N * (H + K) + e * T * case["leaves"] * W * (K + 1), "flops": 3 * flops}
