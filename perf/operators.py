"""The operators around a forest's leaves, as cases to be timed and checked.

A tree sends every row to a leaf; a leaf may hold a linear map of its own (a linear leaf,
or an expert with several outputs), and the class scores that come out are turned into
answers.  The operators:

  groups    the rows of every leaf from the leaf of every row (`leaf_groups`)
  product   y[n] = sum over trees of W[t, leaf] x[n] + b[t, leaf] (`leaf_product`)
  grads     its gradients: dx, dW, db (`leaf_product_dx`, `leaf_product_dw`)
  dropout   elements or whole rows dropped by a counter-based generator (`dropout`)
  scores    penalties for repeated classes, biases and masks on class scores, raw or as
            probabilities (`adjust_scores`)

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
TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MASK32 = 0xFFFFFFFF

GROUPS = dict(op="groups", rows=1000, trees=1, leaves=31, lost=0.0)
PRODUCT = dict(op="product", rows=1000, cols=28, outputs=1, trees=1, leaves=31, type="f32",
               bias=True, lost=0.0, pad=0)
DROPOUT = dict(op="dropout", rows=1000, cols=2, type="f32", p=0.1, by="element", pad=0)
SCORES = dict(op="scores", rows=64, classes=10, type="f64", kind="transformed", bias=True,
              masks=0, history=0, per_row=False, pad=0)


def listed():
    return [
        # the dispatch of an online request: a few rows through every tree of a forest
        dict(GROUPS, name="groups_request", rows=64, trees=100),
        # the dispatch of a whole training table through one large tree
        dict(GROUPS, name="groups_table", rows=10500000, leaves=255),
        # an online request to a forest of linear leaves: one output, tiny leaves
        dict(PRODUCT, name="product_request", rows=64, trees=100),
        # batch scoring of ten classes by the linear leaves of one tree
        dict(PRODUCT, name="product_classes", rows=2000000, cols=100, outputs=10, leaves=127),
        # a batch through wide experts: matrix products of ragged sizes
        dict(PRODUCT, name="product_experts", rows=40007, cols=2000, outputs=2048, type="bf16"),
        # a few rows through wide experts: the weights of the experts that are hit
        dict(PRODUCT, name="product_few", rows=16, cols=4096, outputs=4096, type="f16"),
        # gradients of the linear leaves of one tree over a table
        dict(PRODUCT, name="grads_classes", op="grads", rows=1000003, cols=100, outputs=10,
             leaves=63),
        # gradients of wide experts where each row goes to two of them
        dict(PRODUCT, name="grads_experts", op="grads", rows=16389, cols=2048, outputs=2048,
             leaves=15, trees=2, type="bf16"),
        # bagging: the gradient pairs of whole rows
        dict(DROPOUT, name="dropout_rows", rows=10500000, p=0.3, by="row"),
        # the inputs of wide experts
        dict(DROPOUT, name="dropout_inputs", rows=32771, cols=4096, type="bf16"),
        # a batch of class scores to probabilities, with prior corrections and the classes
        # that each row may have
        dict(SCORES, name="scores_classes", rows=2000000, masks=1000),
        # few rows over many classes, with what each row was given before
        dict(SCORES, name="scores_vocabulary", rows=64, classes=128007, type="bf16", masks=7,
             history=1000, per_row=True),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("groups", "product", "product", "grads", "dropout", "scores"))
    if op == "groups":
        trees = rng.choice((1, 1, _between(rng, 2, 200)))
        return dict(GROUPS, rows=_between(rng, 1, 10000000 // trees), trees=trees,
                    leaves=rng.choice((2, 15, 31, 63, 127, 255, 1000)),
                    lost=rng.choice((0.0, 0.0, 0.1)))
    if op in ("product", "grads"):
        trees = rng.choice((1, 1, 1, 2, 5, 50))
        case = dict(PRODUCT, op=op, trees=trees, leaves=rng.choice((2, 7, 15, 31, 127)),
                    type=rng.choice(("f32", "bf16", "f16")), bias=rng.choice((True, False)),
                    lost=rng.choice((0.0, 0.0, 0.1)), pad=rng.choice((0, 0, 1, 8)))
        case["cols"] = _between(rng, 1, 4096)
        case["outputs"] = rng.choice((1, _between(rng, 2, 32), _between(rng, 33, 4096)))
        weights = trees * case["leaves"] * case["cols"] * case["outputs"]
        if weights > 500000000:  # the gradient of the weights is as large in 32 bits
            case["trees"] = 1
            case["leaves"] = min(case["leaves"], 15)
        # no more rows than 150 GFLOP or a table of 800 MB give
        most = min(75e9 / (case["cols"] * case["outputs"] * case["trees"]),
                   2e8 / (max(case["cols"], case["outputs"]) * case["trees"]), 2e6)
        case["rows"] = _between(rng, 1, max(1, int(most)))
        return case
    if op == "dropout":
        by = rng.choice(("element", "row"))
        cols = 2 if by == "row" else _between(rng, 1, 8192)
        return dict(DROPOUT, by=by, cols=cols, rows=_between(rng, 1, int(6e7 / cols)),
                    type=rng.choice(("f32", "bf16", "f16")), pad=rng.choice((0, 0, 3)),
                    p=rng.choice((0.0, 0.05, 0.1, 0.3, 0.5, 0.9)))
    classes = rng.choice((_between(rng, 2, 300), _between(rng, 300, 150000)))
    return dict(SCORES, classes=classes, rows=_between(rng, 1, max(1, min(1000000, int(1.5e7 / classes)))),
                type=rng.choice(("f64", "f32", "bf16", "f16")), bias=rng.choice((True, False)),
                kind=rng.choice(("raw", "transformed")), masks=rng.choice((0, 1, 5)),
                history=rng.choice((0, 3, 50)) if classes < 300 else rng.choice((0, 100, 3000)),
                per_row=rng.choice((True, False)), pad=rng.choice((0, 0, 1)))


# ---- inputs -----------------------------------------------------------------------------

def _matrix(case, gen, rows, cols, scale=1.0, pad=0, dtype=None):
    """N(0, 1) * scale; `pad` columns more in memory than in the matrix."""
    dtype = dtype or TYPES[case["type"]]
    out = torch.empty((rows, cols + pad), device=DEVICE, dtype=dtype)
    step = max(1, 50000000 // (cols + pad))
    for r in range(0, rows, step):
        b = out[r:r + step]
        b.copy_(torch.randn(b.shape, generator=gen, device=DEVICE) * scale)
    return out[:, :cols]


def _leaves(case, gen):
    """The leaf of every row in every tree: sizes spread as exp(N(0, 1)), one leaf in ten
    without rows; -1 where a row is lost (a tree that it does not take part in)."""
    N, T, L = case["rows"], case["trees"], case["leaves"]
    leaf = torch.empty((N, T), device=DEVICE, dtype=torch.int32)
    for t in range(T):
        size = torch.randn(L, generator=gen, device=DEVICE).exp()
        size[torch.rand(L, generator=gen, device=DEVICE) < 0.1] = 0
        size[int(torch.randint(L, (1,), generator=gen, device=DEVICE))] += 0.5
        edges = (size.cumsum(0) / size.sum()).contiguous()
        u = torch.rand(N, generator=gen, device=DEVICE)
        leaf[:, t] = torch.bucketize(u, edges, right=True).clamp_(max=L - 1).int()
    if case["lost"]:
        leaf[torch.rand((N, T), generator=gen, device=DEVICE) < case["lost"]] = -1
    return leaf


def _groups(leaf, leaves):
    """order [trees, rows], begin and count [trees, leaves]: the rows of a tree by their
    leaf, those of one leaf ascending, those in no leaf last."""
    trees = leaf.shape[1]
    key = leaf.t().long()
    key = torch.where((key < 0) | (key >= leaves), leaves, key)
    order = torch.sort(key, dim=1, stable=True).indices
    base = torch.arange(trees, device=leaf.device)[:, None] * (leaves + 1)
    count = torch.zeros(trees * (leaves + 1), dtype=torch.int64, device=leaf.device)
    count.index_add_(0, (key + base).flatten(), torch.ones_like(key).flatten())
    count = count.view(trees, leaves + 1)[:, :leaves]
    begin = count.cumsum(1) - count
    return order.int(), begin.int(), count.int()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    state = {"case": case, "seed": int(seed)}
    if own:
        from lightgbm_rs_amd import HipBackend, LeafGroups
        state["be"] = HipBackend(0)
    N = case["rows"]
    if case["op"] == "groups":
        state["leaf"] = _leaves(case, gen)
        return state
    if case["op"] in ("product", "grads"):
        K, M, G = case["cols"], case["outputs"], case["trees"] * case["leaves"]
        state["x"] = _matrix(case, gen, N, K, pad=case["pad"])
        state["w"] = _matrix(case, gen, G * M, K, scale=K ** -0.5).view(G, M, K)
        state["b"] = _matrix(case, gen, G, M) if case["bias"] else None
        if case["op"] == "grads":
            state["dy"] = _matrix(case, gen, N, M, pad=case["pad"])
        groups = _groups(_leaves(case, gen), case["leaves"])
        state["groups"] = LeafGroups(*groups) if own else groups
        return state
    if case["op"] == "dropout":
        state["x"] = _matrix(case, gen, N, case["cols"], pad=case["pad"])
        return state
    V = case["classes"]
    # scores of a trained model: a few classes stand out
    state["x"] = _matrix(case, gen, N, V, scale=2.0, pad=case["pad"])
    state["bias"] = _matrix(case, gen, 1, V)[0] if case["bias"] else None
    state["mask"] = state["mask_rows"] = state["ids"] = state["offsets"] = None
    if case["masks"]:
        words = (V + 31) // 32
        bits = torch.randint(-2 ** 31, 2 ** 31, (2, case["masks"], words), generator=gen,
                             device=DEVICE).int()
        state["mask"] = bits[0] | bits[1]
        state["mask"][0] = bits[0][0] & bits[1][0]
        # the mask of every row; -1: every class may be answered
        state["mask_rows"] = torch.randint(-1, case["masks"], (N,), generator=gen, device=DEVICE).int()
    if case["history"]:
        length = torch.rand(N, generator=gen, device=DEVICE) ** 2 * 3 * case["history"]
        offsets = torch.zeros(N + 1, dtype=torch.int64, device=DEVICE)
        offsets[1:] = length.long().cumsum(0)
        state["offsets"] = offsets
        u = torch.rand(int(offsets[-1]), generator=gen, device=DEVICE)
        # classes that come back: low numbers more often
        state["ids"] = (u ** 3 * V).int().clamp_(max=V - 1)
    state["penalties"] = (1.2, 0.1, 0.3)
    if case["per_row"]:
        p = torch.rand((N, 3), generator=gen, device=DEVICE)
        state["penalties"] = p + torch.tensor([0.8, -0.2, 0.0], device=DEVICE)
    return state


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    case, be = s["case"], s["be"]
    if case["op"] == "groups":
        g = be.leaf_groups(s["leaf"], case["leaves"])
        return g.order, g.begin, g.count
    if case["op"] == "product":
        return be.leaf_product(s["x"], s["w"], s["groups"], bias=s["b"])
    if case["op"] == "grads":
        dx = be.leaf_product_dx(s["dy"], s["w"], s["groups"])
        dw, db = be.leaf_product_dw(s["dy"], s["x"], s["groups"], bias=case["bias"])
        return (dx, dw, db) if case["bias"] else (dx, dw)
    if case["op"] == "dropout":
        return be.dropout(s["x"], case["p"], s["seed"], by=case["by"])
    repetition, frequency, presence = (1.0, 0.0, 0.0) if case["per_row"] else s["penalties"]
    return be.adjust_scores(s["x"], kind=case["kind"], bias=s["bias"], mask=s["mask"],
                            mask_rows=s["mask_rows"], ids=s["ids"], offsets=s["offsets"],
                            repetition=repetition, frequency=frequency, presence=presence,
                            penalties=s["penalties"] if case["per_row"] else None)


def _run_plain(s):
    case = s["case"]
    if case["op"] == "groups":
        return _groups(s["leaf"], case["leaves"])
    if case["op"] == "product":
        return _plain_product(s)
    if case["op"] == "grads":
        return _plain_grads(s)
    if case["op"] == "dropout":
        return _plain_dropout(s)
    return _plain_scores(s)


def _few(case):
    """Whether a copy of the weights for every row and tree is small."""
    return case["rows"] * case["trees"] * case["cols"] * case["outputs"] <= 10000000


def _leaf_of(groups, leaves):
    """The leaf of every row, [rows, trees], back from the groups (`leaves`: in none)."""
    order, begin, count = (v.long() for v in groups)
    place = torch.arange(order.shape[1], device=order.device)
    by_end = torch.sort(begin + count, dim=1).values
    # leaves stand in order of their numbers here, so the ends ascend
    leaf = torch.searchsorted(by_end, place.expand(order.shape).contiguous(), right=True)
    out = torch.empty_like(leaf)
    out.scatter_(1, order, leaf.clamp(max=leaves))
    return out.t()


def _each_leaf(groups):
    """(leaf of the forest, its rows) for every leaf that has rows."""
    order, begin, count = groups
    for t, (bs, cs) in enumerate(zip(begin.tolist(), count.tolist())):
        for l, (b, c) in enumerate(zip(bs, cs)):
            if c:
                yield t * len(bs) + l, order[t, b:b + c].long()


def _plain_product(s):
    case, x, w, b = s["case"], s["x"].float(), s["w"], s["b"]
    N, M, T, L = case["rows"], case["outputs"], case["trees"], case["leaves"]
    if _few(case):
        leaf = _leaf_of(s["groups"], L)
        at = (leaf.clamp(max=L - 1) + torch.arange(T, device=x.device) * L)
        y = (w[at].float() * x[:, None, None, :]).sum(3)
        if b is not None:
            y = y + b[at].float()
        return (y * (leaf < L)[:, :, None]).sum(1).to(s["x"].dtype)
    y = torch.zeros((N, M), device=x.device)
    for g, rows in _each_leaf(s["groups"]):
        part = x[rows] @ w[g].float().t()
        y[rows] += part if b is None else part + b[g].float()
    return y.to(s["x"].dtype)


def _plain_grads(s):
    case, x, w, dy = s["case"], s["x"].float(), s["w"], s["dy"].float()
    dx = torch.zeros_like(x)
    dw = torch.zeros(w.shape, device=x.device)
    db = torch.zeros(w.shape[:2], device=x.device)
    for g, rows in _each_leaf(s["groups"]):
        d = dy[rows]
        dx[rows] += d @ w[g].float()
        dw[g] = d.t() @ x[rows]
        db[g] = d.sum(0)
    dx = dx.to(s["x"].dtype)
    return (dx, dw, db) if case["bias"] else (dx, dw)


def _philox(block, seed):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
    1, 2, 3", 2011) of the counter (block, 0) under the key `seed`: four 32-bit words."""
    k0, k1 = seed & MASK32, (seed >> 32) & MASK32
    c0, c1 = block & MASK32, block >> 32
    c2, c3 = torch.zeros_like(block), torch.zeros_like(block)
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products, wrapping
        c0, c1, c2, c3 = (((b >> 32) & MASK32) ^ c1 ^ k0, b & MASK32,
                          ((a >> 32) & MASK32) ^ c3 ^ k1, a & MASK32)
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    return c0, c1, c2, c3


def _plain_dropout(s):
    """Unit e (an element in row-major order, or a row) is kept where 16-bit field e % 8 of
    block e / 8 is at least round(65536 p); what is kept is divided by the share kept."""
    case, x = s["case"], s["x"]
    t = int(round(case["p"] * 65536))
    units = x.numel() if case["by"] == "element" else len(x)
    words = _philox(torch.arange((units + 7) // 8, device=x.device), s["seed"])
    fields = torch.stack([(c >> shift) & 0xFFFF for c in words for shift in (0, 16)], 1)
    keep = (fields >= t).flatten()[:units]
    keep = keep.view(x.shape) if case["by"] == "element" else keep[:, None]
    scale = 65536 / (65536 - t)
    return torch.where(keep, x.float() * scale, 0.0).to(x.dtype)


def _plain_scores(s):
    case, x = s["case"], s["x"]
    N, V = x.shape
    y = x if x.dtype == torch.float64 else x.float()
    if s["ids"] is not None:
        row = torch.repeat_interleave(torch.arange(N, device=x.device), s["offsets"].diff())
        count = torch.zeros(N * V, dtype=torch.int32, device=x.device)
        count.index_add_(0, row * V + s["ids"].long(), torch.ones_like(s["ids"]))
        count = count.view(N, V)
        if case["per_row"]:
            repetition, frequency, presence = (v.to(y.dtype) for v in s["penalties"].split(1, 1))
        else:
            repetition, frequency, presence = s["penalties"]
        seen = torch.where(y > 0, y / repetition, y * repetition) - frequency * count - presence
        y = torch.where(count > 0, seen, y)
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["mask"] is not None:
        at = torch.arange(V, device=x.device)
        allowed = ((s["mask"][:, at // 32] >> (at % 32).int()) & 1).bool()
        m = s["mask_rows"].long()
        y = torch.where(allowed[m.clamp(min=0)] | (m < 0)[:, None], y, -math.inf)
    if case["kind"] == "transformed":
        top = y.amax(1, keepdim=True)
        p = (y - torch.where(top == -math.inf, 0.0, top)).exp()
        total = p.sum(1, keepdim=True)
        y = p / torch.where(total == 0, 1.0, total)
    return y.to(x.dtype)


# ---- the same in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"groups": _groups64, "product": _product64, "grads": _product64,
            "dropout": _dropout64, "scores": _scores64}[case["op"]](case, s)


def _groups64(case, s):
    leaf, L = s["leaf"], case["leaves"]
    order, begin, count = [], [], []
    # a row's key holds its leaf and its number, so that an ordinary sort is enough
    n = torch.arange(len(leaf), device=leaf.device)
    for t in range(leaf.shape[1]):
        l = leaf[:, t].long()
        l = torch.where((l >= 0) & (l < L), l, L)
        order.append(torch.sort(l * len(leaf) + n).values % len(leaf))
        c = torch.bincount(l, minlength=L + 1)[:L]
        count.append(c)
        begin.append(torch.cat([c.new_zeros(1), c.cumsum(0)[:-1]]))
    return tuple(torch.stack(v).int() for v in (order, begin, count))


def _product64(case, s):
    x, w, b, grads = s["x"].double(), s["w"], s["b"], case["op"] == "grads"
    N, K, M, L = case["rows"], case["cols"], case["outputs"], case["leaves"]
    order, begin, count = (v.cpu() for v in s["groups"])
    dy = s["dy"].double() if grads else None
    out = torch.zeros((N, K if grads else M), device=DEVICE, dtype=torch.float64)
    dw = torch.zeros(w.shape, device=DEVICE, dtype=torch.float64) if grads else None
    db = torch.zeros(w.shape[:2], device=DEVICE, dtype=torch.float64) if grads else None
    for g in range(case["trees"] * L):
        t, l = divmod(g, L)
        c = int(count[t, l])
        if not c:
            continue
        rows = order[t, int(begin[t, l]):int(begin[t, l]) + c].to(DEVICE).long()
        wg = w[g].double()
        if grads:
            out.index_add_(0, rows, torch.mm(dy[rows], wg))
            dw[g] = torch.mm(dy[rows].t().contiguous(), x[rows])
            db[g] = dy[rows].sum(0)
        else:
            y = torch.mm(x[rows], wg.t().contiguous())
            out.index_add_(0, rows, y if b is None else y + b[g].double())
    if not grads:
        return out
    return (out, dw, db) if case["bias"] else (out, dw)


def _dropout64(case, s):
    x, seed = s["x"], s["seed"]
    t = int(round(case["p"] * 65536))
    units = x.numel() if case["by"] == "element" else len(x)
    block = torch.arange((units + 7) // 8, device=DEVICE)

    def product(v, m):
        """(high, low) 32 bits of v * m by 16-bit limbs."""
        lo, hi = v & 0xFFFF, v >> 16
        low = lo * (m & 0xFFFF)
        mid = hi * (m & 0xFFFF) + lo * (m >> 16) + (low >> 16)
        return hi * (m >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (low & 0xFFFF)

    c = [block % 2 ** 32, block // 2 ** 32, torch.zeros_like(block), torch.zeros_like(block)]
    for r in range(10):
        k = [(seed + 0x9E3779B9 * r) % 2 ** 32, ((seed >> 32) + 0xBB67AE85 * r) % 2 ** 32]
        h0, l0 = product(c[0], 0xD2511F53)
        h1, l1 = product(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k[0], l1, h0 ^ c[3] ^ k[1], l0]
    field = torch.empty((len(block), 8), device=DEVICE, dtype=torch.int64)
    for j in range(8):
        field[:, j] = c[j // 2] // (65536 if j % 2 else 1) % 65536
    keep = field.view(-1)[:units] >= t
    keep = keep.view(x.shape) if case["by"] == "element" else keep.view(-1, 1).expand(x.shape)
    out = torch.zeros(x.shape, device=DEVICE, dtype=torch.float64)
    out[keep] = x[keep].double() / (1 - t / 65536)
    return out


def _scores64(case, s):
    x, V = s["x"], case["classes"]
    out = torch.empty(x.shape, device=DEVICE, dtype=torch.float64)
    step = max(1, 40000000 // V)
    if s["mask"] is not None:
        bit = torch.arange(32, device=DEVICE)
        masked = (s["mask"].long()[:, :, None] // 2 ** bit % 2 == 0).flatten(1)[:, :V]
    for r in range(0, len(x), step):
        y = x[r:r + step].double()
        n = len(y)
        if s["ids"] is not None:
            off = s["offsets"][r:r + n + 1]
            at = torch.arange(int(off[0]), int(off[-1]), device=DEVICE)
            row = torch.searchsorted(off, at, right=True) - 1
            count = torch.bincount(row * V + s["ids"][int(off[0]):int(off[-1])].long(),
                                   minlength=n * V).view(n, V)
            if case["per_row"]:
                rep, fre, pre = s["penalties"][r:r + n].double().t()[:, :, None]
            else:
                rep, fre, pre = (torch.tensor(float(v), device=DEVICE) for v in s["penalties"])
            ratio = torch.where(y > 0, 1 / rep, rep)
            y = y * torch.where(count > 0, ratio, 1.0) - fre * count - pre * count.clamp(max=1)
        if s["bias"] is not None:
            y = y + s["bias"].double()
        if s["mask"] is not None:
            m = s["mask_rows"][r:r + n].long()
            y[(masked[m.clamp(min=0)]) & (m >= 0)[:, None]] = -math.inf
        if case["kind"] == "transformed":
            none = torch.isneginf(y).all(1)
            y = torch.softmax(y, 1)
            y[none] = 0
        out[r:r + n] = y
    return out


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    N = case["rows"]
    if case["op"] == "groups":
        T, G = case["trees"], case["trees"] * case["leaves"]
        return {"bytes": 8 * N * T + 8 * G, "flops": 0}
    e = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    if case["op"] in ("product", "grads"):
        K, M, T, G = case["cols"], case["outputs"], case["trees"], case["trees"] * case["leaves"]
        hit = min(G, N * T)  # leaves that can have rows
        flops = 2 * N * T * K * M
        common = e * N * (K + M) + e * hit * M * K + 4 * N * T
        if case["op"] == "product":
            return {"bytes": common, "flops": flops}
        return {"bytes": common + e * N * K + 4 * G * M * (K + 1), "flops": 2 * flops}
    if case["op"] == "dropout":
        return {"bytes": 2 * e * N * case["cols"], "flops": N * case["cols"]}
    V = case["classes"]
    mask = case["masks"] * V / 8 + 4 * N if case["masks"] else 0
    return {"bytes": 2 * e * N * V + mask + 4 * N * case["history"], "flops": 8 * N * V}
