"""Checks of the operators around a forest's leaves against leaf_ops_oracle.py, run by
leaf_ops_worker.py on the GPU.

Tolerances.  u = finfo(type).eps / 2 is the largest relative error of a rounding to the
type (and tiny / 2 * eps the absolute one where it is subnormal), U = 2^-24 that of float32.  A sum of n float32 terms
whose magnitudes add up to S is off by at most n U S whatever its order (to first order;
twice that is allowed, for the matrix instructions' own adds), and a result y rounded to
the type by u |y| more.
"""
import ctypes as C

import numpy as np
import torch

from lightgbm_rs_amd import GainConfig, HipBackend, HipError, LeafGroups, Model
from tests import leaf_ops_oracle as oracle

DEV = "cuda:0"
TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24
_backend = []


def backend():
    if not _backend:
        _backend.append(HipBackend(0))
    return _backend[0]


def close():
    for b in _backend:
        b.close()
    _backend.clear()


def wide(t):
    return t.double().cpu().numpy()


def near(got, want, size, terms, dtype, what):
    """got (of a type) against want in 64 bits, a float32 sum of `terms` terms of `size`."""
    info = torch.finfo(dtype)
    # a value that is as good as at the border of the type's range rounds to infinity or not
    tol = info.eps / 2 * np.abs(want) * (1 + 2 * U) + 2 * (terms + 2) * U * size + info.tiny * info.eps
    got = wide(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.abs(got - want)
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(),
                           got[bad][:4], want[bad][:4], tol[bad][:4])


def matrix(rng, rows, cols, dtype, pad=0, lead=0):
    """N(0, 1) on the device; `pad` more columns a row and `lead` elements before the first
    row in memory, all NaN (nothing behind a row's end may matter)."""
    flat = torch.full((lead + rows * (cols + pad),), float("nan"), dtype=dtype)
    view = flat[lead:].view(rows, cols + pad)
    view[:, :cols] = torch.from_numpy(rng.standard_normal((rows, cols))).to(dtype)
    return flat.to(DEV)[lead:].view(rows, cols + pad)[:, :cols]


def leaves_of(rng, rows, trees, leaves, shape):
    """The leaf of every row: "even", "one" (all rows in one leaf), "skew" (sizes fall off,
    the last leaves empty), "lost" (a third in no leaf, by -1 and by numbers past the end)."""
    if shape == "one":
        return np.full((rows, trees), leaves - 1, np.int32)
    if shape == "skew":
        return np.minimum(rng.geometric(0.35, (rows, trees)) - 1, max(leaves - 2, 0)).astype(np.int32)
    leaf = rng.integers(0, leaves, (rows, trees)).astype(np.int32)
    if shape == "lost":
        leaf[rng.random((rows, trees)) < 0.2] = -1
        leaf[rng.random((rows, trees)) < 0.1] = leaves
        leaf[rng.random((rows, trees)) < 0.05] = -2 ** 31
        leaf[rng.random((rows, trees)) < 0.05] = 2 ** 31 - 1
    return leaf


def groups(rows, trees, leaves, shape, pad=0, seed=0):
    rng = np.random.default_rng(seed)
    leaf = leaves_of(rng, rows, trees, leaves, shape)
    t = torch.zeros((rows, trees + pad), dtype=torch.int32)
    t[:, :trees] = torch.from_numpy(leaf)
    g = backend().leaf_groups(t.to(DEV)[:, :trees], leaves)
    for got, want in zip(g, oracle.groups(leaf, leaves)):
        assert np.array_equal(got.cpu().numpy(), want)


def groups_many():
    """So many leaves that blocks for all of them along one axis pass 32 bits of threads."""
    rows, trees, leaves = 4097, 4200, 4095
    leaf = leaves_of(np.random.default_rng(0), rows, 1, leaves, "even")
    t = torch.from_numpy(leaf).to(DEV).int().expand(rows, trees).contiguous()
    for got, want in zip(backend().leaf_groups(t, leaves), oracle.groups(leaf, leaves)):
        assert bool((got == torch.from_numpy(want).to(DEV)).all())


def _case(rows, inputs, outputs, trees, leaves, dtype, shape, pad, seed):
    rng = np.random.default_rng(seed)
    leaf = leaves_of(rng, rows, trees, leaves, shape)
    g = LeafGroups(*(torch.from_numpy(v).to(DEV) for v in oracle.groups(leaf, leaves)))
    dt = TYPES[dtype]
    lead = 3 if pad % 2 else 0
    x = matrix(rng, rows, inputs, dt, pad, lead)
    dy = matrix(rng, rows, outputs, dt, pad, lead)
    w = matrix(rng, trees * leaves * outputs, inputs, dt, 0, lead).view(trees * leaves, outputs, inputs)
    b = matrix(rng, trees * leaves, outputs, dt, 0, lead)
    return leaf, g, x, dy, w, b


def product(rows, inputs, outputs, trees, leaves, dtype, shape="skew", pad=0, bias=True, seed=0):
    leaf, g, x, dy, w, b = _case(rows, inputs, outputs, trees, leaves, dtype, shape, pad, seed)
    b = b if bias else None
    y = backend().leaf_product(x, w, g, bias=b)
    want, size = oracle.product(wide(x), wide(w), None if b is None else wide(b), leaf, leaves)
    near(y, want, size, (inputs + 1) * trees, y.dtype, "y")
    # into the caller's strided output, whose gaps stay as they were
    room = torch.full((rows, outputs + 5), 7.0, dtype=y.dtype, device=DEV)
    out = room[:, 2:2 + outputs]
    assert backend().leaf_product(x, w, g, bias=b, out=out) is out
    assert torch.equal(out, y) and bool((room[:, :2] == 7).all()) and bool((room[:, 2 + outputs:] == 7).all())


def grads(rows, inputs, outputs, trees, leaves, dtype, shape="skew", pad=0, bias=True, seed=0):
    leaf, g, x, dy, w, b = _case(rows, inputs, outputs, trees, leaves, dtype, shape, pad, seed)
    be = backend()
    dx = be.leaf_product_dx(dy, w, g)
    want, size = oracle.product_dx(wide(dy), wide(w), leaf, leaves)
    near(dx, want, size, outputs * trees, dx.dtype, "dx")
    dw, db = be.leaf_product_dw(dy, x, g, bias=bias)
    w_want, w_size, b_want, b_size = oracle.product_dw(wide(dy), wide(x), leaf, leaves)
    assert dw.dtype == torch.float32
    near(dw, w_want, w_size, rows, torch.float32, "dw")
    if bias:
        near(db, b_want, b_size, rows, torch.float32, "db")
    else:
        assert db is None
    # the same bits every time
    dw2, db2 = be.leaf_product_dw(dy, x, g, bias=bias, out=torch.full_like(dw, 3.0))
    assert torch.equal(dw, dw2) and (db is None or torch.equal(db, db2))
    assert torch.equal(dx, be.leaf_product_dx(dy, w, g))


def differences():
    """The gradients against differences of the forward pass: it is linear in x, w and b, so
    a difference of any step is the gradient times the step, but for rounding."""
    leaf, g, x, dy, w, b = _case(37, 9, 4, 3, 5, "f32", "lost", 0, 5)
    be = backend()
    dx = be.leaf_product_dx(dy, w, g)
    dw, db = be.leaf_product_dw(dy, x, g)
    rng = np.random.default_rng(6)
    for name, t, grad in (("x", x, dx), ("w", w, dw), ("b", b, db)):
        step = torch.from_numpy(rng.standard_normal(tuple(t.shape))).float().to(DEV)
        a = {"x": x, "w": w, "b": b}
        lo = be.leaf_product(a["x"], a["w"], g, bias=a["b"])
        a[name] = t + step
        hi = be.leaf_product(a["x"], a["w"], g, bias=a["b"])
        change = ((hi.double() - lo.double()) * dy.double()).sum().item()
        want = (grad.double() * step.double()).sum().item()
        size = (hi.abs().double() + lo.abs().double()).mul(dy.abs().double()).sum().item()
        size += (grad.abs().double() * step.abs().double()).sum().item()
        # each y is off by at most 2 (30 + 2) U times its terms; their sum is at most about
        # eight times |y| here (30 terms of random signs: sqrt(30) = 5.5 on average)
        assert abs(change - want) <= 2 * 32 * U * 16 * size, (name, change, want, size)


def odd_tables(scale=1, inputs=8, outputs=4, dtype="f32"):
    """Tables that do not hold: ranges outside the order and rows outside the matrix are held
    back or passed over, and rows that stand nowhere are left as they were."""
    be, dt, rows = backend(), TYPES[dtype], 50 * scale
    rng = np.random.default_rng(2)
    x = matrix(rng, rows, inputs, dt)
    w = matrix(rng, 3 * outputs, inputs, dt).view(3, outputs, inputs)
    dy = matrix(rng, rows, outputs, dt)
    order = torch.arange(rows, dtype=torch.int32)
    order[7], order[8], order[9] = -5, rows, 2 ** 31 - 1
    sizes = [20 * scale, 10 * scale, 20 * scale]
    for begin, count in (([0, 20 * scale, 30 * scale], sizes), ([-4, 90 * scale, 30], [10, 10, 2000 * scale]),
                         ([0, 0, 0], [-3, rows, 0]), ([2 ** 31 - 1] * 3, [2 ** 31 - 1] * 3)):
        g = LeafGroups(order[None].to(DEV), torch.tensor([begin], dtype=torch.int32, device=DEV),
                       torch.tensor([count], dtype=torch.int32, device=DEV))
        y = be.leaf_product(x, w, g, out=torch.full((rows, outputs), 5.0, device=DEV, dtype=dt))
        dw, db = be.leaf_product_dw(dy, x, g)
        be.leaf_product_dx(dy, w, g)
        if count == sizes:
            leaf = np.repeat([0, 1, 2], sizes)[:, None].astype(np.int32)
            leaf[7:10] = -1
            want, size = oracle.product(wide(x), wide(w), None, leaf, 3)
            want[7:10] = 5.0
            near(y, want, size, inputs, dt, "y")
            w_want, w_size, b_want, b_size = oracle.product_dw(wide(dy), wide(x), leaf, 3)
            near(dw, w_want, w_size, rows, torch.float32, "dw")
            near(db, b_want, b_size, rows, torch.float32, "db")


def odd_tables_large():
    odd_tables(16, 200, 192, "bf16")


def any_order():
    """Leaves in any order of their ranges, as a grown tree's layout has them; NaN and
    infinities reach the rows and leaves that hold them and no others."""
    be = backend()
    rng = np.random.default_rng(3)
    leaf = rng.integers(0, 6, (300, 1)).astype(np.int32)
    place, order, begin, count = 0, [], np.zeros(6, np.int32), np.zeros(6, np.int32)
    for l in (3, 0, 5, 1, 4, 2):
        n = rng.permutation(np.flatnonzero(leaf[:, 0] == l))
        begin[l], count[l] = place, len(n)
        place += len(n)
        order.append(n)
    layout = {"indices": np.concatenate(order).astype(np.uint32), "leaf_begin": begin, "leaf_count": count}
    g = LeafGroups.from_layout(layout)
    for dtype in ("f32", "bf16"):
        x = matrix(rng, 300, 20, TYPES[dtype])
        w = matrix(rng, 6 * 3, 20, TYPES[dtype]).view(6, 3, 20)
        dy = matrix(rng, 300, 3, TYPES[dtype])
        x[17] = float("nan")
        dy[17] = float("inf")
        other = (leaf[:, 0] != leaf[17, 0])
        rest = np.arange(300) != 17
        y = be.leaf_product(x, w, g)
        dx = be.leaf_product_dx(dy, w, g)
        dw, db = be.leaf_product_dw(dy, x, g)
        x0, dy0 = wide(x), wide(dy)
        x0[17] = dy0[17] = 0
        want, size = oracle.product(x0, wide(w), None, leaf, 6)
        near(y[rest], want[rest], size[rest], 20, y.dtype, "y")
        assert bool(y[17].isnan().all())
        want, size = oracle.product_dx(dy0, wide(w), leaf, 6)
        near(dx[rest], want[rest], size[rest], 3, dx.dtype, "dx")
        assert not bool(dx[17].isfinite().any())
        w_want, w_size, b_want, b_size = oracle.product_dw(dy0, x0, leaf, 6)
        l = int(leaf[17, 0])
        keep = np.arange(6) != l
        near(dw[keep], w_want[keep], w_size[keep], 300, torch.float32, "dw")
        near(db[keep], b_want[keep], b_size[keep], 300, torch.float32, "db")
        assert bool(dw[l].isnan().all()) and not bool(db[l].isfinite().any()), other.sum()


def dropout(rows, cols, p, by="element", dtype="f32", pad=0, seed=1, offset=0):
    rng = np.random.default_rng(seed & 0xFFFF)
    dt = TYPES[dtype]
    x = matrix(rng, rows, cols, dt, pad, 1 if pad % 2 else 0)
    be = backend()
    units = rows if by == "row" else rows * cols
    keep, share = oracle.kept(units, p, seed, offset)
    keep = torch.from_numpy(keep).to(DEV)
    keep = keep[:, None].expand(rows, cols) if by == "row" else keep.view(rows, cols)
    scale = torch.tensor(1 / share if share else 0.0, dtype=torch.float32, device=DEV)
    want = torch.where(keep, (x.float() * scale).to(dt), torch.zeros((), dtype=dt, device=DEV))
    got = be.dropout(x, p, seed, offset, by=by)
    assert torch.equal(got, want)
    # dropped values do not matter, in place and by the gradient's call as well
    bad = torch.where(keep, x, torch.full((), float("nan"), dtype=dt, device=DEV))
    assert torch.equal(be.dropout(bad, p, seed, offset, by=by), want)
    room = torch.full((rows, cols + 3), 7.0, dtype=dt, device=DEV)
    room[:, 1:1 + cols] = bad
    inner = room[:, 1:1 + cols]
    assert be.dropout(inner, p, seed, offset, by=by, out=inner) is inner
    assert torch.equal(inner, want) and bool((room[:, 0] == 7).all()) and bool((room[:, 1 + cols:] == 7).all())
    if cols == 1 or by == "element":  # a vector, in place as well
        line = bad.reshape(-1)
        flat = want.reshape(-1)
        assert torch.equal(be.dropout(line, p, seed, offset, by=by), flat)
        assert be.dropout(line, p, seed, offset, by=by, out=line) is line
        assert torch.equal(line, flat)


def dropout_far():
    """Units past 2^32, where the counter's second word comes in."""
    rows, cols = 70001, 65537  # 4.59e9 elements
    x = torch.ones((rows, cols), dtype=torch.float16, device=DEV)
    y = backend().dropout(x, 0.25, 12345678901234567, 2 ** 40 + 3, out=x)
    t = 16384
    for e0 in (0, 2 ** 32 - 64, 2 ** 32 + 8, rows * cols // 8 * 8 - 800):
        words = oracle.philox(np.arange(e0 // 8, e0 // 8 + 100), 2 ** 40 + 3, 12345678901234567)
        fields = np.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)
        got = y.view(-1)[e0:e0 + 800].cpu().numpy() != 0
        assert np.array_equal(got, (fields >= t)[:len(got)]), e0
    kept = sum(int((y[r:r + 10000] != 0).sum()) for r in range(0, rows, 10000))
    # binomial: 6 standard deviations are 6 sqrt(n 3/16)
    assert abs(kept - 0.75 * rows * cols) <= 6 * (rows * cols * 3 / 16) ** 0.5


def _masks(rng, masks, V, density):
    bits = rng.random((masks, (V + 31) // 32 * 32)) < density
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


def scores(rows, classes, dtype, kind, bias=True, masks=0, history=0, per_row=False, pad=0, seed=0,
           by_row_masks=False):
    rng = np.random.default_rng(seed)
    dt = TYPES[dtype]
    x = matrix(rng, rows, classes, dt, pad, 1 if pad % 2 else 0)
    b = matrix(rng, 1, classes, dt)[0] if bias else None
    mask = mask_rows = ids = offsets = None
    if masks:
        mask = _masks(rng, masks, classes, 0.6)
        if not by_row_masks:
            mask_rows = rng.integers(-1, masks, rows).astype(np.int32)
        mask[0] = 0  # nothing allowed
        if masks > 1:
            mask[1] = 0
            mask[1, (classes - 1) // 32] = np.uint32(1) << np.uint32((classes - 1) % 32)  # one class
    pen = np.tile(np.array([[1.3, 0.25, 0.5]]), (rows, 1))
    if history:
        length = rng.integers(0, 2 * history + 1, rows)
        length[0] = 0
        offsets = np.concatenate([[0], np.cumsum(length)]).astype(np.int64)
        ids = (rng.random(offsets[-1]) ** 3 * (classes + 2)).astype(np.int32) - 1  # -1 and `classes` too
        if per_row:
            pen = np.stack([rng.uniform(0.5, 2, rows), rng.uniform(-1, 1, rows), rng.uniform(-1, 1, rows)], 1)
            pen = pen.astype(np.float32).astype(np.float64)
    up = lambda v, t=None: None if v is None else torch.from_numpy(v if t is None else v.view(t)).to(DEV)
    args = dict(kind=kind, bias=b, mask=up(mask, np.int32), mask_rows=up(mask_rows), ids=up(ids),
                offsets=up(offsets))
    if per_row and history:
        args["penalties"] = torch.from_numpy(pen).float().to(DEV)
    else:
        args.update(repetition=1.3, frequency=0.25, presence=0.5)
    got = backend().adjust_scores(x, **args)
    want, size = oracle.scores(wide(x), kind, None if b is None else wide(b), mask, mask_rows, ids, offsets, pen)
    u = 2.0 ** -53 if dtype == "f64" else U
    info = torch.finfo(dt)
    # s is off by at most 6 roundings of its terms
    delta = 6 * u * size
    if kind == "raw":
        tol = info.eps / 2 * np.abs(want) * (1 + 2 * U) + delta + info.tiny * info.eps
    else:
        # e^s by the offsets of s and of the maximum, exp itself (4 u), the sum of `classes`
        # terms and the division
        rel = 2 * delta.max(1, keepdims=True) + (classes + 12) * u
        tol = want * (rel + info.eps / 2 * (1 + rel)) + info.tiny * info.eps
        if dtype in ("f32", "f64"):  # results below the type's normal range may be flushed
            tol = tol + info.tiny
    g = wide(got)
    inf = ~np.isfinite(want)
    assert np.array_equal(g[inf], want[inf]) and bool(np.isfinite(g[~inf]).all())
    off = np.abs(np.where(inf, 0, g) - np.where(inf, 0, want))
    bad = ~(off <= np.where(inf, 0, tol))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), g[bad][:4], want[bad][:4], tol[bad][:4])
    if kind == "transformed":
        assert bool((g[want == 0] == 0).all())
    # in place, in a strided matrix
    room = torch.full((rows, classes + 3), 7.0, dtype=dt, device=DEV)
    inner = room[:, 1:1 + classes]
    inner.copy_(x)
    assert backend().adjust_scores(inner, out=inner, **args) is inner
    assert torch.equal(inner, got) and bool((room[:, 0] == 7).all()) and bool((room[:, 1 + classes:] == 7).all())


def scores_edges(dtype):
    """Infinities, NaN and the type's lowest value, masked and not."""
    dt = TYPES[dtype]
    be = backend()
    inf, nan, low = float("inf"), float("nan"), torch.finfo(dt).min
    V = 70
    x = torch.zeros((8, V), dtype=dt)
    mask = np.full((8, 3), 0xFFFFFFFF, np.uint32)
    x[0, 3], x[0, 69] = nan, inf          # both masked: no trace
    mask[0, 0] &= ~np.uint32(1 << 3)
    mask[0, 2] &= ~np.uint32(1 << 5)
    x[1, 3] = nan                          # not masked
    x[2, 3] = inf
    x[3] = -inf                            # nothing left without a mask
    x[4] = low                             # all alike
    x[5, :69] = low                        # all but one
    x[6] = -inf
    x[6, 40] = low                         # one class, at the lowest value
    mask[7] = 0
    x[7] = nan                             # nothing allowed
    m = torch.from_numpy(mask.view(np.int32)).to(DEV)
    raw = be.adjust_scores(x.to(DEV), mask=m).cpu()
    assert raw[0, 3] == -inf and raw[0, 69] == -inf and bool((raw[0, 4:69] == 0).all())
    assert raw[1, 3].isnan() and raw[2, 3] == inf and bool((raw[7] == -inf).all())
    assert torch.equal(raw[3:7], x[3:7])
    p = wide(be.adjust_scores(x.to(DEV), kind="transformed", mask=m))
    # sums of 68 and 70 float32 or float64 terms, all 1: exact; one division, one rounding
    eps = torch.finfo(dt).eps
    live = np.ones(V, bool)
    live[[3, 69]] = False
    assert (p[0, ~live] == 0).all() and np.allclose(p[0, live], 1 / 68, rtol=2 * eps, atol=0)
    assert np.isnan(p[1]).all()
    assert np.isnan(p[2, 3]) or p[2, 3] == 1
    assert (p[3] == 0).all() and (p[7] == 0).all()
    assert np.allclose(p[4], 1 / 70, rtol=2 * eps, atol=0)
    assert (p[5, :69] == 0).all() and p[5, 69] == 1
    assert (np.delete(p[6], 40) == 0).all() and p[6, 40] == 1


def scores_history():
    """Histories that do not hold: offsets that fall, or lie outside the ids."""
    be = backend()
    x = torch.ones((4, 5), dtype=torch.float32, device=DEV)
    ids = torch.tensor([1, 1, 2, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    offsets = torch.tensor([-7, 2, 1, 2 ** 62, 3], dtype=torch.int64, device=DEV)
    got = be.adjust_scores(x, ids=ids, offsets=offsets, frequency=0.25).cpu()
    want = torch.ones(4, 5)
    want[0, 1] = 0.5   # [0, 2)
    # row 1: [2, 1) is empty; row 2: [1, 5); row 3: [5, 3) is empty
    want[2, 1], want[2, 2] = 0.75, 0.75
    assert torch.equal(got, want)


def empty():
    """No rows: tables and gradients are zeros, the rest has nothing to write."""
    be = backend()
    g = be.leaf_groups(torch.zeros((0, 3), dtype=torch.int32, device=DEV), 4)
    assert g.order.shape == (3, 0) and not bool(g.begin.any()) and not bool(g.count.any())
    x = torch.zeros((0, 5), device=DEV)
    w = torch.zeros((12, 2, 5), device=DEV)
    assert be.leaf_product(x, w, g).shape == (0, 2)
    dy = torch.zeros((0, 2), device=DEV)
    assert be.leaf_product_dx(dy, w, g).shape == (0, 5)
    dw, db = be.leaf_product_dw(dy, x, g, out=torch.ones((12, 2, 5), device=DEV))
    assert not bool(dw.any()) and not bool(db.any())
    assert be.dropout(x, 0.5, 1).shape == (0, 5)
    assert be.adjust_scores(x, kind="transformed").shape == (0, 5)


def layouts():
    """Inputs with strided columns, expanded rows, one dimension."""
    be = backend()
    rng = np.random.default_rng(8)
    leaf = rng.integers(0, 4, (33, 2)).astype(np.int32)
    g = be.leaf_groups(torch.from_numpy(leaf.T.copy()).to(DEV).t(), 4)
    x = matrix(rng, 6, 33, torch.float32).t()
    w = matrix(rng, 6, 8 * 3, torch.float32).t().reshape(8, 3, 6)
    y = be.leaf_product(x, w.transpose(1, 2).contiguous().transpose(1, 2), g)
    assert torch.equal(y, be.leaf_product(x.contiguous(), w.contiguous(), g))
    row = x[:1].expand(33, 6)
    assert torch.equal(be.leaf_product(row, w, g), be.leaf_product(row.contiguous(), w, g))
    v = torch.arange(1000, device=DEV, dtype=torch.float32)
    d = be.dropout(v, 0.5, 9)
    assert torch.equal(d, be.dropout(v[None], 0.5, 9)[0])
    assert torch.equal(be.dropout(v[:, None], 0.5, 9, by="row")[:, 0], d)
    one = be.leaf_groups(torch.from_numpy(leaf[:, 0].copy()).to(DEV), 4)
    assert torch.equal(one.order[0], g.order[0])
    try:
        be.leaf_product(x, w, g, out=torch.empty((3, 33), device=DEV).t())
        raise AssertionError("a transposed out was taken")
    except ValueError:
        pass
    try:
        be.leaf_product_dx(x, w, g, out=x)
        raise AssertionError("shapes that do not fit were taken")
    except ValueError:
        pass
    square = matrix(rng, 8, 6, torch.float32).view(8, 1, 6).expand(8, 6, 6).contiguous()
    try:
        be.leaf_product(x, square, g, out=x)
        raise AssertionError("an output over an input was taken")
    except (HipError, ValueError):
        pass


def _together(be, leaf, x, w, b, bias, mask, ids, offsets, seed):
    """One step as a program that trains and answers makes it."""
    g = be.leaf_groups(leaf, w.shape[0] // leaf.shape[1])
    xd = be.dropout(x, 0.25, seed)
    y = be.leaf_product(xd, w, g, bias=b)
    p = be.adjust_scores(y, kind="transformed", bias=bias, mask=mask, ids=ids, offsets=offsets,
                         repetition=1.2, frequency=0.1, presence=0.2)
    dy = p * 0.5
    dx = be.dropout(be.leaf_product_dx(dy, w, g), 0.25, seed)
    dw, db = be.leaf_product_dw(dy, xd, g)
    return g.order, g.count, xd, y, p, dx, dw, db


def _together_inputs(seed, rows=203, inputs=40, outputs=10, trees=2, leaves=9, dtype="f32"):
    rng = np.random.default_rng(seed)
    leaf = torch.from_numpy(leaves_of(rng, rows, trees, leaves, "lost")).to(DEV)
    x = matrix(rng, rows, inputs, TYPES[dtype])
    w = matrix(rng, trees * leaves * outputs, inputs, TYPES[dtype]).view(-1, outputs, inputs)
    b = matrix(rng, trees * leaves, outputs, TYPES[dtype])
    bias = matrix(rng, 1, outputs, TYPES[dtype])[0]
    mask = torch.from_numpy(_masks(rng, rows, outputs, 0.7).view(np.int32)).to(DEV)
    offsets = torch.arange(rows + 1, device=DEV) * 3
    ids = torch.from_numpy(rng.integers(0, outputs, rows * 3).astype(np.int32)).to(DEV)
    return leaf, x, w, b, bias, mask, ids, offsets


def together(dtype):
    """The operators one after another against the oracle, each on what the one before
    gave."""
    be = backend()
    leaf, x, w, b, bias, mask, ids, offsets = _together_inputs(3, dtype=dtype)
    order, count, xd, y, p, dx, dw, db = _together(be, leaf, x, w, b, bias, mask, ids, offsets, 77)
    lf = leaf.cpu().numpy()
    assert np.array_equal(order.cpu().numpy(), oracle.groups(lf, 9)[0])
    keep, share = oracle.kept(x.numel(), 0.25, 77)
    keep = keep.reshape(x.shape)
    near(xd, np.where(keep, wide(x) / share, 0), np.abs(wide(x)), 1, x.dtype, "dropout")
    want, size = oracle.product(wide(xd), wide(w), wide(b), lf, 9)
    near(y, want, size, 41 * 2, y.dtype, "y")
    want, _ = oracle.scores(wide(y), "transformed", wide(bias), mask.cpu().numpy().view(np.uint32), None,
                            ids.cpu().numpy(), offsets.cpu().numpy(), np.tile([[1.2, 0.1, 0.2]], (203, 1)))
    # as in `scores`: |s| stays below 64 here, so s is off by 6 U 64, e^s by twice that
    tol = want * (2 * 6 * U * 64 + 22 * U + torch.finfo(p.dtype).eps / 2) + torch.finfo(p.dtype).tiny
    assert (np.abs(wide(y)) < 40).all() and (np.abs(wide(p) - want) <= tol).all()
    dy = wide((p * 0.5))
    want, size = oracle.product_dx(dy, wide(w), lf, 9)
    full = be.leaf_product_dx(p * 0.5, w, LeafGroups(*(torch.from_numpy(v).to(DEV) for v in oracle.groups(lf, 9))))
    near(full, want, size, 20, dx.dtype, "dx")
    near(dx, np.where(keep, wide(full) / share, 0), np.abs(wide(full)), 1, dx.dtype, "dropout of dx")
    w_want, w_size, b_want, b_size = oracle.product_dw(dy, wide(xd), lf, 9)
    near(dw, w_want, w_size, 203, torch.float32, "dw")
    near(db, b_want, b_size, 203, torch.float32, "db")


def side_stream():
    """Work on torch's current stream, behind what was queued there before."""
    be = backend()
    args = _together_inputs(4)
    want = [t.clone() for t in _together(be, *args, 5)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        big = torch.randn((4096, 4096), device=DEV)
        for _ in range(20):  # keeps the stream busy, so a call elsewhere would be early
            big = big @ big / 64
        late = [t.clone() for t in args]
        got = _together(be, *late, 5)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # two streams at once
    s2 = torch.cuda.Stream()
    other = _together_inputs(9)
    want2 = [t.clone() for t in _together(be, *other, 6)]
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s):
            got = _together(be, *args, 5)
        with torch.cuda.stream(s2):
            got2 = _together(be, *other, 6)
    torch.cuda.synchronize()
    for a, b in zip(got + got2, want + want2):
        assert torch.equal(a, b)


def captured():
    """Two graphs of the operators, replayed in turn with eager work between, against the
    eager results each time."""
    be = backend()
    graphs = []
    for seed in (11, 12):
        held = _together_inputs(seed)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _together(be, *held, seed)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _together(be, *held, seed)
        graphs.append((seed, held, graph, out))
    for turn in range(4):
        for seed, held, graph, out in graphs:
            fresh = _together_inputs(100 * turn + seed)
            for to, new in zip(held, fresh):
                to.copy_(new)
            graph.replay()
        for seed, held, graph, out in graphs:
            want = _together(be, *held, seed)
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def captured_large():
    """The forms for large tiles, many rows and long rows of scores, replayed from one graph."""
    be = backend()
    rng = np.random.default_rng(8)
    dt = torch.bfloat16
    leaf = torch.from_numpy(leaves_of(rng, 1300, 2, 3, "lost")).to(DEV).int()
    x, dy = matrix(rng, 1300, 264, dt), matrix(rng, 1300, 200, dt)
    w = matrix(rng, 6 * 200, 264, dt).view(6, 200, 264)
    long_leaf = torch.from_numpy(leaves_of(rng, 30000, 1, 9, "skew")).to(DEV).int()
    scores = matrix(rng, 5, 20000, torch.float32)

    def run():
        g = be.leaf_groups(leaf, 3)
        dw, db = be.leaf_product_dw(dy, x, g)
        return (be.leaf_product(x, w, g), be.leaf_product_dx(dy, w, g), dw, db,
                *be.leaf_groups(long_leaf, 9), be.adjust_scores(scores, "transformed"))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for turn in range(3):
        x.copy_(matrix(rng, 1300, 264, dt))
        scores.copy_(matrix(rng, 5, 20000, torch.float32))
        leaf.copy_(torch.from_numpy(leaves_of(rng, 1300, 2, 3, "lost")).to(DEV).int())
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def learner():
    """With the learner: bagged gradients grow a tree, its layout groups the rows, the normal
    equations of linear leaves come from one product, and the fitted leaves lower the squared
    error that the tree's own leaves leave."""
    from lightgbm_rs_amd.synth import config1_like
    be = HipBackend(0)
    try:
        n = 20000
        bins, meta, ub, _ = config1_like(n, seed=3)
        rng = np.random.default_rng(1)
        X = torch.from_numpy(np.concatenate([bins[:6].T.astype(np.float32) / 32, np.ones((n, 1), np.float32)], 1)).to(DEV)
        target = X @ torch.randn(7, generator=torch.Generator().manual_seed(1)).to(DEV)
        target = target + 0.1 * torch.from_numpy(rng.standard_normal(n).astype(np.float32)).to(DEV)
        gh = torch.stack([-target, torch.ones_like(target)], 1)
        bagged = be.dropout(gh, 0.2, 42, by="row")
        keep, share = oracle.kept(n, 0.2, 42)
        assert torch.equal(bagged[:, 1] > 0, torch.from_numpy(keep).to(DEV))
        g, h = (v.cpu().numpy() for v in bagged.t())
        be.upload_resident_bins(bins, meta, ub)
        be.upload_resident_grad_hess(g, h)
        tree, layout = be.grow_tree_on_device_with_cfg(GainConfig.make(min_data_in_leaf=20), 15, -1)
        groups = LeafGroups.from_layout(layout)
        L = groups.begin.shape[1]
        assert L == tree["num_leaves"] and int(groups.count.sum()) == n
        # rows [h x | -g] against x: a leaf's X^T H X and X^T (-g)
        dy = torch.cat([X * bagged[:, 1:], -bagged[:, :1]], 1)
        m, _ = be.leaf_product_dw(dy, X, groups, bias=False)
        A, rhs = m[:, :7].double().cpu(), m[:, 7].double().cpu()
        w = torch.linalg.solve(A + 1e-3 * torch.eye(7), rhs[:, :, None])[:, :, 0]
        pred = be.leaf_product(X, w.float()[:, None].contiguous().to(DEV), groups)[:, 0]
        own = be.leaf_product(torch.ones_like(X[:, :1]), torch.from_numpy(tree["leaf_value"][:L]).float().view(L, 1, 1).to(DEV), groups)[:, 0]
        order = torch.from_numpy(layout["indices"].astype(np.int64))
        for l in range(L):
            b, c = int(layout["leaf_begin"][l]), int(layout["leaf_count"][l])
            rows = order[b:b + c].to(DEV)
            assert bool((own[rows] == np.float32(tree["leaf_value"][l])).all())
        assert float((pred - target).square().mean()) < float((own - target).square().mean())
    finally:
        be.close()


def forest():
    """The leaves that prediction gives: a forest's leaf indices grouped, its leaf values as
    maps of one input, against the prediction's raw scores."""
    import os
    be = backend()
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "predict", "multiclass_model.txt")
    model = Model.from_file(path)
    rng = np.random.default_rng(4)
    X = rng.standard_normal((501, model.max_feature_idx + 1)).astype(np.float32)
    leaf = be.predict(model, X, "leaf")
    raw = be.predict(model, X, "raw")
    K = model.num_tree_per_iteration
    values = [[float(v) for v in line.split("=")[1].split()]
              for line in open(path) if line.startswith("leaf_value=")]
    T, L = leaf.shape[1], max(map(len, values))
    assert T == len(values)
    w = np.zeros((T, L, K, 1))
    for t, v in enumerate(values):
        w[t, :len(v), t % K, 0] = v
    g = be.leaf_groups(torch.from_numpy(leaf).to(DEV), L)
    wt = torch.from_numpy(w).float().to(DEV).view(T * L, K, 1)
    y = be.leaf_product(torch.ones((501, 1), device=DEV), wt, g)
    size = oracle.product(np.ones((501, 1)), np.abs(w).reshape(T * L, K, 1), None, leaf, L)[0]
    # the leaf values are rounded to float32 once more
    near(y, raw, size * 2, T * K, torch.float32, "raw")
    p = be.adjust_scores(torch.from_numpy(raw).to(DEV), kind="transformed")
    want = be.predict(model, X, "transformed")
    assert np.allclose(p.cpu().numpy(), want, rtol=64 * 2.0 ** -53, atol=0)


def threads():
    """A context for each of two threads, on streams of their own."""
    import threading
    results, errors = {}, []

    def work(i):
        try:
            be = HipBackend(0)
            args = _together_inputs(20 + i)
            with torch.cuda.stream(torch.cuda.Stream()):
                torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
                for _ in range(10):
                    out = _together(be, *args, i)
                torch.cuda.current_stream().synchronize()
            results[i] = [t.clone() for t in out]
            torch.cuda.synchronize()
            be.close()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    both = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in both:
        t.start()
    for t in both:
        t.join()
    assert not errors, errors
    for i in (0, 1):
        for a, b in zip(results[i], _together(backend(), *_together_inputs(20 + i), i)):
            assert torch.equal(a, b)


def own_stream():
    """The C entry without a stream: on the context's own, done when it returns."""
    be = backend()
    x = torch.arange(1000, device=DEV, dtype=torch.float32).view(10, 100)
    out = torch.zeros_like(x)
    want = be.dropout(x, 0.5, 3)
    torch.cuda.synchronize()
    assert be.lib.lgbm_hip_dropout(be.ctx, C.c_void_p(x.data_ptr()), C.c_int64(100), C.c_int64(10),
                                   C.c_int64(100), C.c_int32(0), C.c_double(0.5), C.c_uint64(3),
                                   C.c_uint64(0), C.c_int32(0), C.c_void_p(out.data_ptr()),
                                   C.c_int64(100), None) == 0
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        assert torch.equal(out.cpu(), want.cpu())


def refused():
    """What the device entries refuse, with a context."""
    be = backend()
    x = torch.zeros((4, 5), device=DEV)
    for call in (lambda: be.dropout(x, 1.5, 0), lambda: be.dropout(x, float("nan"), 0),
                 lambda: be.leaf_groups(torch.zeros((4, 1), dtype=torch.int32, device=DEV), 5000),
                 lambda: be.leaf_groups(torch.zeros((4, 1), dtype=torch.int32, device=DEV), 0),
                 lambda: be.adjust_scores(x, ids=torch.zeros(0, dtype=torch.int32, device=DEV),
                                          offsets=torch.zeros(5, dtype=torch.int64, device=DEV),
                                          repetition=0.0),
                 lambda: be.adjust_scores(x, mask=torch.zeros((3, 1), dtype=torch.int32, device=DEV)),
                 lambda: be.dropout(x[1:], 0.5, 0, out=x[:3])):
        try:
            call()
        except HipError:
            continue
        raise AssertionError("not refused")


def whole_dw(rows, inputs, outputs, trees, leaves, dtype, shape):
    """Gradients of the maps of whole numbers: every sum is exact, whatever its order, so the
    result has to be the oracle's bit for bit."""
    assert 25 * rows <= 2 ** 24
    rng = np.random.default_rng(rows)
    leaf = leaves_of(rng, rows, trees, leaves, shape)
    g = LeafGroups(*(torch.from_numpy(v).to(DEV) for v in oracle.groups(leaf, leaves)))
    x, dy = oracle.whole_numbers(rng, rows, inputs), oracle.whole_numbers(rng, rows, outputs)
    up = lambda v: torch.from_numpy(v).to(TYPES[dtype]).to(DEV)
    dw, db = backend().leaf_product_dw(up(dy), up(x), g)
    w_want, _, b_want, _ = oracle.product_dw(dy, x, leaf, leaves)
    assert w_want.any() and np.array_equal(wide(dw), w_want) and np.array_equal(wide(db), b_want)


def long_sums(rows, inputs, outputs, dtype):
    """A leaf of many rows, all alike: x = dy = 1 + 2^-5 makes products of 1 + 2^-4 + 2^-10.
    Of at most 8192 rows every partial sum is a whole number of 2^-10 and below 2^14, so it is
    exact in float32's 24 bits, and so are their sums in float64: the result is the exact one,
    rounded once.  (One chain of float32 adds drops the low bits of every term.)"""
    dt = TYPES[dtype]
    g = LeafGroups(torch.arange(rows, dtype=torch.int32, device=DEV)[None],
                   torch.zeros((1, 1), dtype=torch.int32, device=DEV),
                   torch.full((1, 1), rows, dtype=torch.int32, device=DEV))
    x = torch.full((rows, inputs), 1 + 2.0 ** -5, dtype=dt, device=DEV)
    dy = torch.full((rows, outputs), 1 + 2.0 ** -5, dtype=dt, device=DEV)
    dw, db = backend().leaf_product_dw(dy, x, g)
    w_want, b_want = np.float32(rows * (1 + 2.0 ** -5) ** 2), np.float32(rows * (1 + 2.0 ** -5))
    assert bool((dw == float(w_want)).all()), (w_want, dw.min().item(), dw.max().item())
    assert bool((db == float(b_want)).all()), (b_want, db.min().item(), db.max().item())


def odd_tables_large_tiles():
    """As odd_tables, with rows enough for the large tiles of y and dx."""
    odd_tables(400, 200, 192, "bf16")


def captured_tiles():
    """y and dx by large tiles replayed from a graph, over tables that change."""
    be = backend()
    rng = np.random.default_rng(12)
    dt = torch.float16
    x, dy = matrix(rng, 9000, 264, dt), matrix(rng, 9000, 520, dt)
    w = matrix(rng, 6 * 520, 264, dt).view(6, 520, 264)
    leaf = torch.from_numpy(leaves_of(rng, 9000, 2, 3, "even")).to(DEV).int()

    def run():
        g = be.leaf_groups(leaf, 3)
        return be.leaf_product(x, w, g), be.leaf_product_dx(dy, w, g), *be.leaf_product_dw(dy, x, g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for shape in ("lost", "one", "skew"):
        x.copy_(matrix(rng, 9000, 264, dt))
        leaf.copy_(torch.from_numpy(leaves_of(rng, 9000, 2, 3, shape)).to(DEV).int())
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def tree_runs(rows, inputs, width, trees, dtype, strided=False):
    """Planes of more than 4 GiB: trees in runs, the last one shorter.  A row has one input
    that is not 0, and all are whole numbers, so every sum is exact in the type."""
    be, dt, leaves = backend(), TYPES[dtype], 5
    assert trees * rows * width * 4 > 2 ** 32 and trees * 30 <= 2 / torch.finfo(dt).eps
    gen = torch.Generator(device=DEV).manual_seed(rows)
    whole = lambda *shape: torch.randint(-5, 6, shape, generator=gen, device=DEV).to(dt)
    leaf = torch.randint(0, leaves, (rows, trees), generator=gen, device=DEV).int()
    leaf[torch.rand((rows, trees), generator=gen, device=DEV) < 0.1] = -1
    g = be.leaf_groups(leaf, leaves)
    w, b, value = whole(trees * leaves, inputs, width), whole(trees * leaves, width), whole(rows, 1)
    at = torch.randint(0, inputs, (rows, 1), generator=gen, device=DEV)
    x = torch.zeros((rows, inputs), dtype=dt, device=DEV).scatter_(1, at, value)
    room = torch.full((rows, width + 3), 9, dtype=dt, device=DEV) if strided else None
    out = None if room is None else room[:, 1:1 + width]
    y = be.leaf_product(x, w.transpose(1, 2).contiguous(), g, bias=b, out=out)
    want, sums = torch.zeros_like(y), torch.zeros_like(y)
    none = torch.zeros((), dtype=dt, device=DEV)
    for t in range(trees):
        l, there = (leaf[:, t].clamp(min=0) + t * leaves).long(), (leaf[:, t] >= 0)[:, None]
        want += torch.where(there, value * w[l, at[:, 0]], none)
        sums += torch.where(there, value * w[l, at[:, 0]] + b[l], none)
    assert bool(want.any()) and torch.equal(y, sums)
    if strided:
        assert bool((room[:, 0] == 9).all()) and bool((room[:, 1 + width:] == 9).all())
    del y, sums, room, out
    assert torch.equal(be.leaf_product_dx(x, w, g), want)


def versions():
    """Tensors that a call writes: a graph of torch's that saved one refuses its backward pass,
    and one of inference mode is written all the same."""
    be = backend()
    z = lambda *shape: torch.ones(shape, device=DEV)
    g = be.leaf_groups(torch.zeros((6, 1), dtype=torch.int32, device=DEV), 2)
    x, w, dy = z(6, 5), z(2, 3, 5), z(6, 3)
    line, mat, scores = z(40), z(6, 5), z(6, 3)
    for out, call in ((z(6, 3), lambda o: be.leaf_product(x, w, g, out=o)),
                      (z(6, 5), lambda o: be.leaf_product_dx(dy, w, g, out=o)),
                      (z(2, 3, 5), lambda o: be.leaf_product_dw(dy, x, g, out=o)),
                      (z(2, 3), lambda o: be.leaf_product_dw(dy, x, g, bias_out=o)),
                      (z(6, 5), lambda o: be.dropout(x, 0.5, 1, out=o)), (mat, lambda o: be.dropout(mat, 0.5, 1, out=o)),
                      (line, lambda o: be.dropout(line, 0.5, 1, out=o)), (z(40), lambda o: be.dropout(line, 0.5, 1, out=o)),
                      (z(6, 3), lambda o: be.adjust_scores(dy, "transformed", out=o)),
                      (scores, lambda o: be.adjust_scores(scores, "transformed", out=o))):
        leaf = torch.ones_like(out).requires_grad_()
        y = (leaf * out).sum()
        call(out)
        try:
            y.backward()
        except RuntimeError as e:
            assert "inplace" in str(e)
            continue
        raise AssertionError("a saved tensor was written unseen")
    assert not x._version and not dy._version and not w._version
    with torch.inference_mode():
        v = torch.ones((6, 5), device=DEV)
        assert be.dropout(v, 1.0, 1, out=v) is v and not bool(v.any())


def earlier_error():
    """An error that an earlier call of the program left in the HIP runtime is not this call's."""
    be = backend()
    with open("/proc/self/maps") as maps:
        path = next(line.split()[-1] for line in maps if "libamdhip64" in line)
    hip = C.CDLL(path)
    x = torch.ones((4, 5), device=DEV)
    out = torch.empty_like(x)
    want = be.dropout(x, 0.5, 1)
    torch.cuda.synchronize()
    assert hip.hipSetDevice(C.c_int(99)) != 0  # no such device
    try:
        be.dropout(x, 0.5, 1, out=out)
    finally:
        hip.hipGetLastError()
    assert torch.equal(out, want)


def scores_nan(classes, dtype):
    """A NaN that is not masked: the row's probabilities are NaN, also where they would vanish
    beside the row's largest, but for those of classes at -inf."""
    dt, rows = TYPES[dtype], 5
    rng = np.random.default_rng(classes)
    x = torch.from_numpy(rng.standard_normal((rows, classes))).to(dt)
    x[:, 1] = -1000  # e^-1000 is 0 in every type
    x[:, 0], x[:, 2] = -float("inf"), float("inf")
    x[:4, 2] = 3
    at = [classes - 1, 3, classes // 2, 0, 4]
    for n in (0, 1, 2, 4):
        x[n, at[n]] = float("nan")
    allowed = rng.random((rows, classes)) < 0.7
    allowed[:, 1:5] = True
    for n in (0, 1, 2, 4):
        allowed[n, at[n]] = True
    allowed[0, 3] = False
    bits = np.zeros((rows, (classes + 31) // 32 * 32), bool)
    bits[:, :classes] = allowed
    mask = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32)).to(DEV)
    p = wide(backend().adjust_scores(x.to(DEV), "transformed", mask=mask))
    none = ~allowed | np.isneginf(wide(x))
    for n in (0, 1, 2, 4):
        assert (p[n, none[n]] == 0).all() and np.isnan(p[n, ~none[n]]).all(), n
    assert (p[3, none[3]] == 0).all() and p[3, 1] == 0 and abs(p[3].sum() - 1) < 0.05


def side_by_side():
    """Inputs and outputs as columns of one table."""
    be = backend()
    rng = np.random.default_rng(31)
    table = matrix(rng, 300, 40, torch.float32)
    x, y, d, p = table[:, :20], table[:, 20:26], table[:, 26:32], table[:, 34:40]
    kept = table[:, 32:34].clone()
    leaf = torch.from_numpy(leaves_of(rng, 300, 2, 5, "lost")).to(DEV)
    g = be.leaf_groups(leaf, 5)
    w = matrix(rng, 60, 20, torch.float32).view(10, 6, 20)
    x0 = x.clone()
    want = be.leaf_product(x0, w, g)
    assert be.leaf_product(x, w, g, out=y) is y and torch.equal(y, want)
    be.dropout(y, 0.3, 7, out=d)
    assert torch.equal(d, be.dropout(want, 0.3, 7))
    be.adjust_scores(d, "transformed", out=p)
    assert torch.equal(p, be.adjust_scores(d.clone(), "transformed"))
    dx = be.leaf_product_dx(p.clone(), w, g)
    be.leaf_product_dx(p, w, g, out=x)
    assert torch.equal(x, dx) and torch.equal(y, want) and torch.equal(table[:, 32:34], kept)


def odd_counts():
    """A table of a million leaves that all claim every row: together they would have more than
    2^32 parts.  The first leaf's gradient is right, the others' are some value."""
    rows, leaves = 2 ** 26, 2 ** 20 + 300
    one = torch.ones((rows, 1), device=DEV)
    g = LeafGroups(torch.arange(rows, dtype=torch.int32, device=DEV)[None],
                   torch.zeros((1, leaves), dtype=torch.int32, device=DEV),
                   torch.full((1, leaves), rows, dtype=torch.int32, device=DEV))
    dw, db = backend().leaf_product_dw(one, one, g)
    assert dw[0].item() == rows and db[0].item() == rows and bool(dw.isfinite().all())


def short_sums(inputs, outputs):
    """float32 sums go in stretches of 32 rows that start at zero: with c = 1 + 2^-15, 32 c is
    a whole number of 2^-10, exact beside sums below 2^14, and within a stretch sums are whole
    numbers of 2^-15 below 2^6.  So dW and db of x = 1 and dy = c are exact, where a chain of
    single rows or fours drops the 2^-13 of 4 c beside sums above 2^11."""
    rows = 3 * 8192
    g = LeafGroups(torch.arange(rows, dtype=torch.int32, device=DEV)[None],
                   torch.zeros((1, 1), dtype=torch.int32, device=DEV),
                   torch.full((1, 1), rows, dtype=torch.int32, device=DEV))
    x = torch.ones((rows, inputs), device=DEV)
    dy = torch.full((rows, outputs), 1 + 2.0 ** -15, device=DEV)
    dw, db = backend().leaf_product_dw(dy, x, g)
    want = rows * (1 + 2.0 ** -15)
    assert bool((dw == want).all()), (want, dw.min().item(), dw.max().item())
    assert bool((db == want).all()), (want, db.min().item(), db.max().item())
