"""Checks of the leaves' layers, their gradients and of clipping against leaf_layer_oracle.py,
run by leaf_layer_worker.py on the GPU.  The oracle's bounds hold for float32 arithmetic; a
result rounded to a type is off by half a step (u = finfo(type).eps / 2 relative, and tiny *
eps where it is subnormal) more."""
import math

import numpy as np
import torch

from lightgbm_rs_amd import HipError, LeafGroups
from tests import leaf_layer_oracle as oracle
from tests import leaf_ops_oracle
from tests.leaf_ops_checks import DEV, TYPES, backend, close, leaves_of, matrix, wide  # noqa: F401

U = oracle.U


def near(got, want, bound, what):
    info = torch.finfo(got.dtype)
    tol = info.eps / 2 * (np.abs(want) + bound) + bound + info.tiny * info.eps
    got = wide(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4],
                           want[bad][:4], tol[bad][:4])


class Case:
    """One layer: inputs with NaN behind the rows' ends, and the oracle's answer."""

    def __init__(self, rows, inputs, outputs, trees=1, leaves=1, dtype="f32", shape="skew", pad=0,
                 act="silu", gated=False, bias=True, residual=True, seed=0):
        rng = np.random.default_rng(seed)
        self.leaf = leaves_of(rng, rows, trees, leaves, shape)
        self.groups = LeafGroups(*(torch.from_numpy(v).to(DEV) for v in leaf_ops_oracle.groups(self.leaf, leaves)))
        dt, lead = TYPES[dtype], 3 if pad % 2 else 0
        R = 2 * outputs if gated else outputs
        self.dtype, self.rows, self.outputs, self.trees, self.leaves = dt, rows, outputs, trees, leaves
        self.form = dict(activation=act, gated=gated)
        self.x = matrix(rng, rows, inputs, dt, pad, lead)
        self.w = (matrix(rng, trees * leaves * R, inputs, dt, 0, lead) * inputs ** -0.5).view(trees * leaves, R, inputs)
        self.b = matrix(rng, trees * leaves, R, dt, 0, lead) if bias else None
        self.r = matrix(rng, rows, outputs, dt, pad, lead) if residual else None
        self.dy = matrix(rng, rows, outputs, dt, pad, lead)
        opt = lambda t: None if t is None else wide(t)
        self.y, self.y_off, self.z, self.z_size = oracle.layer(
            wide(self.x), wide(self.w), opt(self.b), self.leaf, leaves, act, gated, opt(self.r))
        self.z_off = 2 * (inputs + 3) * U * self.z_size

    def layer(self, **more):
        return backend().leaf_layer(self.x, self.w, self.groups, bias=self.b, residual=self.r, **self.form, **more)

    def grad(self, z, **more):
        return backend().leaf_layer_grad(self.dy, z, self.x, self.w, self.groups, **self.form, **more)

    def want_grads(self, z):
        info = torch.finfo(self.dtype)
        return oracle.grads(wide(self.dy), None if z is None else wide(z), wide(self.x), wide(self.w), self.leaf,
                            self.leaves, self.form["activation"], self.form["gated"], info.eps, info.tiny)


def layer(**args):
    c = Case(**args)
    y = c.layer()
    near(y, c.y, c.y_off, "y")
    assert torch.equal(y, c.layer())
    kept, z = c.layer(keep=True)
    assert torch.equal(y, kept)
    assert z.dtype == torch.float32
    near(z, c.z, c.z_off, "z")
    kept, narrow = c.layer(keep=c.dtype)
    assert torch.equal(y, kept) and torch.equal(narrow, z.to(c.dtype))
    # into the caller's strided output, whose gaps stay as they were
    room = torch.full((c.rows, c.outputs + 5), 7.0, dtype=c.dtype, device=DEV)
    out = room[:, 2:2 + c.outputs]
    assert c.layer(out=out) is out
    assert torch.equal(out, y) and bool((room[:, :2] == 7).all()) and bool((room[:, 2 + c.outputs:] == 7).all())
    if c.r is not None:  # onto the residual itself
        room[:, 2:2 + c.outputs] = c.r
        c.r = out
        assert c.layer(out=out) is out and torch.equal(out, y)


def grads(kept=None, **args):
    c = Case(**args)
    _, z = c.layer(keep=True if kept is None else c.dtype)
    linear = c.form == dict(activation="none", gated=False)
    if linear:
        z = None
    want = c.want_grads(z)
    dx, dw, db = c.grad(z)
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        assert got.dtype == c.dtype
        near(got, *want[name], name)
    # in float32, without the rounding; the same bits every time; each alone
    dw32 = torch.full(dw.shape, 3.0, device=DEV)
    db32 = torch.full(db.shape, 3.0, device=DEV)
    got = c.grad(z, inputs=False, weight_out=dw32, bias_out=db32)
    assert got[0] is None and got[1] is dw32 and got[2] is db32
    near(dw32, *want["dw"], "dw in float32")
    near(db32, *want["db"], "db in float32")
    assert torch.equal(dw32.to(c.dtype), dw) and torch.equal(db32.to(c.dtype), db)
    alone, none, also = c.grad(z, maps=False)
    assert torch.equal(alone, dx) and none is None and also is None
    _, dw2, none = c.grad(z, bias=False)
    assert torch.equal(dw2, dw) and none is None


def differences(act, gated, trees):
    """The gradients against central differences of the oracle's loss sum(dy * y)."""
    c = Case(rows=37, inputs=9, outputs=6, trees=trees, leaves=3, act=act, gated=gated, shape="lost", seed=5)
    _, z = c.layer(keep=True)
    dx, dw, db = c.grad(z)
    rng = np.random.default_rng(1)
    x, w, b, r, dy = (wide(t) for t in (c.x, c.w, c.b, c.r, c.dy))

    def loss(x, w, b):
        return (oracle.layer(x, w, b, c.leaf, c.leaves, act, gated, r)[0] * dy).sum()

    h = 1e-5
    for got, at in ((dx, 0), (dw, 1), (db, 2)):
        args = [x, w, b]
        way = rng.standard_normal(args[at].shape)
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[at] = args[at] + sign * h * way
            ends.append(loss(*moved))
        slope = (ends[0] - ends[1]) / (2 * h)
        # each of the gradient's elements is a float32 sum of at most 37 or 2 x 6 x trees terms
        # of a dz that is off by about 20 U; the differences' error is of h^2 and of 2^-53 / h
        size = (np.abs(wide(got)) * np.abs(way)).sum()
        assert abs((wide(got) * way).sum() - slope) <= 300 * U * size + 1e-7 * max(1.0, size), (at, slope)


def extreme():
    """Pre-activations that their type cannot hold, NaN and infinite inputs, rows in no leaf."""
    be = backend()
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        leaf = torch.tensor([0, 0, 0, -1, 0, 0], dtype=torch.int32, device=DEV)
        g = be.leaf_groups(leaf, 1)
        big = 60000.0 if dt == torch.float16 else 1e30
        x = torch.tensor([[big], [-big], [float("nan")], [float("nan")], [0.0], [1.0]], dtype=dt, device=DEV)
        w = torch.tensor([[[2.0], [2.0]]], dtype=dt, device=DEV)
        dy = torch.ones((6, 1), dtype=dt, device=DEV)
        for act in ("silu", "gelu", "gelu_tanh", "relu", "sigmoid"):
            y, z = be.leaf_layer(x, w, g, activation=act, gated=True, keep=dt)
            assert y[2].isnan().all() and bool((y[3] == 0).all()) and bool((z[0, 3] == 0).all()), act
            assert bool((y[1] == 0).all()) and bool((y[4] == 0).all()) and y[0].isnan().sum() == 0, act
            dx, dw, db = be.leaf_layer_grad(dy, z, x, w, g, activation=act, gated=True)
            assert bool((dx[3] == 0).all()) and dx[2].isnan().all() and not dx[4:].isnan().any(), (act, dx)
            # at either end the slope is that of the limit, not infinity times zero
            if act != "sigmoid":
                assert not dx[0].isnan().any(), (act, dx)
            single, zs = be.leaf_layer(x, w[:, :1].contiguous(), g, activation=act, keep=dt)
            dx, _, _ = be.leaf_layer_grad(dy, zs, x, w[:, :1].contiguous(), g, activation=act)
            top = 0.0 if act == "sigmoid" else 2.0
            assert dx[0].item() == top and dx[1].item() == 0.0 and dx[2].isnan().all() and dx[3].item() == 0, (act, dx)
        # dy of a row in no leaf is not looked at
        dy[3] = float("nan")
        dx, dw, db = be.leaf_layer_grad(dy, be.leaf_layer(x, w, g, activation="relu", gated=True, keep=True)[1],
                                        x.nan_to_num(0, 0, 0), w, g, activation="relu", gated=True)
        assert not dx[3].isnan().any()


def kernels_of_layers():
    """Empty tables: no rows; all rows in no leaf; gradients of leaves without rows are zeros."""
    be = backend()
    for dt in (torch.float32, torch.bfloat16):
        w = torch.ones((3, 4, 5), dtype=dt, device=DEV)
        none = torch.empty((0, 5), dtype=dt, device=DEV)
        g = be.leaf_groups(torch.empty((0, 1), dtype=torch.int32, device=DEV), 3)
        y, z = be.leaf_layer(none, w, g, activation="silu", keep=True)
        assert y.shape == (0, 4) and z.shape == (1, 0, 4)
        dx, dw, db = be.leaf_layer_grad(y, z, none, w, g, activation="silu")
        assert dx.shape == (0, 5) and bool((dw == 0).all()) and bool((db == 0).all())
        x = torch.ones((70, 5), dtype=dt, device=DEV)
        r = torch.full((70, 4), 2.0, dtype=dt, device=DEV)
        g = be.leaf_groups(torch.full((70, 1), -1, dtype=torch.int32, device=DEV), 3)
        y, z = be.leaf_layer(x, w, g, activation="sigmoid", residual=r, keep=True)
        assert torch.equal(y, r) and bool((z == 0).all())
        dx, dw, db = be.leaf_layer_grad(r, z, x, w, g, activation="sigmoid")
        assert bool((dx == 0).all()) and bool((dw == 0).all()) and bool((db == 0).all())


def _list(sizes, dtypes, seed, flat, scale=1.0):
    rng = np.random.default_rng(seed)
    if flat:
        dt = TYPES[dtypes[0]]
        all_of = torch.from_numpy(rng.standard_normal(sum(sizes) + 1) * scale).to(dt).to(DEV)
        return list(all_of[1:].split(list(sizes)))
    return [torch.from_numpy(rng.standard_normal(n) * scale).to(TYPES[dtypes[i % len(dtypes)]]).to(DEV)
            for i, n in enumerate(sizes)]


def clip(sizes, dtypes, seed=0, flat=False, factor=0.5, scale=1.0):
    be = backend()
    ts = _list(sizes, dtypes, seed, flat, scale)
    exact = [wide(t) for t in ts]
    norm = oracle.clip(exact, 0.0)[0]
    limit = factor * norm if norm > 0 else 1.0
    norm, by, want = oracle.clip(exact, limit)
    # float64 sums: a float32's rounding, and 1e-12 for the sums
    tol = norm * (U + 1e-12) + 1e-45
    got = be.grad_norm(ts)
    assert got.dtype == torch.float32 and got.shape == () and abs(float(got) - norm) <= tol, (float(got), norm)
    out = [torch.full_like(t, 5.0) for t in ts]
    before = [t.clone() for t in ts]
    assert torch.equal(be.clip_grads(ts, limit, out=out), got)
    for t, b, o, w in zip(ts, before, out, want):
        assert torch.equal(t, b)
        # the scale and the product are rounded to float32, then to the type
        near(o, w, 2 * U * np.abs(w), "clipped")
        if by == 1.0:
            assert torch.equal(o, b)
    versions = [t._version for t in ts]
    assert torch.equal(be.clip_grads(ts, limit), got)
    assert all(t._version > v for t, v in zip(ts, versions))
    for t, o in zip(ts, out):
        assert torch.equal(t, o)


def clip_special():
    be = backend()
    assert float(be.grad_norm([])) == 0.0 and float(be.clip_grads([], 1.0)) == 0.0
    empty = torch.empty((0, 4), device=DEV)
    assert float(be.clip_grads([empty, empty], 1.0)) == 0.0
    # squares that float32 does not hold
    big, small = torch.full((3,), 1e30, device=DEV), torch.full((4,), 1e-30, device=DEV)
    assert abs(float(be.grad_norm([big])) / (math.sqrt(3) * 1e30) - 1) < 1e-6
    assert abs(float(be.grad_norm([small])) / 2e-30 - 1) < 1e-6
    assert float(be.grad_norm([torch.zeros(9, device=DEV)])) == 0.0
    # a limit of nothing; zeros stay zeros
    t = torch.ones(100, device=DEV)
    assert float(be.clip_grads([t], 0.0)) == 10.0 and bool((t == 0).all())
    assert float(be.clip_grads([t], 0.0)) == 0.0 and bool((t == 0).all())
    # infinite and NaN norms
    t = torch.tensor([1.0, float("inf"), -2.0], device=DEV)
    assert float(be.clip_grads([t], 1.0)) == math.inf
    assert t[0] == 0 and t[1].isnan() and t[2] == 0
    t, other = torch.tensor([1.0, float("nan")], device=DEV), torch.ones(5, dtype=torch.bfloat16, device=DEV)
    assert be.clip_grads([t, other], 1.0).isnan() and t.isnan().all() and other.isnan().all()
    t = torch.tensor([3.0, float("inf")], device=DEV)
    be.clip_grads([t], math.inf)
    assert t.tolist() == [3.0, math.inf]
    # the same tensor twice counts twice; dense tensors in any order of dimensions
    t = torch.randn((6, 5, 4), device=DEV).permute(2, 0, 1)
    once, twice = be.grad_norm([t]), be.grad_norm([t, t])
    assert abs(float(twice) / float(once) - math.sqrt(2)) < 1e-6
    want = t * (0.5 / float(once))
    be.clip_grads([t], 0.5)
    assert torch.allclose(t, want, rtol=1e-6)


def refused():
    be, f32 = backend(), torch.float32
    x = torch.ones((8, 4), device=DEV)
    w = torch.ones((2, 6, 4), device=DEV)
    g = be.leaf_groups(torch.zeros((8, 1), dtype=torch.int32, device=DEV), 2)
    dy, z = torch.ones((8, 6), device=DEV), torch.ones((1, 8, 6), device=DEV)

    def bad(call, text, error=ValueError):
        try:
            call()
        except error as e:
            assert text in str(e), (text, str(e))
            return
        raise AssertionError(f"not refused: {text}")

    bad(lambda: be.leaf_layer(x, w, g, activation="elu"), "activation")
    bad(lambda: be.leaf_layer(x.double(), w.double(), g), "float64")
    bad(lambda: be.leaf_layer(x, w.half(), g), "differ in type")
    bad(lambda: be.leaf_layer(x, w, g, bias=torch.ones((2, 5), device=DEV)), "shape")
    bad(lambda: be.leaf_layer(x, w, g, residual=torch.ones((8, 5), device=DEV)), "shape")
    bad(lambda: be.leaf_layer(x, w, g, gated=True, residual=dy), "shape")
    bad(lambda: be.leaf_layer(x, w[:, :5].contiguous(), g, gated=True), "even")
    bad(lambda: be.leaf_layer(x, w[:1], g), "leaves")
    bad(lambda: be.leaf_layer(x.cpu(), w, g), "cuda:0 is needed")
    bad(lambda: be.leaf_layer(x.clone().requires_grad_(), w, g), "requires gradients")
    bad(lambda: be.leaf_layer(x, w, g, out=torch.ones((8, 12), device=DEV)[:, ::2]), "strided")
    square = torch.ones((2, 4, 4), device=DEV)
    bad(lambda: be.leaf_layer(x, square, g, out=x), "overlaps", HipError)
    wide_room = torch.ones((9, 6), device=DEV)
    bad(lambda: be.leaf_layer(x, w, g, residual=wide_room[1:], out=wide_room[:8]), "in place", HipError)
    bad(lambda: be.leaf_layer_grad(dy, None, x, w, g, activation="silu"), "z is needed")
    bad(lambda: be.leaf_layer(x, w, g, keep=torch.float16), "keep")
    bad(lambda: be.leaf_layer_grad(dy, z.half(), x, w, g, activation="silu"), "float32")
    bad(lambda: be.leaf_layer_grad(dy, z[:, :7], x, w, g, activation="silu"), "shape")
    bad(lambda: be.leaf_layer_grad(dy[:, :5], z, x, w, g, activation="silu"), "shape")
    bad(lambda: be.leaf_layer_grad(dy, z, x, w, g, activation="silu", inputs=False, maps=False), "neither")
    bad(lambda: be.leaf_layer_grad(dy, z, x, w, g, activation="silu", inputs=False, out=x), "not asked")
    bad(lambda: be.leaf_layer_grad(dy, z, x, w, g, activation="silu", weight_out=w.half()), "float32")
    bad(lambda: be.leaf_layer_grad(dy, z, x, w, g, activation="silu", out=x), "overlaps", HipError)
    bad(lambda: be.clip_grads([x, x], 1.0), "overlaps", HipError)
    bad(lambda: be.clip_grads([x[:4], x[3:]], 1.0), "overlaps", HipError)
    bad(lambda: be.clip_grads([x], 1.0, out=[x[:, :3]]), "differ")
    bad(lambda: be.clip_grads([x, w], 1.0, out=[w, x]), "differ")
    bad(lambda: be.clip_grads([x], 1.0, out=[]), "number")
    bad(lambda: be.clip_grads([x], -1.0), "negative", HipError)
    bad(lambda: be.clip_grads([x], float("nan")), "NaN", HipError)
    bad(lambda: be.grad_norm([x[:, :3]]), "gaps")
    bad(lambda: be.grad_norm([x.double()]), "float64")
    bad(lambda: be.grad_norm([x.cpu()]), "cuda:0")
    bad(lambda: be.grad_norm([x.clone().requires_grad_()]), "gradients")
    assert f32 == x.dtype


def block(dtype, act="silu", trees=1):
    """A gated hidden layer, a second layer onto the rows themselves, both gradients and a clip:
    eagerly, on another stream, and captured and replayed over new inputs."""
    be, dt = backend(), TYPES[dtype]
    rows, K, H, L = 300, 48, 64, 4
    gen = torch.Generator(device=DEV).manual_seed(3)
    rand = lambda *s, scale=1.0: (torch.randn(s, generator=gen, device=DEV) * scale).to(dt)
    x, dy = rand(rows, K), rand(rows, K)
    w1, b1 = rand(trees * L, 2 * H, K, scale=K ** -0.5), rand(trees * L, 2 * H)
    w2, b2 = rand(trees * L, K, H, scale=H ** -0.5), rand(trees * L, K)
    leaf = torch.randint(-1, L, (rows, trees), generator=gen, device=DEV).int()

    def step():
        g = be.leaf_groups(leaf, L)
        h, z = be.leaf_layer(x, w1, g, bias=b1, activation=act, gated=True, keep=True)
        y = be.leaf_layer(h, w2, g, bias=b2, residual=x)
        dh, dw2, db2 = be.leaf_layer_grad(dy, None, h, w2, g)
        dx, dw1, db1 = be.leaf_layer_grad(dh, z, x, w1, g, activation=act, gated=True)
        dx += dy
        norm = be.clip_grads([dw1, db1, dw2, db2], 0.5)
        return y, dx, dw1, db1, dw2, db2, norm

    eager = step()
    total = sum(float(t.double().square().sum()) for t in eager[2:6]) ** 0.5
    assert abs(total - 0.5) <= 0.5 * torch.finfo(dt).eps
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(4):
        x.copy_(rand(rows, K))
        leaf.copy_(torch.randint(-1, L, (rows, trees), generator=gen, device=DEV).int())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), turn


def as_products():
    """A layer of no activation and no residual against the linear maps, its gradients bit for bit."""
    be = backend()
    for dtype, rows, K, H, trees, leaves in (("f32", 500, 70, 65, 1, 4), ("bf16", 700, 129, 96, 2, 3),
                                             ("f16", 100, 28, 10, 3, 5), ("bf16", 900, 256, 256, 1, 2)):
        c = Case(rows, K, H, trees, leaves, dtype, act="none", residual=False, seed=rows)
        y = be.leaf_product(c.x, c.w, c.groups, bias=c.b)
        near(y, c.y, c.y_off, "product")
        near(c.layer(), c.y, c.y_off, "layer")
        dx = be.leaf_product_dx(c.dy, c.w, c.groups)
        dw, db = be.leaf_product_dw(c.dy, c.x, c.groups)
        got = c.grad(None, weight_out=torch.empty_like(dw), bias_out=torch.empty_like(db))
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw) and torch.equal(got[2], db)


def far_offsets():
    """Rows whose y and z lie behind 2^31 elements and 2^32 bytes: the last ones, from torch."""
    be = backend()
    rows, K, H = 1100000, 16, 2048
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn((rows, K), generator=gen, device=DEV).bfloat16()
    w = torch.randn((2, H, K), generator=gen, device=DEV).bfloat16()
    leaf = torch.randint(0, 2, (rows, 1), generator=gen, device=DEV).int()
    g = be.leaf_groups(leaf, 2)
    y, z = be.leaf_layer(x, w, g, activation="relu", keep=True)
    assert z.numel() > 2 ** 31
    dx, dw, _ = be.leaf_layer_grad(y, z, x, w, g, activation="relu", bias=False)
    for at in (0, rows // 2, rows - 300):
        n = slice(at, at + 300)
        want = (x[n].double()[:, None, :] @ w[leaf[n, 0].long()].double().transpose(1, 2).contiguous())[:, 0]
        assert (z[0, n].double() - want).abs().max() <= 2 * (K + 3) * U * 16 * K
        assert (y[n].double() - want.clamp(min=0)).abs().max() <= 2.0 ** -8 * want.abs().max()
        # y, and dz = y where z > 0, are bfloat16 here already; dx adds 2048 of them
        dz = torch.where(z[0, n] > 0, y[n].double(), 0.0)
        back = (dz[:, None, :] @ w[leaf[n, 0].long()].double())[:, 0]
        size = (dz.abs()[:, None, :] @ w[leaf[n, 0].long()].double().abs())[:, 0]
        assert bool(((dx[n].double() - back).abs() <= 2.0 ** -8 * back.abs() + 2 * (H + 2) * U * size).all())


def runs_of_planes():
    """More trees than have their planes in the working memory at a time: z, y and dx against
    the same forest, a few trees a call."""
    be = backend()
    rows, K, H, trees, leaves = 150000, 8, 64, 130, 3
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn((rows, K), generator=gen, device=DEV)
    w = torch.randn((trees * leaves, H, K), generator=gen, device=DEV)
    b = torch.randn((trees * leaves, H), generator=gen, device=DEV)
    r, dy = (torch.randn((rows, H), generator=gen, device=DEV) for _ in range(2))
    leaf = torch.randint(-1, leaves, (rows, trees), generator=gen, device=DEV).int()
    g = be.leaf_groups(leaf, leaves)
    assert rows * H * 4 * trees > 2 ** 32
    y, z = be.leaf_layer(x, w, g, bias=b, activation="sigmoid", residual=r, keep=True)
    dx, dw, db = be.leaf_layer_grad(dy, z, x, w, g, activation="sigmoid")
    want, back = r.double(), torch.zeros((rows, K), device=DEV, dtype=torch.float64)
    for t in range(0, trees, 13):
        few = LeafGroups(*(v[t:t + 13].contiguous() for v in g))
        at = slice(t * leaves, (t + 13) * leaves)
        part, kept = be.leaf_layer(x, w[at], few, bias=b[at], activation="sigmoid", keep=True)
        assert torch.equal(kept, z[t:t + 13])
        dxp, dwp, dbp = be.leaf_layer_grad(dy, kept, x, w[at], few, activation="sigmoid")
        # (a forest of fewer trees splits its leaves' rows otherwise, so dw is not bit for bit that)
        n = torch.nonzero(leaf[:, t] == 1)[:, 0]
        p = z[t, n].double().sigmoid()
        dz = dy[n].double() * p * (1 - p)
        # dz is off by slope_error's 16 U (1 + |z|) |dy| (|z| < 18 here is held at 18) and its own
        # rounding; a chain of at most 8192 float32 adds by 2 (8192 + 2) U of the terms' size
        off = dy[n].double().abs() * 16 * U * 19 + 5 * U * dz.abs() + 2 * (8192 + 2) * U * dz.abs()
        assert bool(((dw[t * leaves + 1] - dz.t() @ x[n].double()).abs() <= off.t() @ x[n].double().abs()).all())
        assert bool(((db[t * leaves + 1] - dz.sum(0)).abs() <= off.sum(0)).all())
        want += part
        back += dxp
    # every part is rounded to float32 once, and so is the whole
    assert bool(((y - want).abs() <= U * (11 * 13 + want.abs())).all())
    scale = 11 * U * 13 * H * 6 * 6
    assert (dx - back).abs().max() <= scale


def streams():
    """Calls on two streams at once, and one whose inputs another stream made."""
    be = backend()
    c = [Case(1500, 70, 50, 2, 5, "f32", act="gelu", seed=1), Case(900, 256, 300, 1, 3, "bf16", act="silu", gated=True, seed=2)]
    want = [v.layer(keep=True) for v in c]
    ways = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(5):
        for s in ways:
            s.wait_stream(torch.cuda.current_stream())
        got = [None, None]
        for i, s in enumerate(ways):
            with torch.cuda.stream(s):
                y, z = c[i].layer(keep=True)
                got[i] = (y, z, *c[i].grad(z), be.grad_norm([y, z.to(y.dtype)]))
        for s in ways:
            torch.cuda.current_stream().wait_stream(s)
        for i in range(2):
            again = c[i].grad(want[i][1])
            for a, b in zip(got[i], (*want[i], *again)):
                assert torch.equal(a, b), (turn, i)


def graph_of_norms():
    """A clip captured and replayed over new gradients, long lists among them."""
    be = backend()
    flat = torch.zeros(300007, device=DEV)
    ts = list(flat.split([1000] * 300 + [7]))
    other = torch.zeros(5000, dtype=torch.bfloat16, device=DEV)
    out = [torch.empty_like(t) for t in ts + [other]]
    graph = torch.cuda.CUDAGraph()
    be.clip_grads(ts + [other], 3.0, out=out)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        norm = be.clip_grads(ts + [other], 3.0, out=out)
    for turn in range(4):
        flat.copy_(torch.randn(flat.shape, device=DEV) * 10.0 ** (turn - 3))
        other.copy_(torch.randn(other.shape, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got, held = norm.clone(), [o.clone() for o in out]
        assert torch.equal(got, be.clip_grads(ts + [other], 3.0, out=out))
        for a, b in zip(held, out):
            assert torch.equal(a, b), turn


def inference():
    """Tensors of inference mode, which have no version to count."""
    be = backend()
    with torch.inference_mode():
        t = [torch.ones(10, device=DEV), torch.ones(6, device=DEV)]
        assert float(be.clip_grads(t, 2.0)) == 4.0 and bool((t[0] == 0.5).all())
        c = Case(50, 20, 10, act="gelu")
        near(c.layer(out=torch.empty((50, 10), device=DEV)), c.y, c.y_off, "y")


def _of_one_input(z, dtype, outputs, inputs):
    """x [rows, inputs] and weights [1, outputs, inputs] whose products are z [rows], exactly."""
    x = torch.zeros((len(z), inputs), dtype=TYPES[dtype], device=DEV)
    x[:, 0] = torch.from_numpy(z).to(DEV).to(x.dtype)
    w = torch.zeros((1, outputs, inputs), dtype=x.dtype, device=DEV)
    w[:, :, 0] = 1
    return x, w


def gelu_tails(dtype, rows, inputs, outputs):
    """gelu and its slope relative to their values, as far as the type holds them."""
    be, far = backend(), 5.4 if dtype == "f16" else 12.8
    z = np.concatenate([-np.linspace(0.01, far, rows - rows // 4), np.linspace(0.0, 9.0, rows // 4)])
    x, w = _of_one_input(np.random.default_rng(0).permutation(z), dtype, outputs, inputs)
    g = be.leaf_groups(torch.zeros((rows, 1), dtype=torch.int32, device=DEV), 1)
    value, off, slope, slope_off = oracle.gelu_tails(wide(x[:, 0]), dtype == "f32")
    y = be.leaf_layer(x, w, g, activation="gelu")
    near(y[:, 0], value, off, "gelu")
    assert torch.equal(y, y[:, :1].expand(rows, outputs))
    # dz itself: one output, whose map is a one
    dx, _, _ = be.leaf_layer_grad(torch.ones_like(x[:, :1]), x[None, :, :1].contiguous(), x, w[:, :1].contiguous(), g,
                                  activation="gelu", maps=False)
    near(dx[:, 0], slope, slope_off, "slope")


def sigmoid_slope_tails(dtype):
    """The sigmoid's slope relative to its value, on either side, where 1 - p has few digits left or none."""
    be, far = backend(), 15.0 if dtype == "f16" else 80.0
    x, w = _of_one_input(np.linspace(-far, far, 2001), dtype, 1, 4)
    g = be.leaf_groups(torch.zeros((2001, 1), dtype=torch.int32, device=DEV), 1)
    slope, off = oracle.sigmoid_slope_tails(wide(x[:, 0]))
    for kept in (True, x.dtype):
        _, z = be.leaf_layer(x, w, g, activation="sigmoid", keep=kept)
        dx, _, _ = be.leaf_layer_grad(torch.ones_like(x[:, :1]), z, x, w, g, activation="sigmoid", maps=False)
        near(dx[:, 0], slope, off, "slope")


def clip_beyond_float32():
    """Finite gradients whose norm float32 does not hold, and scales below its normal numbers."""
    be = backend()
    for sizes, value, dtypes in (([4], 3e38, ["f32"]), ([300000, 7], 3e38, ["f32", "bf16"]), ([100], 1e38, ["bf16"]),
                                 ([5000], 1.0, ["f32"])):
        for limit in (1.0, 1e-3, 1e-12, 1e-30, 1e-38, 3e-41):
            ts = [torch.full((n,), value, device=DEV).to(TYPES[dtypes[i % len(dtypes)]]) for i, n in enumerate(sizes)]
            ts[0][0] = -value / 3
            norm, _, want = oracle.clip([wide(t) for t in ts], limit)
            out = [torch.empty_like(t) for t in ts]
            got = float(be.clip_grads(ts, limit, out=out))
            assert got == math.inf if norm > 3.5e38 else abs(got - norm) <= 2 * U * norm, (got, norm)
            for o, w in zip(out, want):
                # the scale's rounding, the product's and, where that is subnormal, the first factor's
                near(o, w, 3 * U * np.abs(w), (value, limit))
            be.clip_grads(ts, limit)
            assert all(torch.equal(t, o) for t, o in zip(ts, out))
