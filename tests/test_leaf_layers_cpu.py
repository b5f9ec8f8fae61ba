"""Layers of a forest's leaves and the clipping of gradients without a GPU: what the C entries
and the Python methods refuse, the sizes of working memory, and the oracle of the GPU tests."""
import ctypes as C
import math
import os
import re

import numpy as np
import pytest

from lightgbm_rs_amd.backend import HipBackend, load_library
from lightgbm_rs_amd.leaves import _GRAD, LeafGroups, _Layer, _LayerGrad, _Maps
from tests import leaf_layer_oracle as oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, MISMATCH, CAPABILITY = -6, -1, -3
# addresses that are never read: every call here is refused, the last for its null context
ORDER, X, WEIGHT, BIAS, RES, Y, Z, WS, DW, DB = (0x10000000000 * k for k in range(1, 11))
BEGIN, COUNT = ORDER + 0x8000000000, ORDER + 0x9000000000


@pytest.fixture(scope="module")
def lib():
    return load_library()


def refused(lib, rc, code, text):
    buf = C.create_string_buffer(512)
    lib.lgbm_hip_last_error(None, buf, 512)
    assert rc == code and text in buf.value.decode(), (rc, buf.value.decode())


def maps(rows=100, trees=1, leaves=7, inputs=5, outputs=3, dtype=0, order=ORDER):
    return _Maps(order, BEGIN, COUNT, rows, trees, leaves, inputs, outputs, dtype, 0)


def layer(lib, m=None, act=2, gated=0, x=X, ldx=5, w=WEIGHT, bias=BIAS, res=RES, ldr=3, y=Y, ldy=3, z=Z,
          z_dtype=0, ws=WS, size=1 << 40):
    a = _Layer(maps(**(m or {})), act, gated, x, ldx, w, bias, res, ldr, y, ldy, z, z_dtype, 0)
    return lib.lgbm_hip_leaf_layer(None, C.byref(a), C.c_void_p(ws), C.c_size_t(size), None)


@pytest.mark.parametrize("change,code,text", [
    (dict(), INVALID, "null context"), (dict(res=None, ldr=0, bias=None, z=None), INVALID, "null context"),
    (dict(m=dict(rows=0)), INVALID, "null context"), (dict(res=Y), INVALID, "null context"),
    (dict(m=dict(rows=-1)), INVALID, "out of range"), (dict(m=dict(inputs=0)), INVALID, "not positive"),
    (dict(m=dict(dtype=1)), INVALID, "dtype"), (dict(act=6), INVALID, "activation"), (dict(act=-1), INVALID, "activation"),
    (dict(gated=2), INVALID, "gated"), (dict(z_dtype=2), INVALID, "z_dtype"), (dict(m=dict(rows=2 ** 31)), CAPABILITY, "2^31"),
    (dict(m=dict(outputs=2 ** 23 + 1), gated=1, ldr=2 ** 24, ldy=2 ** 24), CAPABILITY, "2^24"),
    (dict(m=dict(leaves=2 ** 30, inputs=2 ** 10, outputs=2 ** 8), gated=1, ldx=2 ** 10, ldy=2 ** 8, ldr=2 ** 8),
     CAPABILITY, "2^48"),
    (dict(ldx=4), INVALID, "stride"), (dict(ldy=2), INVALID, "stride"), (dict(ldr=2), INVALID, "stride"),
    (dict(x=None), INVALID, "null x"), (dict(w=None), INVALID, "null x"), (dict(y=None), INVALID, "null x"),
    (dict(x=X + 2), INVALID, "aligned"), (dict(res=RES + 1), INVALID, "aligned"), (dict(z=Z + 2), INVALID, "aligned"),
    (dict(m=dict(dtype=2), z=Z + 2, z_dtype=0), INVALID, "aligned"),
    (dict(m=dict(dtype=2), z=Z + 2, z_dtype=2), INVALID, "null context"),
    (dict(y=X + 400), INVALID, "overlaps"), (dict(y=WEIGHT + 400), INVALID, "overlaps"),
    (dict(y=WEIGHT + 420, gated=1), INVALID, "overlaps"), (dict(y=WEIGHT + 420), INVALID, "null context"),
    (dict(z=RES + 1196), INVALID, "overlaps"), (dict(z=Y - 1196), INVALID, "overlaps"),
    (dict(y=RES + 4), INVALID, "in place"), (dict(y=RES, ldy=4), INVALID, "in place"),
    (dict(m=dict(trees=4), ws=None), INVALID, "null workspace"), (dict(m=dict(trees=4), size=100), MISMATCH, "smaller"),
    (dict(m=dict(trees=4), ws=WS + 8), INVALID, "16-byte"), (dict(m=dict(trees=4), ws=RES), INVALID, "overlaps"),
    (dict(m=dict(rows=2 ** 24, leaves=2 ** 24, outputs=2 ** 18), ldy=2 ** 18, ldr=2 ** 18), CAPABILITY, "one launch")])
def test_layer_refused(lib, change, code, text):
    refused(lib, layer(lib, **change), code, text)


def grad(lib, m=None, act=2, gated=0, dy=RES, lddy=3, z=Z, x=X, ldx=5, w=WEIGHT, dx=Y, lddx=5, dw=DW, db=DB,
         dw_dtype=0, z_dtype=0, ws=WS, size=1 << 40):
    a = _LayerGrad(maps(**(m or {})), act, gated, dy, lddy, z, x, ldx, w, dx, lddx, dw, db, dw_dtype, z_dtype)
    return lib.lgbm_hip_leaf_layer_grad(None, C.byref(a), C.c_void_p(ws), C.c_size_t(size), None)


@pytest.mark.parametrize("change,code,text", [
    (dict(), INVALID, "null context"), (dict(dx=None, w=None, lddx=0), INVALID, "null context"),
    (dict(dw=None, db=None, x=None, ldx=0), INVALID, "null context"), (dict(db=None), INVALID, "null context"),
    (dict(act=0, z=None), INVALID, "null context"), (dict(act=0, z=Y), INVALID, "null context"),
    (dict(m=dict(rows=0), dw=None, db=None), INVALID, "null context"), (dict(m=dict(rows=0)), INVALID, "null context"),
    (dict(act=0, gated=1, z=None), INVALID, "null dy"), (dict(z=None), INVALID, "null dy"), (dict(dy=None), INVALID, "null dy"),
    (dict(x=None), INVALID, "null dy"), (dict(w=None), INVALID, "null dy"),
    (dict(dx=None, dw=None, db=None), INVALID, "neither"), (dict(dw=None), INVALID, "dbias without"),
    (dict(act=9), INVALID, "activation"), (dict(gated=-1), INVALID, "gated"), (dict(dw_dtype=2), INVALID, "dw_dtype"),
    (dict(z_dtype=3), INVALID, "z_dtype"), (dict(lddy=2), INVALID, "stride"), (dict(ldx=4), INVALID, "stride"),
    (dict(lddx=4), INVALID, "stride"), (dict(dw=DW + 2), INVALID, "aligned"), (dict(dy=RES + 2), INVALID, "aligned"),
    (dict(m=dict(dtype=3), dw_dtype=3, dw=DW + 2), INVALID, "null context"),
    (dict(m=dict(dtype=3), dw_dtype=0, dw=DW + 2), INVALID, "aligned"),
    (dict(dx=RES + 400), INVALID, "overlaps"), (dict(dx=Z + 400), INVALID, "overlaps"), (dict(dw=X + 4), INVALID, "overlaps"),
    (dict(db=DW + 400), INVALID, "overlaps"), (dict(dw=WEIGHT), INVALID, "overlaps"), (dict(ws=Z), INVALID, "overlaps"),
    (dict(ws=None), INVALID, "null workspace"), (dict(size=100), MISMATCH, "smaller"), (dict(ws=WS + 4), INVALID, "16-byte")])
def test_grad_refused(lib, change, code, text):
    refused(lib, grad(lib, **change), code, text)


def test_workspaces(lib):
    """z's gradient, in the type, and what the products of it need."""
    need, one = C.c_size_t(0), C.c_size_t(0)
    for dtype, size in ((0, 4), (2, 2)):
        for gated, trees in ((0, 1), (1, 1), (1, 3)):
            m = maps(rows=1000, trees=trees, inputs=64, outputs=40, dtype=dtype)
            a = _LayerGrad(m, 2, gated, RES, 40, Z, X, 64, WEIGHT, Y, 64, None, None, dtype, 0)
            assert lib.lgbm_hip_leaf_layer_grad_workspace(C.byref(a), C.byref(need)) == 0
            wide = maps(rows=1000, trees=trees, inputs=64, outputs=40 * (1 + gated), dtype=dtype)
            assert lib.lgbm_hip_leaf_product_workspace(C.byref(wide), C.c_int32(1), C.byref(one)) == 0
            dz = 1000 * trees * 40 * (1 + gated) * size
            assert dz + one.value <= need.value <= dz + one.value + 256
            f = _Layer(m, 2, gated, X, 64, WEIGHT, None, None, 0, Y, 40, None, 0, 0)
            assert lib.lgbm_hip_leaf_layer_workspace(C.byref(f), C.byref(need)) == 0
            assert need.value == (0 if trees == 1 else (1000 * 40 * 4 * trees + 15) // 16 * 16)
    # a linear layer's dz is dy
    a = _LayerGrad(maps(), 0, 0, RES, 3, None, X, 5, WEIGHT, Y, 5, None, None, 0, 0)
    assert lib.lgbm_hip_leaf_layer_grad_workspace(C.byref(a), C.byref(need)) == 0 and need.value == 0
    assert lib.lgbm_hip_leaf_layer_grad_workspace(C.byref(a), None) == INVALID
    assert lib.lgbm_hip_leaf_layer_workspace(None, C.byref(need)) == INVALID


def grads_of(*entries):
    a = np.zeros(len(entries), _GRAD)
    for i, e in enumerate(entries):
        a[i] = (*e, 0)
    return a


def clip(lib, a, n=None, limit=1.0, norm=Y, ws=WS, size=1 << 40):
    return lib.lgbm_hip_clip_grads(None, C.c_void_p(a.ctypes.data if len(a) else None), C.c_int64(len(a) if n is None else n),
                                   C.c_double(limit), C.c_void_p(norm), C.c_void_p(ws), C.c_size_t(size), None)


ONE = (X, X, 100, 0)


@pytest.mark.parametrize("entries,change,code,text", [
    ([ONE], dict(), INVALID, "null context"), ([], dict(), INVALID, "null context"),
    ([ONE, (X + 400, X + 400, 10, 2), (0, 0, 0, 0)], dict(), INVALID, "null context"),
    ([(X, DW, 100, 0), (X, DB, 100, 0)], dict(), INVALID, "null context"),  # inputs may be the same
    ([(X + 800, DW + 800, 100, 3), (X, DW, 100, 0)], dict(), INVALID, "null context"),
    ([ONE], dict(n=-1), INVALID, "negative list"), ([ONE], dict(n=2 ** 25), CAPABILITY, "2^24"),
    ([(X, X, -1, 0)], dict(), INVALID, "negative count"), ([(X, X, 10, 1)], dict(), INVALID, "dtype"),
    ([(X, X, 2 ** 49, 0)], dict(), CAPABILITY, "2^48"),
    ([(0, X, 10, 0)], dict(), INVALID, "null gradient"), ([(X, 0, 10, 0)], dict(), INVALID, "null gradient"),
    ([(X + 2, X + 2, 10, 0)], dict(), INVALID, "aligned"), ([(X + 1, X + 1, 10, 2)], dict(), INVALID, "aligned"),
    ([ONE, ONE], dict(), INVALID, "overlaps"), ([ONE, (X + 396, X + 396, 1, 0)], dict(), INVALID, "overlaps"),
    ([(X, X + 4, 100, 0)], dict(), INVALID, "overlaps"), ([(X, DW, 100, 0), (DW, DB, 100, 0)], dict(), INVALID, "overlaps"),
    ([(X, DW, 100, 0), (DB, DW + 396, 100, 0)], dict(), INVALID, "overlaps"),
    ([ONE], dict(norm=X + 8), INVALID, "overlaps"), ([ONE], dict(ws=X - 16), INVALID, "overlaps"),
    ([ONE], dict(norm=None), INVALID, "null norm"), ([ONE], dict(norm=Y + 2), INVALID, "aligned"),
    ([ONE], dict(limit=-0.5), INVALID, "negative"), ([ONE], dict(limit=float("nan")), INVALID, "NaN"),
    ([ONE], dict(ws=None), INVALID, "null workspace"), ([ONE], dict(size=8), MISMATCH, "smaller")])
def test_clip_refused(lib, entries, change, code, text):
    refused(lib, clip(lib, grads_of(*entries), **change), code, text)


def test_norm_refused(lib):
    def norm(a, at=Y, ws=WS):
        return lib.lgbm_hip_grad_norm(None, C.c_void_p(a.ctypes.data), C.c_int64(len(a)), C.c_void_p(at), C.c_void_p(ws),
                                      C.c_size_t(1 << 40), None)
    refused(lib, norm(grads_of((X, 0, 100, 0), (X, 0, 100, 0))), INVALID, "null context")
    refused(lib, norm(grads_of((X, 0, 100, 0)), at=X + 4), INVALID, "overlaps")
    refused(lib, norm(grads_of((X, 0, 100, 0)), ws=X + 16), INVALID, "overlaps")
    refused(lib, norm(grads_of((X, 0, 100, 0)), at=WS), INVALID, "overlaps")


def test_norm_workspace(lib):
    """A sum for every chunk: about 4096 of the whole, and an end of every tensor."""
    need = C.c_size_t(0)
    for counts in ([1], [0, 0], [4096] * 50, [10 ** 9, 5, 10 ** 9], [3] * 5000):
        a = grads_of(*[(X, X, n, 0) for n in counts])
        assert lib.lgbm_hip_grad_norm_workspace(C.c_void_p(a.ctypes.data), C.c_int64(len(a)), C.byref(need)) == 0
        assert need.value <= 16 + 8 * (4097 + len(counts))


def test_struct_layouts(lib):
    """The ctypes structs have the fields of the header's, in its order."""
    text = open(os.path.join(ROOT, "include", "lgbm_hip.h")).read()
    sizes = {"int32_t": C.c_int32, "int64_t": C.c_int64, "lgbm_leaf_maps": _Maps}
    of_numpy = {"d_in": "in", "d_out": "out"}
    for name, struct in (("lgbm_leaf_layer", _Layer), ("lgbm_leaf_layer_grad", _LayerGrad), ("lgbm_grad", None)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = re.findall(r"([\w ]+?)(\*?)\s*\b(\w+);", body)
        if struct is None:
            assert [of_numpy.get(f[2], f[2]) for f in fields] == list(_GRAD.names) and _GRAD.itemsize == 32
            continue
        assert [f[2].replace("d_", "", 1) if f[2].startswith("d_") else f[2] for f in fields] == \
            [n for n, _ in struct._fields_]
        for (kind, star, _), (_, got) in zip(fields, struct._fields_):
            assert got is (C.c_void_p if star else sizes[kind.strip()]), kind


class Plain(HipBackend):
    """The checks that come before the library is called."""

    def __init__(self):
        self.lib, self.ctx, self.device = load_library(), None, 0


def test_python_refuses():
    import torch
    be, z = Plain(), torch.zeros
    g = LeafGroups(*(z(s, dtype=torch.int32) for s in ((1, 6), (1, 4), (1, 4))))
    x, w, dy, k = z((6, 5)), z((4, 2, 5)), z((6, 2)), z((1, 6, 2))
    for call, text in [
            (lambda: be.leaf_layer(x, w, g, activation="swish"), "activation"),
            (lambda: be.leaf_layer(x[0], w, g), "rows, inputs"), (lambda: be.leaf_layer(x, w[:, :1], g, gated=True), "even"),
            (lambda: be.leaf_layer(x, w.half(), g), "differ"), (lambda: be.leaf_layer(x, w, g, bias=z((4, 3))), "shape"),
            (lambda: be.leaf_layer(x, w, g, residual=z((6, 3))), "shape"),
            (lambda: be.leaf_layer(x, w, g, residual=dy.half()), "differ"), (lambda: be.leaf_layer(x, w, g), "is on cpu"),
            (lambda: be.leaf_layer_grad(dy, None, x, w, g, activation="relu"), "z is needed"),
            (lambda: be.leaf_layer_grad(dy, None, x, w, g, gated=True), "shape"),
            (lambda: be.leaf_layer_grad(dy[:5], k, x, w, g, activation="relu"), "shape"),
            (lambda: be.leaf_layer_grad(dy, k, x, w, g, activation="relu", maps=False, inputs=False), "neither"),
            (lambda: be.leaf_layer_grad(dy, k, x, w, g, maps=False, bias_out=z((4, 2))), "not asked"),
            (lambda: be.leaf_layer_grad(dy, None, x, w, g), "is on cpu"),
            (lambda: be.grad_norm([x]), "is on cpu"), (lambda: be.clip_grads([x[:, :2]], 1.0), "gaps"),
            (lambda: be.clip_grads([x], 1.0, out=[x, x]), "number"), (lambda: be.clip_grads([x], 1.0, out=[w]), "differ"),
            (lambda: be.grad_norm([x.int()]), "is on cpu")]:
        with pytest.raises(ValueError, match=text):
            call()


def test_clip_outputs_by_shape():
    import torch
    be, z = Plain(), torch.zeros
    # strides of dimensions of one element do not matter, shapes do, also where strides are the same
    for t, out, text in [(z((1, 6)), z((6, 1)).t(), "is on cpu"), (z((3, 0, 2)), z((2, 0, 3)).permute(2, 1, 0), "is on cpu"),
                         (z((2, 3)), z(6).as_strided((1, 6), (3, 1)), "differ"), (z((2, 3)), z((3, 2)).t(), "differ"),
                         (z(1), z(()), "differ"), (z((6,)), z((6, 1)), "differ")]:
        with pytest.raises(ValueError, match=text):
            be.clip_grads([t, z(4)], 1.0, out=[out, z(4)])


def test_python_refuses_what_autograd_would_lose():
    import torch
    be, z = Plain(), torch.zeros
    g = LeafGroups(*(z(s, dtype=torch.int32) for s in ((1, 6), (1, 4), (1, 4))))
    calls = [(lambda x, w, dy: be.leaf_layer(x, w, g), "x"), (lambda x, w, dy: be.leaf_layer(x, w, g), "w"),
             (lambda x, w, dy: be.leaf_layer(x, w, g, residual=dy), "dy"),
             (lambda x, w, dy: be.leaf_layer_grad(dy, None, x, w, g), "dy"),
             (lambda x, w, dy: be.grad_norm([x, dy]), "dy"), (lambda x, w, dy: be.clip_grads([w], 1.0), "w")]
    for call, name in calls:
        t = {"x": z((6, 5)), "w": z((4, 2, 5)), "dy": z((6, 2))}
        t[name].requires_grad_()
        with pytest.raises(ValueError, match="requires? gradients"):
            call(**t)
        with torch.no_grad(), pytest.raises(ValueError, match="is on cpu"):
            call(**t)


@pytest.mark.parametrize("act", oracle.ACTIVATIONS)
def test_oracle_slopes(act):
    """The slopes against differences, and the steepest."""
    z = np.linspace(-9, 9, 1801) + 1e-3
    h = 1e-6
    by_differences = (oracle.activation(z + h, act) - oracle.activation(z - h, act)) / (2 * h)
    assert np.abs(oracle.slope(z, act) - by_differences).max() < 1e-8
    assert np.abs(oracle.slope(z, act)).max() <= oracle.STEEPEST


@pytest.mark.parametrize("gated", [False, True])
def test_oracle_against_loops(gated):
    rng = np.random.default_rng(0)
    leaf = rng.integers(-1, 4, (11, 2)).astype(np.int32)
    R = 8 if gated else 4
    x, w, b, r, dy = (rng.standard_normal(s) for s in ((11, 5), (6, R, 5), (6, R), (11, 4), (11, 4)))
    y, z = r.copy(), np.zeros((2, 11, R))
    dx, dw, db = np.zeros((11, 5)), np.zeros((6, R, 5)), np.zeros((6, R))
    for n in range(11):
        for t in range(2):
            if not 0 <= leaf[n, t] < 3:
                continue
            g = 3 * t + leaf[n, t]
            z[t, n] = v = w[g] @ x[n] + b[g]
            p = 1 / (1 + np.exp(-v[:4]))
            f, s = v[:4] * p, p + v[:4] * p * (1 - p)
            y[n] += f * v[4:] if gated else f
            d = np.concatenate([dy[n] * v[4:] * s, dy[n] * f]) if gated else dy[n] * s
            dx[n] += w[g].T @ d
            dw[g] += np.outer(d, x[n])
            db[g] += d
    got, off, kept, _ = oracle.layer(x, w, b, leaf, 3, "silu", gated, r)
    assert np.allclose(got, y) and np.allclose(kept, z) and off.max() < 1e-3
    want = oracle.grads(dy, kept, x, w, leaf, 3, "silu", gated, 2.0 ** -23, 0.0)
    for name, value in (("dx", dx), ("dw", dw), ("db", db)):
        assert np.allclose(want[name][0], value), name


def test_oracle_clip():
    norm, scale, out = oracle.clip([np.array([3.0]), np.array([[0.0, -4.0]])], 2.5)
    assert norm == 5.0 and scale == 0.5 and out[1][0, 1] == -2.0
    assert oracle.clip([np.array([3.0])], 3.0)[1] == 1.0


def test_polynomial_of_erfc():
    """The kernels' polynomial for 16-bit types is off by 4e-8 and 5e-6 of itself at most, where float32 holds it."""
    text = open(os.path.join(ROOT, "lightgbm_rs_amd", "csrc", "leaf_layer.h")).read()
    rate = float(re.search(r"BELOW_RATE = ([\d.]+)f", text).group(1))
    powers = [float(v) for v in re.findall(r"-?[\d.]+(?=f)", re.search(r"BELOW\[7\] = \{(.*?)\}", text, re.S).group(1))]
    a = np.linspace(0.0, 9.2, 20001)
    t = 1 / (1 + rate * a)
    got = 2 * np.exp(-a * a) * sum(c * t ** (k + 1) for k, c in enumerate(powers))
    want = np.array([math.erfc(v) for v in a])
    assert len(powers) == 7 and np.abs(got - want).max() < 4e-8 and (np.abs(got - want) / want).max() < 5e-6


def test_python_refuses_tangents():
    """Forward-mode differentiation would go on without the tangent of the output: refused, also under
    no_grad, which does not turn it off; the primal, and what a Function's methods get, go on."""
    import torch
    from torch.autograd import forward_ad
    be, z = Plain(), torch.zeros
    g = LeafGroups(*(z(s, dtype=torch.int32) for s in ((1, 6), (1, 4), (1, 4))))
    calls = [(lambda x, w, dy: be.leaf_layer(x, w, g), "x"), (lambda x, w, dy: be.leaf_layer(x, w, g), "w"),
             (lambda x, w, dy: be.leaf_layer(x, w, g, residual=dy), "dy"),
             (lambda x, w, dy: be.leaf_layer_grad(dy, None, x, w, g), "dy"),
             (lambda x, w, dy: be.leaf_layer_grad(dy, dy[None], x, w, g, activation="silu"), "x"),
             (lambda x, w, dy: be.grad_norm([x, dy]), "dy"), (lambda x, w, dy: be.clip_grads([w], 1.0), "w"),
             (lambda x, w, dy: be.clip_grads([w], 1.0, out=[z((4, 2, 5))]), "w"),
             (lambda x, w, dy: be.leaf_product(x, w, g), "x"), (lambda x, w, dy: be.leaf_product_dx(dy, w, g), "w"),
             (lambda x, w, dy: be.leaf_product_dw(dy, x, g), "x"), (lambda x, w, dy: be.dropout(x, 0.5, 1), "x"),
             (lambda x, w, dy: be.dropout(x[:, 0], 0.5, 1), "x"), (lambda x, w, dy: be.adjust_scores(x, bias=w[0, 0]), "w")]

    class Through(torch.autograd.Function):
        @staticmethod
        def forward(ctx, call, x, w, dy):
            call(x, w, dy)

    for call, name in calls:
        t = {"x": z((6, 5)), "w": z((4, 2, 5)), "dy": z((6, 2))}
        with forward_ad.dual_level():
            with pytest.raises(ValueError, match="is on cpu"):
                call(**t)
            t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
            with pytest.raises(ValueError, match="has a tangent"):
                call(**t)
            with torch.no_grad(), pytest.raises(ValueError, match="has a tangent"):
                call(**t)
            with pytest.raises(ValueError, match="is on cpu"):
                Through.apply(call, t["x"], t["w"], t["dy"])
            with pytest.raises(ValueError, match="is on cpu"):
                call(**{k: v.detach() for k, v in t.items()})
            t[name] = forward_ad.unpack_dual(t[name]).primal
            with pytest.raises(ValueError, match="is on cpu"):
                call(**t)
