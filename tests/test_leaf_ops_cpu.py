"""The operators around a forest's leaves without a GPU: what the C entries and the Python
methods refuse, the sizes of working memory, and the oracle of the GPU tests."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from lightgbm_rs_amd.backend import HipBackend, load_library
from lightgbm_rs_amd.leaves import LeafGroups, _Maps, _Scores
from tests import leaf_ops_oracle as oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, MISMATCH, CAPABILITY = -6, -1, -3
# addresses that are never read: every call here is refused, the last for its null context
A, B, D, E, F, W = (0x10000000000 * k for k in range(1, 7))


@pytest.fixture(scope="module")
def lib():
    return load_library()


def message(lib):
    buf = C.create_string_buffer(512)
    lib.lgbm_hip_last_error(None, buf, 512)
    return buf.value.decode()


def refused(lib, rc, code, text):
    assert rc == code and text in message(lib), (rc, message(lib))


def groups(lib, leaf=A, ld=3, rows=10, trees=3, leaves=7, order=B, begin=D, count=E, ws=W, size=1 << 30):
    p = C.c_void_p
    return lib.lgbm_hip_leaf_groups(None, p(leaf), C.c_int64(ld), C.c_int64(rows), C.c_int32(trees),
                                    C.c_int32(leaves), p(order), p(begin), p(count), p(ws),
                                    C.c_size_t(size), None)


@pytest.mark.parametrize("change,code,text", [
    (dict(), INVALID, "null context"), (dict(rows=-1), INVALID, "out of range"),
    (dict(trees=0), INVALID, "out of range"), (dict(leaves=0), INVALID, "out of range"),
    (dict(rows=2 ** 31), CAPABILITY, "2^31"), (dict(trees=65536, ld=65536), CAPABILITY, "65535"),
    (dict(leaves=4096), CAPABILITY, "4095"), (dict(ld=2), INVALID, "stride"),
    (dict(leaf=None), INVALID, "null leaf"), (dict(count=None), INVALID, "null leaf"),
    (dict(order=B + 2), INVALID, "aligned"), (dict(rows=10 ** 6, ws=None), INVALID, "null workspace"),
    (dict(rows=10 ** 6, ws=W + 4), INVALID, "16-byte"), (dict(rows=10 ** 6, size=8), MISMATCH, "smaller"),
    (dict(order=A + 40), INVALID, "overlap"), (dict(count=D + 40), INVALID, "overlap"),
    (dict(rows=10 ** 6, ws=A - 64), INVALID, "overlap"), (dict(ld=2 ** 41), INVALID, "stride"),
    (dict(rows=2 ** 30, ld=2 ** 34), INVALID, "stride")])
def test_groups_refused(lib, change, code, text):
    refused(lib, groups(lib, **change), code, text)


def maps(order=A, begin=B, count=B + 4096, rows=100, trees=1, leaves=7, inputs=5, outputs=3, dtype=0):
    return _Maps(order, begin, count, rows, trees, leaves, inputs, outputs, dtype, 0)


def calls(lib, m, p1=D, ld1=5, p2=E, p3=None, out=F, ldo=3, ws=W, size=1 << 40):
    """The three products on the same shape: (y, dx, dw)."""
    p, i64, n = C.c_void_p, C.c_int64, C.c_size_t
    ref = None if m is None else C.byref(m)
    yield lib.lgbm_hip_leaf_product(None, ref, p(p1), i64(ld1), p(p2), p(p3), p(out), i64(ldo), p(ws), n(size), None)
    yield lib.lgbm_hip_leaf_product_dx(None, ref, p(p1), i64(ldo), p(p2), p(out), i64(ld1), p(ws), n(size), None)
    yield lib.lgbm_hip_leaf_product_dw(None, ref, p(p1), i64(ldo), p(p2), i64(ld1), p(out), p(p3), p(ws), n(size), None)


@pytest.mark.parametrize("m,change,code,text", [
    (dict(), dict(), INVALID, "null context"), (None, dict(), INVALID, "null maps"),
    (dict(rows=-1), dict(), INVALID, "out of range"), (dict(leaves=0), dict(), INVALID, "out of range"),
    (dict(inputs=0), dict(), INVALID, "not positive"), (dict(outputs=-2), dict(), INVALID, "not positive"),
    (dict(dtype=1), dict(), INVALID, "dtype"), (dict(dtype=9), dict(), INVALID, "dtype"),
    (dict(order=None), dict(), INVALID, "null order"), (dict(count=None), dict(), INVALID, "null order"),
    (dict(rows=2 ** 31), dict(), CAPABILITY, "2^31"), (dict(trees=65536), dict(), CAPABILITY, "65535"),
    (dict(trees=65535, leaves=2 ** 20), dict(), CAPABILITY, "2^31"),
    (dict(inputs=2 ** 25), dict(ld1=2 ** 25), CAPABILITY, "2^24"),
    (dict(), dict(ld1=4), INVALID, "stride"), (dict(), dict(ldo=2), INVALID, "stride"),
    (dict(), dict(p1=None), INVALID, "null"), (dict(), dict(p2=None), INVALID, "null"),
    (dict(), dict(out=None), INVALID, "null"), (dict(), dict(p1=D + 2), INVALID, "aligned"),
    (dict(), dict(out=F + 1), INVALID, "aligned"), (dict(), dict(out=D + 400), INVALID, "overlaps"),
    (dict(), dict(out=E - 400), INVALID, "overlaps"), (dict(), dict(out=A + 396), INVALID, "overlaps"),
    (dict(), dict(out=B + 4096), INVALID, "overlaps"),
    (dict(leaves=2 ** 30, outputs=4096, inputs=4096), dict(ld1=4096, ldo=4096), CAPABILITY, "2^48"),
    (dict(rows=8192, leaves=8192, outputs=2 ** 17, inputs=2 ** 17), dict(ld1=2 ** 17, ldo=2 ** 17),
     CAPABILITY, "one launch")])
def test_products_refused(lib, m, change, code, text):
    for rc in calls(lib, None if m is None else maps(**m), **change):
        refused(lib, rc, code, text)


def test_products_refused_workspace(lib):
    m = maps(trees=4)
    need = C.c_size_t(0)
    for what, cols in ((0, 3), (1, 5)):
        assert lib.lgbm_hip_leaf_product_workspace(C.byref(m), C.c_int32(what), C.byref(need)) == 0
        assert need.value >= 4 * 100 * cols * 4
    for change, code, text in ((dict(ws=None), INVALID, "null workspace"), (dict(size=100), MISMATCH, "smaller"),
                               (dict(ws=W + 8), INVALID, "16-byte"), (dict(ws=D), INVALID, "overlaps")):
        it = calls(lib, m, **change)
        for _ in range(2):
            refused(lib, next(it), code, text)
    assert lib.lgbm_hip_leaf_product_workspace(C.byref(m), C.c_int32(3), C.byref(need)) == INVALID
    assert lib.lgbm_hip_leaf_product_workspace(C.byref(m), C.c_int32(0), None) == INVALID


def dropout(lib, x=A, ldx=8, rows=100, cols=8, dtype=0, p=0.5, out=B, ldo=8):
    return lib.lgbm_hip_dropout(None, C.c_void_p(x), C.c_int64(ldx), C.c_int64(rows), C.c_int64(cols),
                                C.c_int32(dtype), C.c_double(p), C.c_uint64(1), C.c_uint64(0), C.c_int32(0),
                                C.c_void_p(out), C.c_int64(ldo), None)


@pytest.mark.parametrize("change,code,text", [
    (dict(), INVALID, "null context"), (dict(rows=0), INVALID, "null context"),
    (dict(out=A), INVALID, "null context"), (dict(p=-0.1), INVALID, "p outside"),
    (dict(p=1.01), INVALID, "p outside"), (dict(p=float("nan")), INVALID, "p outside"),
    (dict(dtype=1), INVALID, "dtype"), (dict(rows=-1), INVALID, "negative"),
    (dict(cols=9), INVALID, "stride"), (dict(x=None), INVALID, "null x"), (dict(out=None), INVALID, "null x"),
    (dict(x=A + 2), INVALID, "aligned"), (dict(out=A + 32), INVALID, "other than in place"),
    (dict(out=A, ldo=16), INVALID, "other than in place")])
def test_dropout_refused(lib, change, code, text):
    refused(lib, dropout(lib, **change), code, text)


def score_args(**change):
    a = dict(x=A, ldx=40, num_rows=6, num_classes=40, dtype=0, kind=0, num_masks=0, bias=None, mask=None,
             mask_rows=None, ids=None, offsets=None, num_ids=0, repetition=1.0, frequency=0.0,
             presence=0.0, penalties=None, out=B, ldo=40)
    a.update(change)
    return _Scores(*a.values())


HISTORY = dict(ids=D, offsets=E, num_ids=50)


@pytest.mark.parametrize("change,code,text", [
    (dict(), INVALID, "null context"), (dict(num_rows=0), INVALID, "null context"),
    (dict(out=A), INVALID, "null context"), (dict(dtype=4), INVALID, "dtype"),
    (dict(kind=2), INVALID, "kind"), (dict(num_classes=0), INVALID, "out of range"),
    (dict(num_rows=-1), INVALID, "out of range"), (dict(num_rows=2 ** 31), CAPABILITY, "too many"),
    (dict(ldx=39), INVALID, "stride"), (dict(ldo=39), INVALID, "stride"), (dict(x=None), INVALID, "null x"),
    (dict(out=None), INVALID, "null x"), (dict(mask=D), INVALID, "without masks"),
    (dict(mask=D, num_masks=3), MISMATCH, "mask_rows"),
    (dict(mask=D, num_masks=6), INVALID, "null context"),
    (dict(HISTORY, offsets=None), INVALID, "history"), (dict(HISTORY, ids=None), INVALID, "history"),
    (dict(HISTORY, num_ids=-1), INVALID, "history"), (dict(HISTORY, repetition=0.0), INVALID, "repetition"),
    (dict(HISTORY, repetition=-1.0), INVALID, "repetition"),
    (dict(HISTORY, presence=float("inf")), INVALID, "not finite"),
    (dict(HISTORY, frequency=float("nan")), INVALID, "not finite"),
    (dict(HISTORY, repetition=0.0, penalties=F), INVALID, "null context"),
    (dict(HISTORY, offsets=E + 4), INVALID, "aligned"), (dict(x=A + 1), INVALID, "aligned"),
    (dict(out=A + 160), INVALID, "in place"), (dict(bias=B + 800), INVALID, "overlaps"),
    (dict(HISTORY, ids=B), INVALID, "overlaps"), (dict(mask=B + 900, num_masks=1), INVALID, "overlaps")])
def test_scores_refused(lib, change, code, text):
    rc = lib.lgbm_hip_adjust_scores(None, C.byref(score_args(**change)), C.c_void_p(W), C.c_size_t(1 << 40), None)
    refused(lib, rc, code, text)


def test_struct_layouts(lib):
    """The ctypes structs have the fields of the header's, in its order."""
    text = open(os.path.join(ROOT, "include", "lgbm_hip.h")).read()
    for name, struct in (("lgbm_leaf_maps", _Maps), ("lgbm_score_args", _Scores)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = re.findall(r"([\w ]+?)(\*?)\s*\b(\w+);", body)
        sizes = {"int32_t": C.c_int32, "int64_t": C.c_int64, "double": C.c_double}
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
    be = Plain()
    z = torch.zeros
    i32 = torch.int32
    g = LeafGroups(z((1, 6), dtype=i32), z((1, 4), dtype=i32), z((1, 4), dtype=i32))
    x, w, dy = z((6, 5)), z((4, 3, 5)), z((6, 3))
    cases = [
        lambda: be.leaf_groups(z((6, 2)), 4), lambda: be.leaf_groups(z((6, 0), dtype=i32), 4),
        lambda: be.leaf_product(x.double(), w.double(), g), lambda: be.leaf_product(x, w.half(), g),
        lambda: be.leaf_product(x, z((4, 3, 6)), g), lambda: be.leaf_product(x, w[0], g),
        lambda: be.leaf_product(x, w, g, bias=z((4, 2))), lambda: be.leaf_product(x, w, g, bias=z((4, 3)).half()),
        lambda: be.leaf_product_dx(x, w, g), lambda: be.leaf_product_dw(dy, x.half(), g),
        lambda: be.leaf_product_dw(dy, x[:5], g), lambda: be.leaf_product_dw(dy, x, g, bias=False, bias_out=z((4, 3))),
        lambda: be.dropout(x, 0.5, 1, by="column"), lambda: be.dropout(x.int(), 0.5, 1),
        lambda: be.dropout(z((2, 2, 2)), 0.5, 1), lambda: be.adjust_scores(x, kind="leaf"),
        lambda: be.adjust_scores(x[0]), lambda: be.adjust_scores(x, bias=z(4)),
        lambda: be.adjust_scores(x, bias=z(5).half()), lambda: be.adjust_scores(x, mask=z((6, 2), dtype=i32)),
        lambda: be.adjust_scores(x, mask=z((6, 1))), lambda: be.adjust_scores(x, mask_rows=z(6, dtype=i32)),
        lambda: be.adjust_scores(x, ids=z(3, dtype=i32)),
        lambda: be.adjust_scores(x, ids=z(3, dtype=i32), offsets=z(6, dtype=torch.int64)),
        lambda: be.adjust_scores(x, ids=z(3, dtype=i32), offsets=z(7, dtype=i32)),
        lambda: be.adjust_scores(x, penalties=z((6, 2))),
        # on another device
        lambda: be.leaf_product(x, w, g), lambda: be.dropout(x, 0.5, 1), lambda: be.adjust_scores(x),
        lambda: be.leaf_groups(z((6, 2), dtype=i32), 4)]
    for i, call in enumerate(cases):
        with pytest.raises(ValueError):
            call()
            print(i)


def test_philox_known_answers():
    """The published answers of Philox4x32-10 for the counters and keys of all zeros and all
    ones."""
    assert [hex(v) for v in oracle.philox([0], 0, 0)[0]] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    ones = 2 ** 64 - 1
    assert [hex(v) for v in oracle.philox([ones], ones, ones)[0]] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6",
                                                                     "0x6d5451fd"]


def test_oracle_against_loops():
    rng = np.random.default_rng(0)
    leaf = rng.integers(-1, 4, (11, 2)).astype(np.int32)
    order, begin, count = oracle.groups(leaf, 3)
    for t in range(2):
        assert sorted(order[t]) == list(range(11))
        for l in range(3):
            assert all(leaf[n, t] == l for n in order[t, begin[t, l]:begin[t, l] + count[t, l]])
    x, w, b, dy = (rng.standard_normal(s) for s in ((11, 5), (6, 4, 5), (6, 4), (11, 4)))
    y, dx = np.zeros((11, 4)), np.zeros((11, 5))
    dw, db = np.zeros((6, 4, 5)), np.zeros((6, 4))
    for n in range(11):
        for t in range(2):
            if 0 <= leaf[n, t] < 3:
                g = 3 * t + leaf[n, t]
                y[n] += w[g] @ x[n] + b[g]
                dx[n] += w[g].T @ dy[n]
                dw[g] += np.outer(dy[n], x[n])
                db[g] += dy[n]
    assert np.allclose(oracle.product(x, w, b, leaf, 3)[0], y)
    assert np.allclose(oracle.product_dx(dy, w, leaf, 3)[0], dx)
    got = oracle.product_dw(dy, x, leaf, 3)
    assert np.allclose(got[0], dw) and np.allclose(got[2], db)


def test_whole_numbers_show_every_row():
    """What the GPU's exact gradients are compared with: a row left out, or taken twice, is
    seen in every element of its leaf, and sums stay within float32's whole numbers."""
    rng = np.random.default_rng(1)
    x, dy = oracle.whole_numbers(rng, 400, 7), oracle.whole_numbers(rng, 400, 3)
    assert np.abs(x).max() == 5 and x.min() == -3 and x.all() and dy.all()
    leaf = rng.integers(0, 3, (400, 1)).astype(np.int32)
    dw, _, db, _ = oracle.product_dw(dy, x, leaf, 3)
    for row in (0, 17, 399):
        l = leaf[row, 0]
        lost = leaf.copy()
        lost[row] = -1
        w, _, b, _ = oracle.product_dw(dy, x, lost, 3)
        assert (w[l] != dw[l]).all() and (b[l] != db[l]).all()
        twice = np.concatenate([np.arange(400), [row]])
        w, _, b, _ = oracle.product_dw(dy[twice], x[twice], leaf[twice], 3)
        assert (w[l] != dw[l]).all() and (b[l] != db[l]).all()


@pytest.mark.parametrize("rows,inputs,outputs,dtype", [(100000, 256, 512, 2), (1000000, 256, 256, 3), (60000, 200, 192, 2)])
def test_gradients_take_the_card(lib, rows, inputs, outputs, dtype):
    """The rows of one leaf go to about as many blocks as there are CUs, also where large tiles
    make few of the leaf's map: working memory holds the parts' sums."""
    need = C.c_size_t(0)
    m = maps(rows=rows, leaves=1, inputs=inputs, outputs=outputs, dtype=dtype)
    assert lib.lgbm_hip_leaf_product_workspace(C.byref(m), C.c_int32(2), C.byref(need)) == 0
    tiles = -(-inputs // 256) * -(-outputs // 256)
    # two slots for each stretch of the order that is as long as a part, of at least 512 rows
    parts = need.value // (4 * outputs * (inputs + 1)) // 2
    assert parts * tiles >= min(200, rows // 512 * tiles)


@pytest.mark.parametrize("dtype", [0, 2])
def test_parts_are_few(lib, dtype):
    """The parts' working memory goes by the rows, not by the leaves, most of which are a part
    of their own."""
    need, other = C.c_size_t(0), C.c_size_t(0)
    for leaves, into in ((1, need), (5000, other)):
        m = maps(rows=100000, leaves=leaves, inputs=65, outputs=70, dtype=dtype)
        assert lib.lgbm_hip_leaf_product_workspace(C.byref(m), C.c_int32(2), C.byref(into)) == 0
    assert 0 < need.value == other.value <= 2 * (100000 // 512 + 1) * 4 * 70 * 66


@pytest.mark.parametrize("what,cols", [(0, 10), (1, 100)])
def test_planes_are_bounded(lib, what, cols):
    """However many trees there are: planes of 4 GiB, one plane at least, and a float64 one that
    carries the sums."""
    need = C.c_size_t(0)
    for rows, trees in ((1000000, 500), (1000000, 5000), (200000000, 3), (10500000, 100), (7, 65535)):
        m = maps(rows=rows, trees=trees, inputs=100, outputs=10)
        assert lib.lgbm_hip_leaf_product_workspace(C.byref(m), C.c_int32(what), C.byref(need)) == 0
        plane = rows * cols * 4
        assert plane <= need.value <= max(plane, 2 ** 32) + 2 * plane + 16
        if trees * plane <= 2 ** 32:
            assert trees * plane <= need.value <= trees * plane + 16


def test_python_refuses_what_autograd_would_lose():
    """A tensor that requires gradients is refused while torch records; without recording, and
    detached, the call goes on to its next check."""
    import torch
    be = Plain()
    z = torch.zeros
    i32 = torch.int32
    g = LeafGroups(z((1, 6), dtype=i32), z((1, 4), dtype=i32), z((1, 4), dtype=i32))
    calls = [
        (lambda x, w, dy: be.leaf_product(x, w, g), "x"), (lambda x, w, dy: be.leaf_product(x, w, g), "weight"),
        (lambda x, w, dy: be.leaf_product(x, w, g, bias=dy[:4]), "bias"),
        (lambda x, w, dy: be.leaf_product(x, w, g, out=dy), "out"),
        (lambda x, w, dy: be.leaf_product_dx(dy, w, g), "dy"), (lambda x, w, dy: be.leaf_product_dw(dy, x, g), "x"),
        (lambda x, w, dy: be.dropout(x, 0.5, 1), "x"), (lambda x, w, dy: be.dropout(x[:, 0], 0.5, 1), "x"),
        (lambda x, w, dy: be.adjust_scores(x), "scores"), (lambda x, w, dy: be.adjust_scores(x, bias=w[0, 0]), "bias")]
    holder = {"x": "x", "weight": "w", "bias": None, "out": "dy", "dy": "dy", "scores": "x"}
    for i, (call, name) in enumerate(calls):
        t = {"x": z((6, 5)), "w": z((4, 3, 5)), "dy": z((6, 3))}
        t[holder[name] or ("dy" if i == 2 else "w")].requires_grad_()
        with pytest.raises(ValueError, match=f"{name} requires gradients"):
            call(**t)
        with torch.no_grad(), pytest.raises(ValueError, match="is on cpu"):
            call(**t)
        with pytest.raises(ValueError, match="is on cpu"):
            call(**{k: v.detach() for k, v in t.items()})


@pytest.mark.parametrize("out,ldx,ldo,text", [
    (A + 32, 16, 16, "null context"), (A - 32, 16, 16, "null context"), (A + 64 * 7 + 32, 16, 16, "null context"),
    (A + 28, 16, 16, "in place"), (A + 36, 16, 16, "in place"), (A - 28, 16, 16, "in place"),
    (A - 36, 16, 16, "in place"), (A + 64, 16, 16, "in place"), (A - 64 * 3, 16, 16, "in place"),
    (A + 32, 16, 24, "in place"), (A + 32, 8, 8, "in place"), (A + 3200, 8, 8, "null context")])
def test_tables_side_by_side(lib, out, ldx, ldo, text):
    """Eight columns of a table may go to eight others: rows of one stride overlap where their
    columns do, other matrices where their memory does."""
    refused(lib, dropout(lib, out=out, ldx=ldx, ldo=ldo), INVALID, text)


def test_products_side_by_side(lib):
    """x or dy, and y or dx, as columns of one table."""
    it = calls(lib, maps(), p1=D, ld1=20, out=D + 5 * 4, ldo=20)
    refused(lib, next(it), INVALID, "null context")
    it = calls(lib, maps(), p1=D, ld1=20, out=D + 4 * 4, ldo=20)
    refused(lib, next(it), INVALID, "overlaps")
    rc = lib.lgbm_hip_adjust_scores(None, C.byref(score_args(ldx=80, ldo=80, out=A + 160)), C.c_void_p(W),
                                    C.c_size_t(1 << 40), None)
    refused(lib, rc, INVALID, "null context")
    rc = lib.lgbm_hip_adjust_scores(None, C.byref(score_args(ldx=80, ldo=80, out=A + 164)), C.c_void_p(W),
                                    C.c_size_t(1 << 40), None)
    refused(lib, rc, INVALID, "in place")


@pytest.mark.parametrize("change", [dict(repetition=1e-46), dict(repetition=1e39), dict(frequency=-1e39), dict(presence=1e300)])
@pytest.mark.parametrize("dtype", [0, 1, 2, 3])
def test_penalties_in_the_type_of_the_arithmetic(lib, change, dtype):
    """What is 0 or infinite as a float32 is refused where the arithmetic is float32."""
    rc = lib.lgbm_hip_adjust_scores(None, C.byref(score_args(**HISTORY, dtype=dtype, **change)), C.c_void_p(W),
                                    C.c_size_t(1 << 40), None)
    refused(lib, rc, INVALID, "null context" if dtype == 1 else "not positive, or a penalty not finite")


def test_python_refuses_no_masks():
    """A table of no masks has no memory, which the C entry would take as no table."""
    import torch
    be, x = Plain(), torch.zeros((6, 5))
    with pytest.raises(ValueError, match="without masks"):
        be.adjust_scores(x, mask=torch.zeros((0, 1), dtype=torch.int32))
    with pytest.raises(ValueError, match="is on cpu"):
        be.adjust_scores(x, mask=torch.zeros((0, 1), dtype=torch.int32), mask_rows=torch.zeros(6, dtype=torch.int32))
    with pytest.raises(ValueError, match="is on cpu"):
        be.adjust_scores(x[:0], mask=torch.zeros((0, 1), dtype=torch.int32))
