"""The operators around a forest's leaves on the GPU: rows by leaf, leaf products and their
gradients, dropout, class scores, alone and together, on streams and in graphs.  The checks
are in leaf_ops_checks.py; they run in one child process, which imports torch first."""
import json
import os
import select
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


class Worker:
    def __init__(self):
        self.log = []
        self.p = subprocess.Popen([sys.executable, "-u", os.path.join(HERE, "leaf_ops_worker.py")],
                                  stdin=subprocess.PIPE, stdout=subprocess.PIPE, text=True)
        self.answer()

    def answer(self):
        ready, _, _ = select.select([self.p.stdout], [], [], 110)
        line = self.p.stdout.readline() if ready else ""
        if not line:
            self.p.kill()
            raise AssertionError("the worker ended" if ready else "the worker gave no answer")
        return json.loads(line)["error"]

    def __call__(self, name, **args):
        if self.p.poll() is not None:
            pytest.fail("the worker ended in an earlier test")
        self.p.stdin.write(json.dumps({"name": name, "args": args}) + "\n")
        self.p.stdin.flush()
        error = self.answer()
        assert error is None, error

    def close(self):
        self.p.stdin.close()
        try:
            self.p.wait(60)
        except subprocess.TimeoutExpired:
            self.p.kill()


@pytest.fixture(scope="module")
def check():
    w = Worker()
    yield w
    w.close()


@pytest.mark.parametrize("rows,trees,leaves,shape,pad", [
    (1, 1, 1, "even", 0), (1, 3, 4095, "one", 0), (63, 1, 2, "even", 0), (64, 100, 31, "even", 0),
    (65, 7, 31, "lost", 2), (4096, 1, 255, "skew", 0), (4097, 2, 256, "even", 0),
    (20011, 3, 63, "lost", 1), (100003, 1, 1000, "even", 0), (30000, 1, 4095, "skew", 0),
    (50000, 1, 1, "lost", 0), (3000, 300, 15, "even", 0), (300007, 2, 31, "one", 0),
    (1025, 65, 127, "lost", 3), (8192, 2, 100, "lost", 0), (8193, 2, 100, "skew", 0),
    (2200001, 1, 255, "lost", 0), (4200000, 1, 3, "even", 1)])
def test_groups(check, rows, trees, leaves, shape, pad):
    check("groups", rows=rows, trees=trees, leaves=leaves, shape=shape, pad=pad)


def test_groups_of_many_leaves(check):
    check("groups_many")


# one row and one input; outputs and inputs around 16, 32, 64, 128 and 256; rows of a leaf
# from one to hundreds; several trees; odd strides and addresses
SHAPES = [
    (1, 1, 1, 1, 1, "one", 0), (5, 3, 2, 1, 3, "even", 1), (64, 28, 1, 20, 31, "even", 0),
    (17, 16, 16, 1, 1, "one", 0), (100, 33, 17, 2, 7, "lost", 3), (257, 64, 64, 1, 4, "skew", 8),
    (300, 100, 10, 1, 31, "even", 0), (129, 128, 130, 1, 2, "even", 8), (500, 200, 96, 3, 5, "lost", 0),
    (16, 520, 300, 1, 31, "even", 0), (3, 1000, 260, 2, 3, "even", 0), (1000, 70, 257, 1, 3, "skew", 1),
    (700, 256, 256, 1, 2, "one", 0), (2000, 13, 3, 5, 63, "skew", 0), (40, 2000, 1, 1, 7, "even", 0),
    (600, 530, 20, 1, 2, "skew", 0), (170, 140, 7, 2, 3, "lost", 1),
    (333, 65, 8, 1, 1, "lost", 2), (900, 129, 33, 2, 15, "even", 8), (2500, 40, 10, 1, 2, "one", 0)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,inputs,outputs,trees,leaves,shape,pad", SHAPES)
def test_product(check, rows, inputs, outputs, trees, leaves, shape, pad, dtype):
    check("product", rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves,
          shape=shape, pad=pad, dtype=dtype, bias=rows % 2 == 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,inputs,outputs,trees,leaves,shape,pad", SHAPES)
def test_gradients(check, rows, inputs, outputs, trees, leaves, shape, pad, dtype):
    check("grads", rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves,
          shape=shape, pad=pad, dtype=dtype, bias=rows % 2 == 0)


@pytest.mark.parametrize("what", ["product", "grads"])
@pytest.mark.parametrize("rows,inputs,outputs,trees,leaves,dtype", [
    (9000, 24, 6, 1, 2, "f32"), (9000, 30, 9, 1, 2, "bf16"), (5000, 320, 272, 1, 3, "bf16"),
    (5000, 272, 320, 1, 3, "f16"), (1500, 600, 512, 2, 2, "bf16"), (40000, 5, 1, 1, 300, "f32"),
    (9000, 65, 513, 1, 3, "bf16"), (9000, 515, 33, 1, 3, "f16"), (3000, 200, 1100, 5, 2, "f16"),
    (2000, 264, 520, 1, 5, "bf16"), (70000, 600, 20, 1, 2, "bf16"),
    (400, 200, 192, 70, 2, "f16"), (200, 192, 200, 1030, 1, "bf16"), (1000, 2048, 256, 1, 1, "bf16")])
def test_long(check, what, rows, inputs, outputs, trees, leaves, dtype):
    check(what, rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves, dtype=dtype,
          shape="even")


# narrow products over tables beyond the caches
@pytest.mark.parametrize("what", ["product", "grads"])
@pytest.mark.parametrize("rows,inputs,outputs,trees,leaves,shape,pad,dtype", [
    (300000, 61, 10, 1, 3, "lost", 1, "f32"), (270001, 140, 3, 2, 5, "skew", 0, "bf16"),
    (150000, 120, 31, 1, 7, "even", 8, "f32"), (140000, 300, 20, 1, 1, "lost", 0, "f16"),
    (200000, 90, 1, 1, 2, "one", 0, "f32")])
def test_tables(check, what, rows, inputs, outputs, trees, leaves, shape, pad, dtype):
    check(what, rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves, shape=shape,
          pad=pad, dtype=dtype)


@pytest.mark.parametrize("name", ["differences", "odd_tables", "odd_tables_large", "any_order", "empty", "layouts",
                                  "scores_history", "refused", "own_stream", "side_stream",
                                  "captured", "captured_large", "threads", "forest", "learner"])
def test_plain(check, name):
    check(name)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,p,by,pad,seed,offset", [
    (1, 1, 0.5, "element", 0, 1, 0), (7, 9, 0.1, "element", 0, 2 ** 63 + 5, 2 ** 64 - 1),
    (100, 64, 0.3, "element", 0, 7, 1), (33, 31, 0.5, "element", 5, 8, 0),
    (1000, 8, 0.05, "element", 8, 9, 2 ** 32), (3, 10000, 0.9, "element", 1, 10, 0),
    (1000, 2, 0.3, "row", 0, 11, 3), (999, 1, 0.5, "row", 0, 12, 0), (257, 7, 0.2, "row", 1, 13, 0),
    (130, 100, 0.5, "row", 4, 14, 0), (50, 16, 0.0, "element", 0, 15, 0),
    (50, 16, 1.0, "element", 0, 16, 0), (50, 3, 1.0, "row", 0, 17, 0),
    (600, 1024, 0.25, "element", 0, 18, 0), (1001, 4, 0.2, "row", 0, 20, 0),
    (5, 70001, 0.5, "row", 0, 24, 0), (5, 4099, 0.5, "element", 3, 25, 2), (40, 2100, 0.3, "row", 8, 26, 1),
    (300, 5, 0.4, "element", 1, 27, 0), (70001, 3, 0.4, "element", 2, 28, 0), (515, 8, 0.2, "row", 0, 21, 0), (77, 64, 0.2, "row", 0, 22, 5), (9, 1, 0.2, "row", 0, 23, 0), (70000, 2, 0.4, "row", 0, 19, 0)])
def test_dropout(check, rows, cols, p, by, pad, seed, offset, dtype):
    check("dropout", rows=rows, cols=cols, p=p, by=by, pad=pad, seed=seed, offset=offset, dtype=dtype)


def test_dropout_far(check):
    check("dropout_far")


@pytest.mark.parametrize("kind", ["raw", "transformed"])
@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,classes,bias,masks,history,per_row,pad", [
    (1, 1, False, 0, 0, False, 0), (1, 5000, True, 1, 40, False, 0), (300, 2, True, 3, 3, True, 0),
    (1000, 10, True, 5, 0, False, 0), (257, 31, False, 2, 5, False, 1), (65, 64, True, 2, 70, True, 8),
    (33, 255, False, 0, 20, True, 3), (5, 1023, True, 3, 500, True, 0), (4, 4097, False, 2, 6000, False, 1),
    (3, 20001, True, 2, 100, True, 0), (300, 32, True, 2, 9, False, 0), (9, 256, True, 1, 30, False, 1),
    (9, 257, False, 2, 30, True, 0), (7, 512, True, 0, 60, False, 0), (6, 513, True, 2, 60, False, 3),
    (5, 2048, False, 1, 90, True, 0), (5, 2049, True, 2, 90, False, 0), (5, 4096, True, 1, 900, False, 1),
    (150, 8200, True, 3, 50, True, 1), (2, 70000, True, 1, 0, False, 0),
    (90, 70003, False, 2, 30, True, 0), (301, 33000, True, 0, 20, False, 0), (130, 33, True, 0, 1, False, 0)])
def test_scores(check, rows, classes, bias, masks, history, per_row, pad, dtype, kind):
    check("scores", rows=rows, classes=classes, dtype=dtype, kind=kind, bias=bias, masks=masks,
          history=history, per_row=per_row, pad=pad, seed=rows)


def test_scores_mask_for_each_row(check):
    check("scores", rows=37, classes=90, dtype="f32", kind="transformed", masks=37, by_row_masks=True)


@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
def test_scores_edges(check, dtype):
    check("scores_edges", dtype=dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_together(check, dtype):
    check("together", dtype=dtype)


# every form of the maps' gradients, over leaves of one part and of many
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,inputs,outputs,trees,leaves,shape", [
    (300000, 61, 10, 1, 3, "lost"), (270001, 140, 3, 2, 5, "skew"), (200000, 90, 1, 1, 1, "one"),
    (140000, 300, 20, 1, 1, "lost"), (30011, 100, 64, 2, 4, "skew"), (30000, 9, 130, 1, 3, "even"),
    (300, 70, 20, 3, 5, "lost"), (30000, 200, 264, 1, 7, "skew"), (40000, 200, 192, 2, 100, "skew"),
    (12000, 192, 200, 5, 60, "one"), (25000, 264, 520, 1, 3, "lost"), (16384, 192, 192, 1, 2, "one")])
def test_whole_gradients(check, rows, inputs, outputs, trees, leaves, shape, dtype):
    check("whole_dw", rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves, shape=shape,
          dtype=dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("inputs,outputs", [(192, 192), (100, 64), (64, 10), (140, 10), (10, 64)])
def test_long_sums(check, inputs, outputs, dtype):
    check("long_sums", rows=600000, inputs=inputs, outputs=outputs, dtype=dtype)


# enough tiles of 256 x 256 for the CUs, or just too few (19000 rows of two leaves: 75; 18000: 71)
@pytest.mark.parametrize("what", ["product", "grads"])
@pytest.mark.parametrize("rows,inputs,outputs,trees,leaves,shape,pad,dtype", [
    (19000, 200, 192, 1, 2, "even", 8, "bf16"), (18000, 200, 192, 1, 2, "even", 8, "bf16"),
    (9000, 320, 272, 2, 3, "lost", 0, "f16"), (9000, 272, 320, 2, 3, "skew", 16, "bf16"),
    (5000, 1024, 1032, 1, 4, "one", 0, "bf16"), (3000, 1288, 520, 3, 15, "lost", 8, "f16")])
def test_large_tiles(check, what, rows, inputs, outputs, trees, leaves, shape, pad, dtype):
    check(what, rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves, shape=shape,
          pad=pad, dtype=dtype)


@pytest.mark.parametrize("name", ["odd_tables_large_tiles", "captured_tiles"])
def test_large_tiles_plain(check, name):
    check(name)


# runs of 4 and 3 trees, 3 and 3 and 1, 1 and 1 and 1, 16 and 16
@pytest.mark.parametrize("rows,inputs,width,trees,dtype,strided", [
    (2500000, 1, 96, 7, "bf16", False), (3000001, 3, 101, 7, "f32", True), (2900000, 192, 200, 3, "bf16", False),
    (3000000, 1, 17, 32, "f32", False), (2800000, 5, 200, 3, "f16", True)])
def test_trees_in_runs(check, rows, inputs, width, trees, dtype, strided):
    check("tree_runs", rows=rows, inputs=inputs, width=width, trees=trees, dtype=dtype, strided=strided)


@pytest.mark.parametrize("name", ["versions", "earlier_error", "side_by_side", "odd_counts"])
def test_contracts(check, name):
    check(name)


@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [6, 32, 33, 300, 700, 5000, 20000, 100001])
def test_scores_nan(check, classes, dtype):
    check("scores_nan", classes=classes, dtype=dtype)


@pytest.mark.parametrize("inputs,outputs", [(1280, 1280), (2000, 7), (7, 2000), (28, 1), (100, 10)])
def test_short_sums(check, inputs, outputs):
    check("short_sums", inputs=inputs, outputs=outputs)
