"""Layers of a forest's leaves, their gradients and the clipping of gradients on the GPU, alone
and together, on streams and in graphs.  The checks are in leaf_layer_checks.py; they run in one
child process, which imports torch first."""
import os
import subprocess
import sys

import pytest

from tests.test_gpu_leaf_ops import Worker

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


class LayerWorker(Worker):
    def __init__(self):
        self.p = subprocess.Popen([sys.executable, "-u", os.path.join(HERE, "leaf_layer_worker.py")],
                                  stdin=subprocess.PIPE, stdout=subprocess.PIPE, text=True)
        self.answer()


@pytest.fixture(scope="module")
def check():
    w = LayerWorker()
    yield w
    w.close()


ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid"]

# rows, inputs, outputs, trees, leaves, leaves' sizes, pad: one of each; around 8, 16, 32, 64, 128
# and 256; few and many rows a leaf; several trees; odd strides and addresses; rows in no leaf
SHAPES = [
    (1, 1, 1, 1, 1, "one", 0), (5, 3, 2, 1, 3, "even", 1), (64, 28, 1, 20, 31, "even", 0),
    (17, 16, 16, 1, 1, "one", 0), (100, 33, 17, 2, 7, "lost", 3), (257, 64, 64, 1, 4, "skew", 8),
    (300, 100, 10, 1, 31, "even", 0), (129, 128, 130, 1, 2, "even", 8), (500, 200, 96, 3, 5, "lost", 0),
    (16, 520, 300, 1, 31, "even", 0), (1, 1000, 260, 2, 1, "one", 0), (64, 1030, 264, 1, 1, "one", 1),
    (1000, 70, 257, 1, 3, "skew", 1), (700, 256, 256, 1, 2, "one", 0), (2000, 13, 3, 5, 63, "skew", 0),
    (40, 2000, 1, 1, 7, "even", 0), (600, 530, 20, 1, 2, "skew", 0), (33, 600, 40, 1, 1, "lost", 1)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_layer(check, shape, dtype, gated):
    i = SHAPES.index(shape)
    rows, inputs, outputs, trees, leaves, sizes, pad = shape
    check("layer", rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves, dtype=dtype,
          shape=sizes, pad=pad, act=ACTS[(i + gated) % 6], gated=gated, bias=i % 4 != 3, residual=i % 3 != 1)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_grads(check, shape, dtype, gated):
    i = SHAPES.index(shape)
    rows, inputs, outputs, trees, leaves, sizes, pad = shape
    check("grads", rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves, dtype=dtype,
          shape=sizes, pad=pad, act=ACTS[(i + 2 * gated) % 6], gated=gated, kept="narrow" if i % 5 == 0 else None)


# every activation by the kernels of few outputs, of few rows and of 64 x 64 tiles (the others: below)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_activations(check, dtype, act, gated):
    for rows, inputs, outputs, leaves in ((90, 40, 6, 2), (12, 600, 50, 3), (200, 72, 80, 2)):
        check("layer", rows=rows, inputs=inputs, outputs=outputs, leaves=leaves, dtype=dtype, act=act, gated=gated)
        check("grads", rows=rows, inputs=inputs, outputs=outputs, leaves=leaves, dtype=dtype, act=act, gated=gated)


# large tiles of 16-bit types: whole and ragged, rows off 16 bytes, several trees
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,inputs,outputs,trees,leaves,dtype,shape,pad", [
    (4000, 256, 1024, 1, 2, "bf16", "skew", 0), (9001, 264, 520, 1, 3, "f16", "lost", 8),
    (3000, 328, 776, 2, 3, "bf16", "even", 0), (5000, 200, 512, 1, 2, "bf16", "one", 1),
    (2600, 1000, 1288, 1, 1, "f16", "lost", 8)])
def test_large(check, rows, inputs, outputs, trees, leaves, dtype, shape, pad, gated):
    args = dict(rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves, dtype=dtype,
                shape=shape, pad=pad, gated=gated)
    check("layer", act="gelu", residual=not gated, **args)
    check("grads", act="silu", **args)


# more large tiles than a round of blocks: whole rounds and what is behind them, of y (or dx, whose
# columns are the inputs), with ends of rows and columns, rows in no leaf, two trees
@pytest.mark.parametrize("rows,inputs,outputs,trees,leaves,dtype,shape,gated", [
    (5200, 200, 6200, 1, 1, "bf16", "one", False), (5003, 208, 3140, 1, 3, "f16", "lost", True),
    (2600, 200, 6200, 2, 2, "bf16", "lost", False), (2570, 200, 3200, 1, 1, "bf16", "one", True)])
def test_rounds_of_large_tiles(check, rows, inputs, outputs, trees, leaves, dtype, shape, gated):
    check("layer", rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves, dtype=dtype,
          shape=shape, gated=gated, act="gelu_tanh")


@pytest.mark.parametrize("rows,inputs,outputs,trees,leaves,dtype,shape,gated", [
    (5200, 6200, 200, 1, 1, "bf16", "one", False), (2600, 6208, 104, 2, 2, "f16", "lost", True)])
def test_rounds_of_large_tiles_of_dx(check, rows, inputs, outputs, trees, leaves, dtype, shape, gated):
    check("grads", rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves, dtype=dtype,
          shape=shape, gated=gated, act="silu")


@pytest.mark.parametrize("trees", [1, 3])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "sigmoid"])
def test_differences(check, act, gated, trees):
    check("differences", act=act, gated=gated, trees=trees)


def test_extreme_values(check):
    check("extreme")


def test_empty_tables(check):
    check("kernels_of_layers")


def test_linear_layers_are_products(check):
    check("as_products")


@pytest.mark.parametrize("sizes,dtypes,flat", [
    ([1], ["f32"], False), ([7, 0, 1], ["bf16", "f32"], False), ([4096, 4095, 4097], ["f16"], True),
    ([100003, 5, 70000], ["f32", "bf16", "f16"], False), ([13] * 300, ["bf16"], True),
    ([1000, 0] * 128 + [9], ["f32"], True), ([20000003, 3], ["bf16"], True), ([9000001] * 2, ["f32", "f16"], False)])
@pytest.mark.parametrize("factor", [0.25, 1.5])
def test_clip(check, sizes, dtypes, flat, factor):
    check("clip", sizes=sizes, dtypes=dtypes, flat=flat, factor=factor)


@pytest.mark.parametrize("sizes,dtypes,flat", [
    ([40000003, 0, 5], ["f32"], False), ([70000001, 4096, 1], ["bf16"], True), ([35000001] * 2, ["f16", "f32"], False)])
def test_clip_beyond_the_cache(check, sizes, dtypes, flat):
    check("clip", sizes=sizes, dtypes=dtypes, flat=flat, factor=0.25)


def test_clip_special_values(check):
    check("clip_special")


def test_refused(check):
    check("refused")


@pytest.mark.parametrize("dtype,trees", [("f32", 1), ("bf16", 1), ("f16", 2), ("bf16", 3)])
def test_block(check, dtype, trees):
    check("block", dtype=dtype, trees=trees)


def test_offsets_beyond_32_bits(check):
    check("far_offsets")


def test_runs_of_planes(check):
    check("runs_of_planes")


def test_streams(check):
    check("streams")


def test_graph_of_norms(check):
    check("graph_of_norms")


def test_inference_mode(check):
    check("inference")


# by the kernels of few outputs, few rows, tiles of 64 x 64 and of 128 x 128, and large tiles
@pytest.mark.parametrize("rows,inputs,outputs", [
    (1500, 4, 3), (40, 600, 50), (700, 8, 70), (17000, 100, 256), (17000, 200, 600)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gelu_tails(check, dtype, rows, inputs, outputs):
    check("gelu_tails", dtype=dtype, rows=rows, inputs=inputs, outputs=outputs)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_sigmoid_slope_tails(check, dtype):
    check("sigmoid_slope_tails", dtype=dtype)


def test_clip_beyond_float32(check):
    check("clip_beyond_float32")


# the forms of the kernels between those: two groups of rows a leaf of few rows, 17 to 32 outputs of many
# rows, and 128 x 128 tiles of 16-bit types (rows off 16 bytes, or inputs that are no whole ones)
FORMS = [(200, 600, 50, 1, 8, "even", 0), (250, 520, 130, 2, 9, "lost", 1), (700, 60, 24, 1, 3, "skew", 0),
         (900, 100, 32, 3, 4, "lost", 3), (9000, 130, 512, 1, 2, "skew", 1), (4700, 72, 520, 2, 3, "lost", 3)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", FORMS)
def test_forms(check, shape, dtype, gated):
    i = FORMS.index(shape)
    rows, inputs, outputs, trees, leaves, sizes, pad = shape
    args = dict(rows=rows, inputs=inputs, outputs=outputs // 2 if gated and outputs > 500 else outputs, trees=trees,
                leaves=leaves, dtype=dtype, shape=sizes, pad=pad, gated=gated)
    for act in (ACTS[i], ACTS[(i + 3) % 6]):
        check("layer", act=act, residual=i % 3 != 1, bias=i % 4 != 3, **args)
    check("grads", act=ACTS[(i + 2) % 6], kept="narrow" if i % 2 else None, **args)


# large tiles: y, z and the gradients of every activation, alone, beside a residual, and of two trees
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_large_by_activation(check, dtype, act, gated):
    i = ACTS.index(act) + gated
    args = dict(rows=5000, inputs=200, outputs=520 if gated else 1032, dtype=dtype, act=act, gated=gated, pad=i % 2 * 8)
    check("layer", leaves=2, shape="skew", residual=i % 2 == 0, bias=i % 3 != 1, **args)
    check("grads", leaves=2, shape="lost", **args)
    check("layer", trees=2, leaves=3, shape="lost", **dict(args, rows=2500))


# the large cases above whose gradients begin from silu's z: that z, and y
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,inputs,outputs,trees,leaves,dtype,shape,pad", [
    (4000, 256, 1024, 1, 2, "bf16", "skew", 0), (9001, 264, 520, 1, 3, "f16", "lost", 8),
    (3000, 328, 776, 2, 3, "bf16", "even", 0), (2600, 1000, 1288, 1, 1, "f16", "lost", 8)])
def test_large_silu(check, rows, inputs, outputs, trees, leaves, dtype, shape, pad, gated):
    check("layer", rows=rows, inputs=inputs, outputs=outputs, trees=trees, leaves=leaves, dtype=dtype,
          shape=shape, pad=pad, gated=gated, act="silu", residual=not gated)


# as many tiles behind a whole round as go to smaller ones, the next number that does not, and an end of one row
@pytest.mark.parametrize("rows,inputs,outputs,gated", [
    (5120, 200, 4096, False), (5376, 200, 4096, False), (5121, 200, 2040, True), (5120, 208, 2048, True)])
def test_rounds_to_their_limit(check, rows, inputs, outputs, gated):
    check("layer", rows=rows, inputs=inputs, outputs=outputs, dtype="bf16", shape="one", gated=gated, act="silu")


@pytest.mark.parametrize("rows", [5120, 5376])
def test_rounds_of_dx_to_their_limit(check, rows):
    check("grads", rows=rows, inputs=4096, outputs=200, dtype="f16", shape="one", act="gelu")
