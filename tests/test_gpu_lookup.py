"""Looked-up rows of a table (cbh_lookup_rows) and the table's gradient (cbh_lookup_gradients) on device
buffers, against plain implementations in 64 bits.

Bars: a sum of m values in f32 is off by at most m 2^-24 of the sum of their sizes whatever its order, the product with the scale by a
rounding (the scale's own another), and the result by half a step of its type.  Whatever order a gradient's places
are added in, two runs give the same bits.
"""
import numpy as np
import pytest

import catboost_rs_amd as cb
from tests import class_scores_oracle as O
from tests import student_oracle as S
from tests.device_buffers import Buffers
from tests.test_gpu_class_scores import TYPE, laid, put, workspace

pytestmark = pytest.mark.gpu

# rows, list, entries, dim
SHAPES = [(1, 1, 1, 1), (3, 1, 5, 4), (70, 1, 10, 33), (1000, 1, 50, 8), (5, 7, 3, 130), (300, 40, 1280, 10), (4097, 1, 2047, 5),
          (4096, 2, 2048, 12), (1, 300, 20, 64), (20000, 1, 9, 3), (513, 3, 100003, 7), (60, 5, 300, 1000), (17, 1, 5000, 257),
          (2, 1, 7, 4099), (16384, 1, 40, 16), (16385, 1, 70000, 16), (70001, 5, 131, 6),
          (8192, 1, 600, 9), (8193, 1, 600, 9), (32769, 1, 5000, 2), (131073, 1, 3000, 8), (200000, 3, 70000, 1), (9000, 1, 5000000, 2),
          (2500, 41, 300, 70), (700, 33, 5, 3), (5000, 100, 1500, 19), (1500, 9, 40, 200),
          (512, 1, 70000, 300), (513, 1, 900, 30), (100, 5, 1500, 9), (255, 2, 3, 700),
          (16500, 33, 700, 70), (150001, 8, 60, 16), (21000, 13, 2100, 100)]


def indices(g, rows, many, entries, how):
    if how == "one":          # all places the same entry, but a few
        index = np.full((rows, many), entries // 2)
        index[g.random((rows, many)) < 0.01] = 0
    elif how == "uneven":
        index = np.floor((entries + 1.0) ** g.random((rows, many))).astype(np.int64) - 1
    else:
        index = g.integers(0, entries, (rows, many))
    index[g.random((rows, many)) < 0.05] = -1
    index[g.random((rows, many)) < 0.02] = entries
    if rows > 2:
        index[1] = -2147483648   # a row without an entry
    return index.astype(np.int32)


def run_lookup(table, index, scale, kind, order):
    L = cb.load()
    rows, many = index.shape
    with Buffers() as b:
        out = b.put(np.full((rows, table.shape[1]), 77, np.float32 if kind == "f32" else np.float16 if kind == "f16" else np.uint16))
        p, t, entries, dim, rs, cs = put(b, table, kind, order)
        cb._check(L.cbh_lookup_rows(p, t, entries, dim, rs, cs, b.put(index), rows, many, scale, out, None))
        return O.from_bits(b.get(out), kind)


def run_gradient(grad, index, entries, scale, kind, order, out_kind, strides=None):
    L = cb.load()
    (rows, many), dim = index.shape, grad.shape[1]
    with Buffers() as b:
        out = b.put(np.full((entries, dim), 77, np.float32 if out_kind == "f32" else np.float16 if out_kind == "f16" else np.uint16))
        p, t, _, _, rs, cs = put(b, grad, kind, order)
        rs, cs = strides or (rs, cs)
        ws = workspace(b, L.cbh_lookup_gradients_workspace(rows, many, entries, dim))
        cb._check(L.cbh_lookup_gradients(p, t, rows, dim, rs, cs, b.put(index), many, entries, scale, out, TYPE[out_kind], *ws, None))
        if ws[0]:
            b.get(ws[0])
        return O.from_bits(b.get(out), out_kind)


def bar(want, size, terms, kind):
    return size * (terms + 2) * 2.0 ** -24 + np.abs(want) * (O.half_step(kind) + 2.0 ** -24) + O.smallest(kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,many,entries,dim", SHAPES)
def test_lookup_shapes(rows, many, entries, dim, kind):
    g = np.random.default_rng(rows + dim)
    for order, scale in (("rows", 1.0), ("padded", 0.1), ("classes", -3.0), ("reversed", 16.0)):
        table, index = O.scores(g, entries, dim, "normal"), indices(g, rows, many, entries, "even")
        got = run_lookup(table, index, scale, kind, order)
        want, size = S.lookup(O.round_to(table, kind), index, scale)
        assert (np.abs(got - want) <= bar(want, size, many, kind)).all(), (order, scale)
        if many == 1 and scale == 1.0:
            assert np.array_equal(got, want)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,many,entries,dim", SHAPES)
def test_gradient_shapes(rows, many, entries, dim, kind):
    g = np.random.default_rng(rows + dim)
    for how, order, scale, out_kind in (("even", "rows", 1.0, "f32"), ("uneven", "padded", 0.1, kind), ("one", "classes", -3.0, "f32"),
                                        ("uneven", "reversed", 16.0, "bf16"), ("one", "rows", 1.0, "f16")):
        grad, index = O.scores(g, rows, dim, "normal") * 0.1, indices(g, rows, many, entries, how)
        got = run_gradient(grad, index, entries, scale, kind, order, out_kind)
        want, size, count = S.table_gradient(O.round_to(grad, kind), index, entries, scale)
        assert (got[count == 0] == 0).all(), how
        with np.errstate(over="ignore"):
            want = np.where(np.abs(want) < 65000, want, np.nan) if out_kind == "f16" else want
        ok = np.isfinite(want)
        over = np.abs(np.where(ok, got - want, 0)) - bar(np.where(ok, want, 0), size, count[:, None], out_kind)
        assert over.max() <= 0, (how, order, over.max())


def test_no_rows_have_no_gradient():
    got = run_gradient(np.zeros((0, 5), np.float32), np.zeros((0, 3), np.int32), 40, 1.0, "f32", "rows", "f32")
    assert (got == 0).all()
    index = np.full((50, 3), -1, np.int32)
    got = run_gradient(np.full((50, 5), np.nan, np.float32), index, 40, 1.0, "f32", "rows", "f32")
    assert (got == 0).all()


def test_a_gradient_of_one_value_for_all():
    """Strides of 0, as of an expanded tensor: an entry's gradient is how often it occurs."""
    g = np.random.default_rng(3)
    index = indices(g, 5000, 3, 70, "uneven")
    got = run_gradient(np.ones((5000, 9), np.float32), index, 70, 1.0, "f32", "rows", "f32", strides=(0, 0))
    ok = (index >= 0) & (index < 70)
    assert np.array_equal(got, np.bincount(index[ok], minlength=70)[:, None].repeat(9, 1))


def test_nan_and_infinity_stay_with_their_entries():
    g = np.random.default_rng(4)
    grad, index = O.scores(g, 400, 6, "normal"), indices(g, 400, 1, 30, "even")
    grad[7], grad[9, 2] = np.nan, np.inf
    index[7], index[9] = 4, 5
    got = run_gradient(grad, index, 30, 1.0, "f32", "rows", "f32")
    assert np.isnan(got[4]).all() and got[5, 2] == np.inf
    fine = np.ones((30, 6), bool)
    fine[4] = fine[5, 2] = False
    assert np.isfinite(got[fine]).all()
    table = O.scores(g, 30, 6, "normal")
    table[3] = np.nan
    got = run_lookup(table, index, 1.0, "f32", "rows")
    assert np.array_equal(np.isnan(got).all(1), index[:, 0] == 3)


@pytest.mark.parametrize("rows,many,entries,dim", [(70001, 1, 300, 40), (3000, 40, 1280, 64), (40000, 1, 200000, 4)])
def test_runs_give_the_same_bits(rows, many, entries, dim):
    g = np.random.default_rng(5)
    grad, index = O.scores(g, rows, dim, "normal"), indices(g, rows, many, entries, "uneven")
    a, b = (run_gradient(grad, index, entries, 1.0, "f32", "rows", "f32") for _ in range(2))
    assert np.array_equal(a, b)
