"""The operators on class scores (cbh_top_classes, cbh_distill_gradients, cbh_sample_classes) on
device buffers, against plain implementations in 64 bits.

Bars, counted from the arithmetic: the log-sum-exp and the probabilities are f32 exponentials of
d = (x - max) / t (an error of |d| 2^-23 and a rounding each) added up in f32 by the thread (n / 64 sums at
most) and in f64 across threads; losses and what belongs to listed classes are f64 from there;
a result is rounded once to its type.  Values, indexes and drawn classes are exact.
"""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import catboost_rs_amd as cb
from tests import class_scores_oracle as O
from tests.device_buffers import Buffers

pytestmark = pytest.mark.gpu

TYPE = {"f32": 0, "f16": 1, "bf16": 2}


def laid(x, kind, order):
    """The memory block of scores in an order, and where they lie in it: block, offset, strides."""
    rows, n = x.shape
    if order == "classes":
        return O.to_bits(np.ascontiguousarray(x.T), kind), 0, 1, rows
    if order == "padded":
        wide = np.full((rows, n + 13), np.nan, np.float32)
        wide[:, 5:5 + n] = x
        return O.to_bits(wide, kind), 5, n + 13, 1
    if order == "reversed":
        return O.to_bits(np.ascontiguousarray(x[::-1, ::-1]), kind), rows * n - 1, -n, -1
    return O.to_bits(x, kind), 0, n, 1


def put(b, x, kind, order):
    block, at, rs, cs = laid(x, kind, order)
    p = b.put(block, fill=0xFF)   # (NaN behind the block)
    return p + at * block.itemsize, TYPE[kind], x.shape[0], x.shape[1], rs, cs


def workspace(b, n):
    return (b.put(np.full(n, 0xEE, np.uint8)), n) if n else (None, 0)


def run_top(x, k, t, kind, order):
    rows, n = x.shape
    L = cb.load()
    with Buffers() as b:
        v, i, s = b.out((rows, k), np.float32), b.out((rows, k), np.int32), b.out(rows, np.float32)
        ws = workspace(b, L.cbh_top_classes_workspace(rows, n, k))
        cb._check(L.cbh_top_classes(*put(b, x, kind, order), k, t, v, i, s, *ws, None))
        if ws[0]:
            b.get(ws[0])
        return b.get(v), b.get(i), b.get(s)


def reach(x, t):
    """Largest |x - max| / t of a score that adds to the sums, for the bars."""
    f = np.where(np.isfinite(x) & (x > O.LOWEST), x, np.nan)
    with np.errstate(all="ignore"):
        d = np.nanmax(np.where(np.isfinite(f), np.nanmax(f, 1, keepdims=True) - f, 0.0)) if np.isfinite(f).any() else 0.0
    return min(float(d) / t, 110.0)


def check_top(x, k, t, kind, order, tag=""):
    v, i, s = run_top(x, k, t, kind, order)
    ev, ei, es = O.top(O.round_to(x, kind), k, t)
    assert np.array_equal(i, ei), tag
    assert np.array_equal(v.astype(np.float64), ev, equal_nan=True), tag
    n = x.shape[1]
    tol = (n / 64 + 16 + reach(x, t)) * 2.0 ** -23
    fin = np.isfinite(es)
    assert np.array_equal(np.where(fin, 0, s), np.where(fin, 0, es), equal_nan=True), tag
    assert (np.abs(s[fin] - es[fin]) <= tol + np.abs(es[fin]) * 2.0 ** -24).all(), (tag, np.abs(s[fin] - es[fin]).max(), tol)


TOP_SHAPES = [(1, 1, 1), (3, 2, 2), (5, 7, 3), (700, 10, 10), (70, 32, 32), (9, 33, 5), (5, 64, 64), (4, 1000, 5),
              (3, 2048, 256), (2, 2049, 300), (2, 5000, 1024), (5, 50021, 20), (2, 8193, 128), (1, 70001, 64), (3, 140003, 257)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,k", TOP_SHAPES)
def test_top_shapes(rows, n, k, kind):
    g = np.random.default_rng(rows * n + k)
    for order, t in (("rows", 1.0), ("padded", 1.5)) + ((("classes", 0.7), ("reversed", 2.0)) if n <= 9000 else ()):
        check_top(O.scores(g, rows, n, "normal"), k, t, kind, order, (order, t))


@pytest.mark.parametrize("values", ["ties", "equal", "rising", "masked", "sharp"])
def test_top_values(values):
    g = np.random.default_rng(5)
    for rows, n, k in ((40, 20, 7), (4, 500, 300), (3, 9001, 130), (2, 40000, 700), (2, 33000, 40)):
        for kind in ("f32", "bf16"):
            check_top(O.scores(g, rows, n, values), k, 1.0, kind, "rows", (rows, n, k, kind))


def test_top_nan_and_infinities():
    g = np.random.default_rng(6)
    for rows, n, k in ((6, 20, 9), (6, 3000, 100), (6, 70000, 100)):
        x = O.scores(g, rows, n, "normal")
        x[0, n // 2] = np.nan
        x[1, [3, n - 1]] = np.nan, -np.nan
        x[2, 5] = np.inf
        x[3, g.integers(0, n, 4)] = np.inf
        x[4] = np.where(g.random(n) < 0.5, 0.0, -0.0)
        x[5] = np.nan
        v, i, s = run_top(x, k, 1.0, "f32", "rows")
        ev, ei, es = O.top(x, k, 1.0)
        assert np.array_equal(i, ei) and np.array_equal(v.astype(np.float64), ev, equal_nan=True), n
        assert np.isnan(s[[0, 1, 5]]).all() and (s[[2, 3]] == np.inf).all() and np.isfinite(s[4]), n


def run_distill(x, u, ix, base, t, w, kind, order, want_loss=True, want_grad=True):
    rows, n = x.shape
    L = cb.load()
    with Buffers() as b:
        loss = b.out(rows, np.float32) if want_loss else None
        dt = np.uint16 if kind == "bf16" else O.to_bits(x[:1, :1], kind).dtype
        gshape = (n, rows) if order == "classes" else (rows, n)
        grad = b.out(gshape, dt) if want_grad else None
        grs, gcs = (1, rows) if order == "classes" else (n, 1)
        ws = workspace(b, L.cbh_distill_gradients_workspace(rows, n))
        opt = [None if a is None else b.put(np.asarray(a, np.float32)) for a in (base, w)]
        args = put(b, x, kind, order)
        cb._check(L.cbh_distill_gradients(*args, b.put(np.asarray(u, np.float32)), b.put(np.asarray(ix, np.int32)),
                                          u.shape[1], opt[0], t, opt[1], loss, grad, grs, gcs, *ws, None))
        got_loss = b.get(loss) if want_loss else None
        if not want_grad:
            return got_loss, None
        gr = O.from_bits(b.get(grad), kind)
        return got_loss, gr.T if order == "classes" else gr


def teacher(g, x, k, t):
    """A teacher near the student: its top k with the log-sum-exp."""
    with np.errstate(invalid="ignore"):
        y = np.where(np.isfinite(x), x, 0) * 0.7 + g.standard_normal(x.shape)
    u, ix, lse = O.top(y.astype(np.float32), k, t)
    return u.astype(np.float32), ix.astype(np.int32), lse.astype(np.float32)


def check_distill(x, u, ix, base, t, w, kind, order, tag=""):
    loss, grad = run_distill(x, u, ix, base, t, w, kind, order)
    x = O.round_to(x, kind)
    el, eg, size = O.distill(x, u, ix, base, t, w)
    n = x.shape[1]
    rel = (n / 64 + 32 + 2 * reach(x, t)) * 2.0 ** -23
    ww = np.ones(x.shape[0]) if w is None else np.abs(w)
    fin = np.isfinite(el)
    assert np.array_equal(np.where(fin, 0, loss), np.where(fin, 0, el), equal_nan=True), tag
    # the loss is a sum of logarithms that are each off by `rel`, and rounded once
    bar = ww * t * t * rel * (2 + (0 if base is None else 1)) + np.abs(el) * 2.0 ** -24
    assert (np.abs(loss - el)[fin] <= bar[fin]).all(), (tag, np.abs(loss - el)[fin].max(), bar.max())
    nan = np.isnan(eg)
    assert np.array_equal(np.isnan(grad), nan), tag
    # an other class of small gradient is a product of f32 terms; H - rest / others is f64 from sums off by `rel`
    h = (ww * t)[:, None] * np.where(nan, 0, np.abs(eg))
    bar = rel * (size + h + (ww * t)[:, None] * prob(x, t) * (1 + rest_share(x, u, ix, base, t))[:, None])
    bar = bar + np.abs(np.where(nan, 0, eg)) * O.half_step(kind) * (1 + 2 ** -10) + O.smallest(kind)
    off = np.abs(np.where(nan, 0, grad) - np.where(nan, 0, eg))
    assert (off <= bar).all(), (tag, (off - bar).max(), np.unravel_index((off - bar).argmax(), off.shape))


def prob(x, t):
    z = x.astype(np.float64) / t
    with np.errstate(all="ignore"):
        p = np.exp(z - O.log_sum_exp(z)[:, None])
    return np.where(np.isfinite(p), p, 0)


def rest_share(x, u, ix, base, t):
    """rest / (sum of the other classes' p), per row."""
    if base is None:
        return np.zeros(x.shape[0])
    p, out = prob(x, t), np.zeros(x.shape[0])
    for r in range(x.shape[0]):
        at = ix[r][(ix[r] >= 0) & (ix[r] < x.shape[1])]
        free = np.ones(x.shape[1], bool)
        free[at] = False
        o = p[r][free].sum()
        out[r] = max(0.0, 1 - np.exp(u[r].astype(float) / t - base[r]).sum()) / o if o > 0 else 0.0
    return out


DISTILL_SHAPES = [(1, 1, 1), (3, 2, 1), (300, 10, 3), (33, 32, 32), (65, 17, 17), (7, 33, 4), (4, 1000, 16), (3, 2049, 256),
                  (2, 9001, 1024), (3, 50021, 20), (1, 65537, 64), (9, 8192, 1), (1, 300007, 30)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,k", DISTILL_SHAPES)
def test_distill_shapes(rows, n, k, kind):
    g = np.random.default_rng(rows + n + k)
    for order, t, rest, weighted in (("rows", 1.0, True, False), ("padded", 2.0, False, True)) + (
            (("classes", 1.5, True, True), ("reversed", 1.0, False, False)) if n <= 9001 else ()):
        x = O.scores(g, rows, n, "normal")
        u, ix, lse = teacher(g, x, k, t)
        w = np.where(g.random(rows) < 0.3, 0, g.random(rows) + 0.5).astype(np.float32) if weighted else None
        check_distill(x, u, ix, lse if rest else None, t, w, kind, order, (order, t, rest, weighted))


@pytest.mark.parametrize("values", ["masked", "sharp", "equal"])
def test_distill_values(values):
    g = np.random.default_rng(8)
    for rows, n, k in ((40, 20, 7), (6, 500, 30), (4, 9001, 130), (3, 40000, 60)):
        x = O.scores(g, rows, n, values)
        for base in (True, False):
            u, ix, lse = teacher(g, x, k, 1.0)
            u[:, -1] = -np.inf if k > 1 else u[:, -1]   # a teacher's entry without mass
            check_distill(x, u, ix, lse if base else None, 1.0, None, "f32", "rows", (rows, n, k, base))


def test_distill_short_lists_and_left_out_rows():
    """Indexes outside the classes are no entries; a row of weight 0 is left out whatever it holds; NaN
    and +inf stay in their row."""
    g = np.random.default_rng(9)
    for rows, n, k in ((12, 20, 6), (8, 700, 40), (6, 20001, 40)):
        x = O.scores(g, rows, n, "normal")
        u, ix, lse = teacher(g, x, k, 1.0)
        ix[0] = -1
        ix[1, k // 2:] = n
        ix[2, ::2] = 2 ** 31 - 1
        ix[3, 1:] = -2 ** 31
        w = np.ones(rows, np.float32)
        w[4] = 0
        x[4] = np.nan
        x[5, 3] = np.nan
        for base in (lse, None):
            check_distill(x, u, ix, base, 1.0, w, "f32", "rows", (rows, n, base is None))
        x[5, 3] = np.inf
        check_distill(x, u, ix, lse, 1.0, w, "f32", "rows", (rows, n, "inf"))


def test_distill_one_output_alone():
    g = np.random.default_rng(10)
    for rows, n, k in ((5, 12, 3), (4, 5000, 8), (2, 70000, 8)):
        x = O.scores(g, rows, n, "normal")
        u, ix, lse = teacher(g, x, k, 1.0)
        loss, grad = run_distill(x, u, ix, lse, 1.0, None, "f32", "rows")
        assert np.array_equal(run_distill(x, u, ix, lse, 1.0, None, "f32", "rows", want_grad=False)[0], loss)
        assert np.array_equal(run_distill(x, u, ix, lse, 1.0, None, "f32", "rows", want_loss=False)[1], grad)


@pytest.mark.parametrize("rows,n,k", [(6, 9, 3), (3, 400, 12), (2, 3000, 40)])
def test_distill_gradient_against_differences(rows, n, k):
    """The gradient against central differences of the loss along random directions.  With h = 2^-5 the
    difference quotient of a loss off by e is off by e / h, and by h^2 / 6 times the third derivative along
    the direction (below 4 / t times its largest entry cubed, for a softmax)."""
    g = np.random.default_rng(11)
    for t, rest in ((1.0, True), (2.0, False)):
        x = O.scores(g, rows, n, "normal")
        u, ix, lse = teacher(g, x, k, t)
        base, h = (lse if rest else None), 2.0 ** -5
        _, grad = run_distill(x, u, ix, base, t, None, "f32", "rows")
        for _ in range(4):
            d = g.choice([-1.0, 1.0], (rows, n)).astype(np.float32)
            up, _ = run_distill((x + h * d).astype(np.float32), u, ix, base, t, None, "f32", "rows")
            dn, _ = run_distill((x - h * d).astype(np.float32), u, ix, base, t, None, "f32", "rows")
            e = (n / 64 + 32 + 2 * reach(x, t)) * 2.0 ** -23 * 3 * t * t + 2.0 ** -24 * np.abs(up)
            want = (grad.astype(np.float64) * d).sum(1)
            step = 2.0 ** -22 * np.abs(x).max() * np.abs(grad).sum(1) / h   # (x + h d is rounded)
            assert (np.abs((up - dn) / (2 * h) - want) <= e / h + h * h / 6 * 8 * max(1, 1 / t) + step).all()


def words_of(allowed):
    rows, n = allowed.shape
    bits = np.zeros((rows, (n + 31) // 32 * 32), np.uint8)
    bits[:, :n] = allowed
    bits[:, n:] = 1   # (bits past the classes mean nothing)
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


def run_sample(x, u, t=1.0, k=0, p=1.0, min_p=0.0, allowed=None, kind="f32", order="rows"):
    rows, n = x.shape
    L = cb.load()

    def both(b, v, dt):
        return (0, b.put(np.asarray(v, dt))) if np.ndim(v) else (v, None)

    with Buffers() as b:
        index, lp = b.out(rows, np.int32), b.out(rows, np.float32)
        ws = workspace(b, L.cbh_sample_classes_workspace(rows, n))
        a = None if allowed is None else b.put(words_of(allowed))
        stride = 0 if allowed is None or allowed.shape[0] != rows else (n + 31) // 32
        args = put(b, x, kind, order)
        cb._check(L.cbh_sample_classes(*args, b.put(np.asarray(u, np.float64)), *both(b, t, np.float32),
                                       *both(b, k, np.int32), *both(b, p, np.float32), *both(b, min_p, np.float32), a, stride,
                                       index, lp, *ws, None))
        if ws[0]:
            b.get(ws[0])
        return b.get(index), b.get(lp)


def check_sample(x, u, t=1.0, k=0, p=1.0, min_p=0.0, allowed=None, kind="f32", order="rows", tag=""):
    rows, n = x.shape
    index, lp = run_sample(x, u, t, k, p, min_p, allowed, kind, order)

    def rowwise(v, dt):   # (settings of a row are f32, one number for all rows f64)
        return np.asarray(v, dt).astype(np.float64) if np.ndim(v) else np.full(rows, float(v))

    mask = None if allowed is None else np.broadcast_to(allowed, (rows, n))
    want = O.sample(O.round_to(x, kind), u, rowwise(t, np.float32), rowwise(k, np.int32), rowwise(p, np.float32),
                    rowwise(min_p, np.float32), mask)
    O.check_sample(index, lp, want, u, n, tag)


SAMPLE_SHAPES = [(1, 1), (40, 2), (400, 10), (60, 32), (60, 33), (30, 64), (20, 65), (12, 1000), (6, 2048), (5, 2049),
                 (4, 20001), (2, 65536), (1, 131072), (3, 200001)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n", SAMPLE_SHAPES)
def test_sample_shapes(rows, n, kind):
    g = np.random.default_rng(rows * 7 + n)
    for how, order in ((dict(), "rows"), (dict(p=0.9), "padded"), (dict(t=0.8, k=50, p=0.95), "rows"),
                       (dict(t=1.3, k=5000), "rows"), (dict(min_p=0.05), "padded"), (dict(t=0.0), "rows"),
                       (dict(p=0.8), "classes"), (dict(k=7, min_p=0.3), "reversed")):
        if n > 9000 and order in ("classes", "reversed"):
            continue
        check_sample(O.scores(g, rows, n, "normal"), g.random(rows), kind=kind, order=order, tag=(how, order), **how)


@pytest.mark.parametrize("rows,n", [(200, 9), (64, 40), (48, 777), (24, 5003), (24, 70001)])
def test_sample_mixed_settings(rows, n):
    """Every row with settings of its own, and lists of allowed classes: a list a row, one list for all rows,
    rows that allow nothing or one class."""
    g = np.random.default_rng(n)
    for masked in ("none", "rows", "one"):
        allowed = None
        if masked != "none":
            allowed = g.random((rows if masked == "rows" else 1, n)) < 0.6
            if masked == "rows":
                allowed[0] = False
                allowed[1] = False
                allowed[1, n // 3] = True
        check_sample(O.scores(g, rows, n, "normal"), g.random(rows), t=g.choice([0.0, 0.6, 1.0, 1.3, -1.0], rows),
                     k=g.choice([0, 1, 2, 20, 300, 5000, n, -3], rows), p=g.choice([1.0, 0.95, 0.5, 0.0, 1.5], rows),
                     min_p=g.choice([0.0, 0.02, 0.3, 1.0, 2.0], rows), allowed=allowed, tag=(masked,))


@pytest.mark.parametrize("values", ["ties", "equal", "rising", "masked", "sharp"])
def test_sample_values(values):
    g = np.random.default_rng(13)
    for rows, n in ((60, 20), (20, 500), (8, 9001), (4, 70000)):
        x = O.scores(g, rows, n, values)
        for how in (dict(), dict(k=n // 3 + 1), dict(p=0.7), dict(k=n // 2 + 1, p=0.5), dict(min_p=0.2), dict(t=0.0),
                    dict(t=30.0, p=0.99), dict(t=1e-3)):
            check_sample(x, g.random(rows), kind="bf16" if n == 500 else "f32", tag=(n, how), **how)


def test_rows_of_more_classes_than_have_groups():
    """Beyond 2^18 classes the draws take top_k from a histogram, and the top classes split every row."""
    g = np.random.default_rng(17)
    rows, n = 2, 600_011
    x = O.scores(g, rows, n, "normal")
    for how in (dict(k=50), dict(k=50, p=0.9), dict(k=3001), dict(p=0.9), dict(), dict(min_p=0.1), dict(t=0.0)):
        check_sample(x, g.random(rows), kind="f16", tag=how, **how)
    check_top(x, 40, 1.0, "f16", "rows")
    u, ix, lse = teacher(g, x, 40, 1.0)
    check_distill(x, u, ix, lse, 1.0, None, "f16", "rows")


def test_sample_ends_of_the_uniform_range():
    g = np.random.default_rng(14)
    for rows, n in ((9, 10), (9, 3000), (9, 40000)):
        x = O.scores(g, rows, n, "normal")
        u = np.array([0.0, np.nextafter(1, 0), 1.0, 2.0, -1.0, np.nan, 0.5, 1e-300, 1 - 1e-9])
        for how in (dict(), dict(p=0.6), dict(k=5)):
            index, lp = run_sample(x, u, **how)
            want = O.sample(x, u, np.ones(rows), np.full(rows, float(how.get("k", 0))), np.full(rows, how.get("p", 1.0)), np.zeros(rows), None)
            for r in range(rows):
                kept = np.flatnonzero(want[r]["kept"] > 0)
                assert index[r] in kept
                if r in (0, 4, 5):
                    assert index[r] == kept[0]
                if r in (1, 2, 3):   # (the last classes may hold less mass than the number can tell)
                    assert want[r]["cum"][index[r]] >= want[r]["cum"][-1] * (1 - 2.0 ** -40)


def test_sample_infinities_and_nan():
    g = np.random.default_rng(15)
    for rows, n in ((6, 12), (6, 900), (6, 30000)):
        x = O.scores(g, rows, n, "normal")
        x[0, 4] = np.nan
        x[1, 7] = np.inf
        x[2, [2, 9]] = np.inf
        x[3] = np.nan
        x[4] = -np.inf
        x[5, 1:] = -np.inf
        u = np.array([0.3, 0.9, 0.9, 0.5, 0.5, 0.99])
        for how in (dict(), dict(p=0.9), dict(k=3, p=0.9), dict(t=0.0)):
            index, lp = run_sample(x, u, **how)
            assert index[1] == 7 and index[2] == (2 if how.get("t") == 0.0 else 9) and index[3] == -1 and index[4] == -1
            assert index[5] == 0 and lp[5] == 0 and lp[3] == -np.inf and lp[4] == -np.inf and index[0] != 4


def test_the_operators_again_and_in_turn_give_the_same():
    """No call depends on what the one before left behind."""
    g = np.random.default_rng(16)
    x = O.scores(g, 3, 70001, "normal")
    u, ix, lse = teacher(g, x, 30, 1.0)
    r = g.random(3)
    first = [run_top(x, 30, 1.0, "f32", "rows"), run_distill(x, u, ix, lse, 1.0, None, "f32", "rows"), run_sample(x, r, p=0.9)]
    for _ in range(3):
        again = [run_top(x, 30, 1.0, "f32", "rows"), run_distill(x, u, ix, lse, 1.0, None, "f32", "rows"), run_sample(x, r, p=0.9)]
        for a, b in zip(first, again):
            for p, q in zip(a, b):
                assert np.array_equal(p, q)


def test_torch_tensors():
    """The functions on torch tensors, in a process of its own: torch brings its own copy of the HIP runtime,
    and one serves a process (tests/torch_class_scores.py names each check as it begins)."""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-u", os.path.join(here, "torch_class_scores.py")], cwd=os.path.dirname(here),
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    print(r.stdout)
    assert r.returncode == 0, r.stdout[-3000:]
    assert r.stdout.rstrip().endswith("all checks passed")
