"""Log probabilities of given classes, entropy, alternatives (cbh_class_logprobs) and their gradient
(cbh_logprob_gradients) on device buffers, against plain implementations in 64 bits.

Bars, counted from the arithmetic: log Z as the log-sum-exp of the top classes (f32 exponentials of d, an error of
|d| 2^-23 and a rounding each, added up in f32 by the thread, n / 64 sums at most); a log probability is f64 beside it and rounded
once; E is a sum of products of the same exponentials with d, over Z, all of one sign: its relative error is that of the
products (one more rounding, and d's own) and of Z.  A gradient's p is 2^y / Z of f32 y, with log Z as the stats
hold it; the factor beside it and its sums are a few roundings more; an entry's own is f64.  A result is rounded once
to its type.  Indexes are exact.
"""
import numpy as np
import pytest

import catboost_rs_amd as cb
from tests import class_scores_oracle as O
from tests import student_oracle as S
from tests.device_buffers import Buffers
from tests.test_gpu_class_scores import TYPE, laid, put, reach, workspace

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1, 1), (3, 2, 2, 1), (700, 10, 3, 3), (70, 32, 1, 32), (9, 33, 2, 5), (5, 64, 64, 64), (4, 1000, 1, 5),
          (3, 2048, 7, 256), (2, 2049, 1, 300), (2, 5000, 3, 1024), (5, 50021, 4, 20), (2, 8193, 1, 0), (1, 70001, 1, 64),
          (3, 140003, 2, 257), (600, 4099, 1, 9), (1, 40000, 1024, 0), (300, 20, 40, 0),
          (333, 70, 1, 14), (65, 129, 8, 0), (70, 256, 9, 64), (31, 257, 2, 65), (1001, 40, 1, 0), (9, 700, 1, 0), (6, 2048, 1, 64),
          (2, 40000, 1, 200), (2, 9000, 1, 256), (2100, 2500, 1, 130), (300, 40, 3, 40), (259, 64, 2, 7), (70, 17, 1, 0), (70, 33, 9, 0)]


def words(allowed):
    """Bit words of [rows][n] truth values."""
    rows, n = allowed.shape
    b = np.packbits(np.pad(allowed, ((0, 0), (0, -n % 32))), axis=1, bitorder="little")
    return np.ascontiguousarray(b).view(np.uint32)


def mask_args(b, allowed, rows):
    if allowed is None:
        return None, 0
    w = words(allowed)
    return b.put(w, fill=0xFF), 0 if len(w) == 1 and rows != 1 else w.shape[1]


def run(x, given, t, k, kind, order, allowed=None):
    rows, n = x.shape
    L = cb.load()
    m = given.shape[1]
    with Buffers() as b:
        out = [b.out((rows, m), np.float32), b.out(rows, np.float32), b.out((rows, 3), np.float32),
               b.out((rows, k), np.float32), b.out((rows, k), np.int32)]
        ws = workspace(b, L.cbh_class_logprobs_workspace(rows, n, k))
        gp = b.put(given.astype(np.int32))
        cb._check(L.cbh_class_logprobs(*put(b, x, kind, order), gp, m, t, *mask_args(b, allowed, rows), k, *out, *ws, None))
        if ws[0]:
            b.get(ws[0])
        return [b.get(p) for p in out]


def close(got, want, tol, tag):
    """Equal where not finite, within tol where finite."""
    tol = np.broadcast_to(tol, want.shape)
    fin = np.isfinite(want)
    assert np.array_equal(np.where(fin, 0, got), np.where(fin, 0, want), equal_nan=True), tag
    assert np.isfinite(got[fin]).all(), tag
    over = np.abs(got[fin].astype(np.float64) - want[fin]) - tol[fin]
    assert not over.size or over.max() <= 0, (tag, over.max(), tol[fin][over.argmax()])


def free_rows(allowed, rows, n):
    return None if allowed is None else np.broadcast_to(allowed, (rows, n))


def check(x, given, t, k, kind, order, allowed=None, tag=""):
    rows, n = x.shape
    lp, ent, st, top, index = run(x, given, t, k, kind, order, allowed)
    free = free_rows(allowed, rows, n)
    h = O.round_to(x, kind)
    elp, eent, est, etop, eindex = S.logprobs(h, given, t, k, free)
    assert np.array_equal(index, eindex), tag
    far = reach(S.masked(h, free), t)
    z = (n / 64 + 16 + far) * 2.0 ** -23
    e = np.nan_to_num(est[:, 2]) * 2 * z
    close(lp, elp, z + np.abs(np.where(np.isfinite(elp), elp, 0)) * 2.0 ** -24, (tag, "logprob"))
    close(top, etop, z + np.abs(np.where(np.isfinite(etop), etop, 0)) * 2.0 ** -24, (tag, "top"))
    close(ent, eent, z + e + np.abs(np.nan_to_num(eent)) * 2.0 ** -24, (tag, "entropy"))
    close(st[:, 0], est[:, 0], 0.0, (tag, "largest"))
    close(st[:, 1], est[:, 1], z + np.abs(np.where(np.isfinite(est[:, 1]), est[:, 1], 0)) * 2.0 ** -24, (tag, "log z"))
    close(st[:, 2], est[:, 2], e + np.abs(np.nan_to_num(est[:, 2])) * 2.0 ** -24, (tag, "far"))


def run_grad(x, given, g, h, st, t, kind, order, allowed=None, to=None):
    rows, n = x.shape
    L = cb.load()
    with Buffers() as b:
        block, at, grs, gcs = laid(np.zeros_like(x), kind, to or order)
        out = b.put(np.full(block.shape, 77, block.dtype))
        gp, up, sp = b.put(given.astype(np.int32)), b.put(g.astype(np.float32)), b.put(st.astype(np.float32))
        hp = None if h is None else b.put(h.astype(np.float32))
        cb._check(L.cbh_logprob_gradients(*put(b, x, kind, order), gp, given.shape[1], up, hp, sp, t,
                                          *mask_args(b, allowed, rows), out + at * block.itemsize, grs, gcs, None))
        flat = b.get(out)
        i = at + np.arange(rows)[:, None] * grs + np.arange(n)[None] * gcs
        rest = np.ones(flat.size, bool)
        rest[i.ravel()] = False
        assert (flat.reshape(-1)[rest] == 77).all(), "written between the rows"
        return O.from_bits(flat.reshape(-1)[i], kind)


def check_grad(x, given, g, h, t, kind, order, allowed=None, tag=""):
    rows, n = x.shape
    free = free_rows(allowed, rows, n)
    v = O.round_to(x, kind)
    _, m, log_z, far = S.row_stats(v, t, free)
    got = run_grad(x, given, g, h, np.stack([m, log_z, far], 1), t, kind, order, allowed)
    g, h = g.astype(np.float32), None if h is None else h.astype(np.float32)
    want, size = S.logprob_gradients(v, given, g, h, t, free)
    near = reach(S.masked(v, free), t)
    with np.errstate(invalid="ignore"):
        tol = np.nan_to_num(size) * (near + 24 + np.where(np.isfinite(log_z), log_z, 0)[:, None]) * 2.0 ** -23
        # the sum of an entry's own derivatives is f64, rounded with the rest
        tol += np.abs(np.nan_to_num(want)) * (O.half_step(kind) + 2.0 ** -24) + O.smallest(kind)
    close(got, want, tol, tag)


def given_of(g, rows, n, m):
    given = g.integers(0, n, (rows, m))
    given[g.random((rows, m)) < 0.15] = -1
    given[g.random((rows, m)) < 0.05] = n + 3
    if m > 1:
        given[0, 1] = given[0, 0]   # a class twice
    return given


def masks(g, rows, n):
    one = g.random((1, n)) < 0.6
    each = g.random((rows, n)) < 0.5
    each[-1] = False                # a row that allows nothing
    return (("none", None), ("shared", one), ("rows", each))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,m,k", SHAPES)
def test_shapes(rows, n, m, k, kind):
    g = np.random.default_rng(rows * n + k)
    for order, t in (("rows", 1.0), ("padded", 1.5)) + ((("classes", 0.7), ("reversed", 2.0)) if n <= 9000 and rows * n < 2_000_000 else ()):
        x, given = O.scores(g, rows, n, "normal"), given_of(g, rows, n, m)
        for name, allowed in masks(g, rows, n):
            tag = (order, t, name)
            check(x, given, t, k, kind, order, allowed, tag)
            up = g.standard_normal((rows, m))
            check_grad(x, given, up, None, t, kind, order, allowed, tag)
            check_grad(x, given, up, g.standard_normal(rows), t, kind, order, allowed, tag)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("order", ["rows", "classes", "padded"])
def test_every_number_of_few_classes(order, kind):
    g = np.random.default_rng(11)
    for n in range(1, 72):
        rows = 67
        x, given = O.scores(g, rows, n, "normal"), given_of(g, rows, n, 2)
        for name, allowed in masks(g, rows, n)[::2]:
            for k in (0, min(n, 3), n):
                check(x, given, 1.2, k, kind, order, allowed, (n, k, name))
            up = g.standard_normal((rows, 2))
            check_grad(x, given, up, None if n % 2 else g.standard_normal(rows), 1.2, kind, order, allowed, (n, name))


@pytest.mark.parametrize("values", ["ties", "equal", "rising", "masked", "sharp"])
def test_values(values):
    g = np.random.default_rng(5)
    for rows, n, k in ((40, 20, 7), (4, 500, 300), (3, 9001, 130), (2, 40000, 700), (2, 33000, 40), (3, 3000, 0)):
        for kind in ("f32", "bf16"):
            x, given = O.scores(g, rows, n, values), given_of(g, rows, n, 3)
            for name, allowed in masks(g, rows, n):
                check(x, given, 1.0, k, kind, "rows", allowed, (rows, n, k, kind, name))
                check_grad(x, given, g.standard_normal((rows, 3)), g.standard_normal(rows), 1.0, kind, "rows", allowed,
                           (rows, n, kind, name))


def test_nan_and_infinities():
    g = np.random.default_rng(6)
    for rows, n, k in ((6, 20, 9), (6, 500, 30), (6, 3000, 20), (6, 3000, 700), (6, 70000, 100)):
        x, given = O.scores(g, rows, n, "normal"), given_of(g, rows, n, 3)
        given[:, 2] = 5
        x[0, n // 2] = np.nan
        x[1, [3, n - 1]] = np.nan, -np.nan
        x[2, 5] = np.inf
        x[3, g.integers(0, n, 4)] = np.inf
        x[4] = np.where(g.random(n) < 0.5, 0.0, -0.0)
        x[5] = np.nan
        check(x, given, 1.0, k, "f32", "rows", None, (rows, n, k))
        up, h = g.standard_normal((rows, 3)), g.standard_normal(rows)
        check_grad(x, given, up, h, 1.0, "f32", "rows", None, (rows, n))
        # where they are not allowed, they have no part
        free = np.isfinite(x)
        check(x, given, 1.0, k, "f32", "rows", free, (rows, n, k, "masked"))
        check_grad(x, given, up, h, 1.0, "f32", "rows", free, (rows, n, "masked"))


def test_rows_without_a_derivative_are_not_read():
    """Rows whose derivatives are 0 have gradient 0 whatever they and their stats hold; so has a row of no entry."""
    g = np.random.default_rng(7)
    for rows, n in ((5, 10), (5, 300), (4, 20000)):
        x, given = O.scores(g, rows, n, "normal"), given_of(g, rows, n, 2)
        up = g.standard_normal((rows, 2))
        x[1], up[1] = np.nan, 0
        given[2] = -1
        for order in ("rows", "classes"):
            check_grad(x, given, up, None, 1.0, "f32", order, None, (rows, n, order))
            check_grad(x, given, up, np.where(np.arange(rows) == 3, 0.5, 0.0), 1.0, "f32", order, None, (rows, n, order))


@pytest.mark.parametrize("rows,n", [(70, 10), (70, 40), (9, 700), (5, 5003)])
def test_a_gradient_laid_otherwise_than_the_scores(rows, n):
    g = np.random.default_rng(12)
    x, given = O.scores(g, rows, n, "normal"), given_of(g, rows, n, 2)
    up, h = g.standard_normal((rows, 2)), g.standard_normal(rows)
    _, *st = S.row_stats(x, 1.0)
    st = np.stack(st, 1)
    want = run_grad(x, given, up, h, st, 1.0, "f32", "rows")
    for order, to in (("rows", "classes"), ("classes", "rows"), ("padded", "reversed"), ("reversed", "padded"), ("classes", "padded")):
        got = run_grad(x, given, up, h, st, 1.0, "f32", order, to=to)
        # (the ways differ in where a class with entries is rounded, not in what it is)
        assert np.allclose(got, want, rtol=2.0 ** -19, atol=2.0 ** -21), (order, to)


@pytest.mark.parametrize("t", [1e-38, 1e-20, 1e-3, 1e3, 1e20, 1e36])
def test_far_temperatures(t):
    """Scores of the temperature's size keep their weights; others are the largest alone, or all alike."""
    g = np.random.default_rng(8)
    for rows, n, k in ((5, 9, 3), (4, 700, 5), (3, 9000, 6)):
        for size in (1.0, min(max(t, 1e-37), 1e36)):
            x = (O.scores(g, rows, n, "normal").astype(np.float64) * size).astype(np.float32)
            x = np.where(np.abs(x) < 2.0 ** -126, 0, x).astype(np.float32)
            given = given_of(g, rows, n, 2)
            lp, ent, st, top, index = run(x, given, t, k, "f32", "rows")
            elp, eent, est, etop, eindex = S.logprobs(x, given, t, k)
            assert np.array_equal(index, eindex)
            z = (n / 64 + 16 + 110) * 2.0 ** -23
            with np.errstate(over="ignore"):
                for a, b in ((lp, elp), (top, etop)):
                    b = b.astype(np.float32).astype(np.float64)   # (beyond f32: infinite)
                    close(a, b, z + np.abs(np.where(np.isfinite(b), b, 0)) * 2.0 ** -23, (t, n))
            close(ent, eent, z + 4 * z * eent, (t, n))


def test_one_row_of_many_classes():
    """The largest rows: 2^24 classes."""
    g = np.random.default_rng(9)
    n = 1 << 24
    x = g.standard_normal((1, n)).astype(np.float32)
    given = np.array([[0, n - 1, n // 2]])
    check(x, given, 1.0, 5, "bf16", "rows", None)
    check_grad(x, given, np.array([[1.0, -2.0, 0.5]]), np.array([0.3]), 1.0, "bf16", "rows", None)


def test_the_gradient_is_that_of_the_forward_pass():
    """Differences of the device's own forward pass, in directions along which it changes by more than its rounding."""
    g = np.random.default_rng(10)
    rows, n, t = 4, 300, 1.3
    x, given = O.scores(g, rows, n, "normal"), given_of(g, rows, n, 3)
    up, h = g.standard_normal((rows, 3)), g.standard_normal(rows)

    def value(x):
        lp, ent, *_ = run(x.astype(np.float32), given, t, 0, "f32", "rows")
        return (lp.astype(np.float64) * up).sum(1) + ent.astype(np.float64) * h

    st = run(x, given, t, 0, "f32", "rows")[2]
    grad = run_grad(x, given, up, h, st, t, "f32", "rows").astype(np.float64)
    d = np.sign(grad).astype(np.float32) * np.float32(2.0 ** -9)
    step = ((x + d).astype(np.float64) - (x - d)) / 2
    # the difference's own error: the third derivatives, at most 8 (|up| + 2 |h|) |d|^3 n p for a move that all classes share,
    # and two evaluations to (n / 64 + 20 + reach) 2^-23 (|up| + |h| entropy)
    scale = np.abs(up).sum(1) + 2 * np.abs(h) * 6
    tol = scale * (8 * 2.0 ** -18 * 2.0 ** -9 / t ** 3 + 2 * (n / 64 + 20 + reach(x, t)) * 2.0 ** -23)
    assert (np.abs((value(x + d) - value(x - d)) / 2 - (grad * step).sum(1)) <= tol).all()
