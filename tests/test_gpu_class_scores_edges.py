"""The operators on class scores where their arithmetic is at its ends: far temperatures, students that are sure of
their answer, infinities beside NaN, teachers without mass, sums of parts.

Scores, buffers and calls are those of test_gpu_class_scores.py.
"""
import os
import subprocess
import sys

import numpy as np
import pytest

from tests import class_scores_oracle as O
from tests.test_gpu_class_scores import check_sample, check_top, reach, run_distill, run_sample, run_top, teacher

pytestmark = pytest.mark.gpu

FAR = [1e-37, 1e-40, 1e-310, 1e37, 1e300, float("inf")]
HOWS = [dict(), dict(k=5), dict(p=0.7), dict(k=300, p=0.5), dict(p=0.9, min_p=0.2), dict(min_p=2.0)]


def sample_in_units(x, t, k, p, min_p, allowed):
    """The draws' plain form with masses as cbhip.h states them, integers in units of 2^-S, so that sums are exact:
    at a far temperature whole rows weigh the same, and a nucleus ends exactly at a class or at the next."""
    rows, n = x.shape
    S = 46 if n <= 32 else min(51, 62 - int(np.ceil(np.log2(n))))
    x = np.where(allowed, x.astype(np.float64), -np.inf)
    out = []
    with np.errstate(all="ignore"):
        for r in range(rows):
            m = x[r].max()
            if m == -np.inf:
                out.append(dict(empty=True))
                continue
            order = np.argsort(-x[r], kind="stable")
            if not t[r] > 0:
                out.append(dict(empty=False, greedy=True, first=int(order[0])))
                continue
            z = np.where(x[r] == m, 0.0, (x[r] - m) / t[r])
            z = np.where(np.isneginf(x[r]), -np.inf, z)
            units = np.rint(np.exp(z) * 2.0 ** S).astype(np.int64)
            s = units[order]
            stay = np.arange(n) < (k[r] if k[r] > 0 else n)
            mass = np.cumsum(np.where(stay, s, 0))
            if p[r] < 1:
                stay &= mass - np.where(stay, s, 0) < np.ceil(p[r] * float(mass[-1]))
            stay &= ~(s < min_p[r] * 2.0 ** S)
            stay[0] = True
            kept = np.zeros(n, np.int64)
            kept[order] = np.where(stay, s, 0)
            out.append(dict(empty=False, greedy=False, kept=kept, cum=np.cumsum(kept) / 2.0 ** S,
                            logprob=z - np.log(units.sum() / 2.0 ** S)))
    return out


def check_far(x, u, t, k=0, p=1.0, min_p=0.0, allowed=None, tag=""):
    rows, n = x.shape
    index, lp = run_sample(x, u, t, k, p, min_p, allowed)
    f = [np.asarray(v, dt).astype(np.float64) if np.ndim(v) else np.full(rows, float(v))
         for v, dt in ((t, np.float32), (k, np.int32), (p, np.float32), (min_p, np.float32))]
    O.check_sample(index, lp, sample_in_units(x, *f, np.ones((rows, n), bool) if allowed is None else allowed), u, n, tag)


@pytest.mark.parametrize("t", FAR)
@pytest.mark.parametrize("rows,n", [(40, 20), (20, 500), (8, 5003), (6, 70001), (2, 300007)])
def test_sample_far_temperatures(rows, n, t):
    """Towards 0 the largest scores alone are drawn, each as often as another; towards infinity all allowed classes
    are; and scores as small or as large as the temperature keep their weights."""
    g = np.random.default_rng(n)
    size = min(max(t, 1e-37), 1e37)
    for values in ("ties", "normal", "masked", "of its size") if n < 50000 else ("ties", "of its size"):
        x = O.scores(g, rows, n, "normal" if values == "of its size" else values)
        if values == "of its size":
            x = (x.astype(np.float64) * size).astype(np.float32)
        for how in HOWS if n < 50000 else HOWS[:4]:
            check_far(x, g.random(rows), t, tag=(values, how), **how)


@pytest.mark.parametrize("rows,n", [(64, 20), (24, 5003), (24, 70001)])
def test_sample_far_temperatures_of_rows(rows, n):
    g = np.random.default_rng(n + 1)
    for values in ("ties", "masked"):
        check_far(O.scores(g, rows, n, values), g.random(rows), t=g.choice([0.0, 1.0, 1e-37, 1e-40, 1e37, np.inf], rows),
                     k=g.choice([0, 0, 3, 300], rows), p=g.choice([1.0, 0.8, 0.5], rows), min_p=g.choice([0.0, 0.1], rows),
                     allowed=g.random((rows, n)) < 0.7, tag=values)


# ---- students that are sure of their answer --------------------------------------------------

def mass_of(z):
    """The largest of some z (0 if all are -inf) and the sum of exp(z - largest): a log-sum-exp in two parts (next to
    the lowest f32 one number would lose the logarithm)."""
    m = z.max() if z.size and z.max() > -np.inf else 0.0
    return m, np.exp(z - m).sum()


def distill_in_logs(x, u, ix, base, t, w):
    """Loss and gradient by the formulas with every softmax mass as a logarithm, and what the bars count against: a
    row's gradient terms before they are subtracted, and the others' largest distance in temperatures."""
    rows, n = x.shape
    loss, grad, size, far = np.zeros(rows), np.zeros((rows, n)), np.zeros((rows, n)), np.zeros(rows)
    with np.errstate(all="ignore"):
        for r in range(rows):
            z = x[r].astype(np.float64) / t
            ok = (ix[r] >= 0) & (ix[r] < n)
            at, lu = ix[r][ok].astype(int), u[r][ok].astype(np.float64) / t
            free = np.ones(n, bool)
            free[at] = False
            big, total = mass_of(z)
            um, us = mass_of(lu) if base is None else (float(base[r]), 1.0)
            lq = np.where(lu > -np.inf, (lu - um) - np.log(us), -np.inf)
            q = np.exp(lq)
            g = np.exp(z - big) / total * q.sum()
            loss[r] = (q[q > 0] * (lq - (z[at] - big) + np.log(total))[q > 0]).sum()
            rest = max(0.0, 1.0 - q.sum()) if base is not None and free.any() else 0.0
            size[r] = g
            if rest > 0:
                om, others = mass_of(z[free])
                loss[r] += rest * (np.log(rest) - (np.log(others) + (om - big) - np.log(total)))
                g = g + np.exp(z - big) / total * rest
                share = np.where(free & (others > 0), rest * np.exp(np.where(free, z - om, 0.0)) / others, 0.0)
                g, size[r] = g - share, g + share
                near = z[free][z[free] > -np.inf]
                far[r] = min(near.max() - near.min(), 110.0) if near.size else 0.0
            g[at] -= q
            size[r][at] += q
            loss[r] *= w * t * t
            grad[r], size[r] = w * t * g, w * t * size[r]
    return loss, grad, size, far


def check_distill_in_logs(x, u, ix, base, t, w, kind, order, tag):
    rows, n = x.shape
    weight = None if w == 1.0 else np.full(rows, w, np.float32)
    loss, grad = run_distill(x, u, ix, base, t, weight, kind, order)
    el, eg, size, far = distill_in_logs(O.round_to(x, kind), u, ix, base, t, w)
    # a mass is a sum of f32 exponentials of d, |d| <= far: off by 3 |d| 2^-24 (difference, scale, product) and 2^-23
    # each, by the f32 additions of 32 of them and by at most a factor of that kind for every tile; a class's
    # gradient is such an exponential times f64 factors of masses, rounded to f32 three times and to the type
    rel = (32 + 4 + 4 * far) * 2.0 ** -24
    fin = np.isfinite(el)
    assert np.array_equal(np.where(fin, 0, loss), np.where(fin, 0, el), equal_nan=True), (tag, loss, el)
    bar = w * t * t * rel * 3 + np.abs(el) * 2.0 ** -23
    assert (np.abs(loss - el)[fin] <= bar[fin]).all(), (tag, loss, el)
    # (an exponential below the normal range may be 0)
    bar = size * 2 * rel[:, None] + np.abs(eg) * O.half_step(kind) + O.smallest(kind) * max(1.0, w * t) * 2
    off = np.abs(grad - eg)
    at = np.unravel_index(np.nanargmax(off - bar), off.shape)
    assert (off <= bar).all(), (tag, at, grad[at], eg[at])


GAPS = [60.0, 86.0, 88.0, 95.0, 120.0, 700.0, 760.0, 2000.0, 1e4]


def sure(g, rows, n, k, t, gap, how):
    """Students whose listed classes (all of them, or one) lie `gap` temperatures above every other class, and
    teachers that leave a tenth of their mass to the others."""
    x = O.scores(g, rows, n, "normal")
    ix = np.stack([g.permutation(n)[:k] for _ in range(rows)]).astype(np.int32)
    raised = ix if how == "all" else ix[:, :1]
    lift = gap * t + x.max(1, keepdims=True) - np.take_along_axis(x, raised, 1).min(1, keepdims=True)
    np.put_along_axis(x, raised, (np.take_along_axis(x, raised, 1) + lift).astype(np.float32), 1)
    q = g.random((rows, k)) + 0.1
    q = 0.9 * q / q.sum(1, keepdims=True)
    base = g.standard_normal(rows).astype(np.float32)
    return x, (t * (np.log(q) + base[:, None])).astype(np.float32), ix, base


@pytest.mark.parametrize("rows,n,k", [(24, 20, 6), (24, 10, 3), (6, 500, 20), (4, 9001, 40), (3, 40000, 30), (2, 140001, 20)])
def test_distill_sure_students(rows, n, k):
    """However far the others lie below a student's answer, they share what the teacher leaves them."""
    g = np.random.default_rng(n + k)
    for how in ("all", "one"):
        for t, w in ((1.0, 1.0), (0.1, 2.0)):
            for gap in GAPS:
                x, u, ix, base = sure(g, rows, n, k, t, gap, how)
                for kind in ("f32", "bf16"):
                    order = "rows" if kind == "f32" else "padded"
                    check_distill_in_logs(x, u, ix, base, t, w, kind, order, (how, t, gap, kind))


@pytest.mark.parametrize("rows,n,k", [(24, 20, 6), (24, 10, 3), (6, 500, 20), (4, 9001, 40), (3, 40000, 30)])
def test_distill_masked_others(rows, n, k):
    """Others at a mask's finite value: -1e4, or the lowest of the type, some of them -inf; and all of them -inf (the
    loss is infinite)."""
    g = np.random.default_rng(n - k)
    for low in (-1e4, O.LOWEST, -np.inf):
        x, u, ix, base = sure(g, rows, n, k, 1.0, 1.0, "all")
        free = np.ones((rows, n), bool)
        np.put_along_axis(free, ix, False, 1)
        x[free] = low
        if low > -np.inf:
            x[free & (g.random((rows, n)) < 0.3)] = -np.inf
        check_distill_in_logs(x, u, ix, base, 1.0, 1.0, "f32", "rows", low)


@pytest.mark.parametrize("rows,n,k", [(24, 20, 6), (24, 10, 3), (6, 500, 20), (4, 9001, 40), (3, 40000, 30)])
def test_distill_teacher_without_mass(rows, n, k):
    """A teacher's entries of -inf hold no mass, all of a row's among them: without top_lse nothing pulls at the
    student, with one of -inf the others hold everything."""
    g = np.random.default_rng(n * k)
    x = O.scores(g, rows, n, "normal")
    ix = np.stack([g.permutation(n)[:k] for _ in range(rows)]).astype(np.int32)
    u = np.full((rows, k), -np.inf, np.float32)
    u[0, 1:] = 0.5
    for base in (None, np.full(rows, -np.inf, np.float32)):
        if base is not None:
            base[0] = 3.0
        check_distill_in_logs(x, u, ix, base, 1.5, 1.0, "f32", "rows", base is None)


# ---- sums of parts, infinities beside NaN ------------------------------------------------------

def test_top_nan_beside_infinity():
    """A NaN makes a row's log-sum-exp NaN, +inf in the row or not."""
    g = np.random.default_rng(21)
    for rows, n, k in ((5, 20, 9), (5, 3000, 100), (5, 20000, 50), (5, 70000, 100), (5, 70000, 1000)):
        x = O.scores(g, rows, n, "normal")
        x[0, [n // 2, 1]] = np.nan, np.inf
        x[1, [1, n - 1]] = np.nan, np.inf
        x[2, 3] = np.inf
        x[3, n // 3] = np.nan
        x[4, [0, 2]] = -np.inf, np.inf
        for kind in ("f32", "f16", "bf16"):
            v, i, s = run_top(x, k, 1.0, kind, "rows")
            ev, ei, _ = O.top(O.round_to(x, kind), k, 1.0)
            assert np.array_equal(i, ei) and np.array_equal(v.astype(np.float64), ev, equal_nan=True), (n, kind)
            assert np.isnan(s[[0, 1, 3]]).all() and (s[[2, 4]] == np.inf).all(), (n, kind, s)


@pytest.mark.parametrize("t", [1e-38, 1e-37, 1e36])
def test_top_at_the_ends_of_the_temperatures(t):
    """Scores of the temperature's size keep their weights beside each other."""
    g = np.random.default_rng(22)
    for rows, n, k in ((40, 20, 7), (6, 3000, 20), (2, 70000, 20)):
        x = (O.scores(g, rows, n, "normal").astype(np.float64) * t).astype(np.float32)
        check_top(x, k, t, "f32", "rows", (n, t))


def test_torch_tensors_at_their_ends():
    """In a process of its own: torch brings its own copy of the HIP runtime, and one serves a process."""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-u", os.path.join(here, "torch_class_scores_edges.py")], cwd=os.path.dirname(here),
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    print(r.stdout)
    assert r.returncode == 0, r.stdout[-3000:]
    assert r.stdout.rstrip().endswith("all checks passed")


def small_beside_one(n, t):
    """A row of one 0, the 4095 classes beside it (a thread adds up the scores of a tile in f32) -inf and the others
    -30, at the temperature where a unit is a factor of 2: every f32 exponential is a power of two, and the sum is
    1 + 2^-30 (n - 4096) without rounding in any thread."""
    x = np.full((1, n), -30.0, np.float32)
    x[0, :4096] = -np.inf
    x[0, 0] = 0.0
    return x, np.log1p((n - 4096) * 2.0 ** -30)


@pytest.mark.parametrize("n", [70001, 300000])
def test_sums_of_parts_keep_their_bits(n):
    """What is little beside 1 in a part of a row still counts: the log-sum-exp, and the log probability of a drawn
    class, are right to a rounding."""
    t = 1.0 / np.log(2.0)
    x, lse = small_beside_one(n, t)
    _, _, s = run_top(x, 3, t, "f32", "rows")
    assert abs(s[0] - lse) <= lse * 2.0 ** -23, (s[0], lse)
    for k in (5, 1000):
        index, lp = run_sample(x, np.zeros(1), t=t, k=k)
        assert index[0] == 0 and abs(lp[0] + lse) <= lse * 2.0 ** -23, (k, lp[0], lse)
    # the teacher is sure of class 0: the loss is -log p of it
    loss, _ = run_distill(x, np.zeros((1, 1)), np.zeros((1, 1), np.int32), None, t, None, "f32", "rows")
    assert abs(loss[0] - t * t * lse) <= t * t * lse * 2.0 ** -23, (loss[0], t * t * lse)


# ---- routes --------------------------------------------------------------------------------------

def check_tiled(got, want, rows, what):
    """Rows repeat with the period of `want`."""
    for r in range(rows):
        assert np.array_equal(got[r], want[r % len(want)], equal_nan=True), (what, r)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(512, 40000, 20), (512, 40000, 256), (520, 130001, 1000), (2, 35002, 130)])
def test_top_long_rows_by_groups(rows, n, k, kind):
    """Rows of many classes that a workgroup takes whole (512 of them and more), for short and long lists, and parts
    of rows with lists beyond 128."""
    g = np.random.default_rng(n + k)
    few = np.concatenate([O.scores(g, 1, n, v) for v in ("normal", "ties", "rising", "normal")])
    few[3, [5, n // 2]] = np.nan, np.inf
    few = O.round_to(few, kind)
    ev, ei, es = O.top(few, k, 1.5)
    x = few[np.arange(rows) % 4]
    v, i, s = run_top(x, k, 1.5, kind, "rows")
    check_tiled(i, ei.astype(np.int32), rows, "index")
    check_tiled(v, ev.astype(np.float32), rows, "values")
    for r in range(rows):
        if r % 4 == 3:
            assert np.isnan(s[r])
        else:
            assert abs(s[r] - es[r % 4]) <= (n / 64 + 16 + reach(few[:3], 1.5)) * 2.0 ** -23 + abs(es[r % 4]) * 2.0 ** -24, r


@pytest.mark.parametrize("kind,n", [("f32", 70001), ("bf16", 140003)])
@pytest.mark.parametrize("rows,k", [(512, 20), (512, 700), (3, 700)])
def test_distill_wide_rows(rows, k, kind, n):
    """Rows of 256 KB and more: whole (512 rows) and in parts, with lists of one and of two entries a thread."""
    g = np.random.default_rng(n + k)
    few = O.scores(g, 3, n, "normal")
    u, ix, lse = teacher(g, few, k, 1.0)
    at = np.arange(rows) % 3
    for base in (lse, None):
        b = None if base is None else base[at]
        loss, grad = run_distill(few[at], u[at], ix[at], b, 1.0, None, kind, "rows")
        for r in range(3, rows):
            assert loss[r] == loss[r % 3] and np.array_equal(grad[r], grad[r % 3]), r
        el, eg, size, far = distill_in_logs(O.round_to(few, kind), u, ix, base, 1.0, 1.0)
        rel = (n / 512 + 36 + 4 * 110) * 2.0 ** -24
        assert (np.abs(loss[:3] - el) <= 3 * rel + np.abs(el) * 2.0 ** -23).all(), (loss[:3], el)
        bar = size * 2 * rel + np.abs(eg) * O.half_step(kind) + O.smallest(kind) * 2
        assert (np.abs(grad[:3] - eg) <= bar).all()


def test_rows_of_the_most_classes():
    """2^24 classes, the most that are taken."""
    g = np.random.default_rng(24)
    n = 1 << 24
    x = g.standard_normal((1, n)).astype(np.float32)
    v, i, s = run_top(x, 40, 1.0, "f32", "rows")
    by = np.argsort(-x[0], kind="stable")[:40]
    assert np.array_equal(i[0], by) and np.array_equal(v[0], x[0][by])
    # exponentials of d, |d| <= 12 (off by 3 |d| 2^-24 + 2^-23), f32 additions of 32 of them, and a rounding
    assert abs(s[0] - O.log_sum_exp(x.astype(np.float64))[0]) <= (3 * 12 + 2 + 10 + s[0]) * 2.0 ** -24
    for how in (dict(p=0.9), dict(k=50)):
        check_sample(x, g.random(1), tag=how, **how)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(6, 5003), (4, 70001)])
def test_sample_masks_that_bar_the_sampled_classes(rows, n, kind):
    """The bins' range is taken from a lane's first class of every tile: a list of allowed classes without any of
    those (or with one alone) draws as any other."""
    g = np.random.default_rng(n + 2)
    each = 4 if kind == "f32" else 8
    j = np.arange(n)
    for one in (False, True):
        allowed = np.broadcast_to((j % 2048 >= 64 * each) | (j % each != 0) | (one & (j == 2048)), (rows, n))
        for values in ("normal", "ties", "masked"):
            x = O.scores(g, rows, n, values)
            for how in (dict(p=0.9), dict(k=2000), dict(k=n // 3, p=0.5), dict(t=3.0, p=0.99, min_p=0.01)):
                check_sample(x, g.random(rows), allowed=allowed, kind=kind, tag=(one, values, how), **how)
