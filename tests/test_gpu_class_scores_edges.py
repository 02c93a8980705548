"""The operators on class scores where their arithmetic is at its ends: far temperatures, students that are sure of
their answer, infinities beside NaN, teachers without mass, sums of parts.

Scores, buffers and calls are those of test_gpu_class_scores.py.
"""
import numpy as np
import pytest

from tests import class_scores_oracle as O
from tests.test_gpu_class_scores import run_sample

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
