"""Log probabilities and their gradient where the arithmetic is at its ends: far temperatures and derivatives."""
import numpy as np
import pytest

from tests import class_scores_oracle as O
from tests import student_oracle as S
from tests.test_gpu_class_logprobs import close, given_of, masks, reach, run_grad

pytestmark = pytest.mark.gpu


def check_far_gradient(x, given, g, h, t, kind, order, allowed, tag):
    """As the gradient of ordinary temperatures (test_gpu_class_logprobs), with what passes the type's range infinite; a
    weight e^d below 2^-125 may count as 0, and its part of the gradient is that times the row's factor."""
    rows, n = x.shape
    free = None if allowed is None else np.broadcast_to(allowed, (rows, n))
    v = O.round_to(x, kind)
    _, m, log_z, far = S.row_stats(v, t, free)
    with np.errstate(over="ignore"):
        st = np.stack([m, log_z, far], 1).astype(np.float32)
    got = run_grad(x, given, g, h, st, t, kind, order, allowed)
    g, h = g.astype(np.float32), h.astype(np.float32)
    want, size = S.logprob_gradients(v, given, g, h, t, free)
    ok = (given >= 0) & (given < n)
    factor = (np.abs(np.where(ok, g, 0)).astype(np.float64).sum(1) + np.abs(h) * (200.0 + far)) / t
    # (of a row with NaN: its allowed classes have NaN and are compared as such, the others 0)
    tol = np.nan_to_num(size) * (reach(S.masked(v, free), t) + 24 + np.where(np.isfinite(log_z), log_z, 0)[:, None]) * 2.0 ** -23
    tol += np.nan_to_num(np.abs(want)) * (O.half_step(kind) + 2.0 ** -24) + O.smallest(kind) + 2.0 ** -125 * np.nan_to_num(factor)[:, None]
    largest = {"f32": 2.0 ** 128, "f16": 65520.0, "bf16": 2.0 ** 128 * (1 - 2.0 ** -9)}[kind]
    # infinite or not by a rounding: not compared.  Few, but in f16, which ends at a size that differences of numbers of 1 / t
    # are off by
    near = np.abs(np.abs(want) - largest) <= tol + 2.0 ** -9 * largest
    assert kind == "f16" or near.sum() <= 2 + 0.01 * near.size, tag
    want, got = np.where(near, 0, want), np.where(near, 0, got)
    want = np.where(np.abs(want) >= largest, np.copysign(np.inf, want), want)
    close(got, want, tol, tag)
    return got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t", [1e-38, 1e-37, 4e-37, 1e-36, 1e-33, 1e-20, 1e-3, 1e3, 1e20, 1e36])
def test_gradients_at_far_temperatures(t, kind):
    """Scores of the temperature's size keep their weights; of others the largest alone, or all alike.  Derivatives of 1
    and far from it: a class without a probability has gradient 0, others what the formula says, also where 1 / t times
    the derivatives alone passes f32."""
    g = np.random.default_rng(8)
    # (thread a row; group of lanes; lists longer than a group takes; a wave a segment)
    for rows, n, m in ((5, 9, 2), (70, 3, 1), (4, 700, 2), (6, 60, 3), (4, 700, 20), (3, 9000, 2)):
        for size in (1.0, min(max(t, 1e-37), 1e36)):
            x = (O.scores(g, rows, n, "normal").astype(np.float64) * size)
            x = np.where(np.abs(x) < 2.0 ** -126, 0, x).astype(np.float32)
            given, up, h = given_of(g, rows, n, m), g.standard_normal((rows, m)), g.standard_normal(rows)
            for s in (1.0, 1e-6, 50.0):
                for order, name, allowed in (("rows", *masks(g, rows, n)[0]), ("classes", *masks(g, rows, n)[2])):
                    check_far_gradient(x, given, up * s, h * s, t, kind, order, allowed, (t, kind, n, size, s, order))


def test_a_row_sure_of_its_class_has_no_gradient_elsewhere():
    """Temperatures at which the entropy's derivative times 1 / t is near the largest f32: gradient 0 of every class
    without a probability."""
    for t in (4e-37, 1e-37, 1e-38):
        for rows, n in ((3, 10), (3, 700), (2, 5000)):
            x = np.zeros((rows, n), np.float32)
            x[:, 1] = 1.0
            x[:, 3] = -np.inf
            given = np.full((rows, 1), 1)
            st = np.tile(np.array([[1.0, 0.0, 0.0]]), (rows, 1))
            got = run_grad(x, given, np.ones((rows, 1)), np.ones(rows), st, t, "f32", "rows")
            assert (got == 0).all(), (t, n)


@pytest.mark.parametrize("scale", [1e30, 3e38])
def test_gradients_of_far_derivatives(scale):
    """Derivatives up to the largest f32 at a temperature of 1."""
    g = np.random.default_rng(9)
    for rows, n, m in ((5, 9, 2), (4, 700, 2), (4, 700, 20), (3, 9000, 2)):
        x, given = O.scores(g, rows, n, "normal"), given_of(g, rows, n, m)
        up, h = g.uniform(-1, 1, (rows, m)) * scale, g.uniform(-1, 1, rows) * scale
        check_far_gradient(x, given, up, h, 1.0, "f32", "rows", None, (scale, n))
