"""Refusals of the operators on class scores: typed errors before any device call (no GPU needed), and
the plain implementations that the GPU tests compare with, checked against each other."""
import numpy as np
import pytest

import catboost_rs_amd as cb
from tests import class_scores_oracle as O

P = 4096   # an aligned address that no call here may reach


@pytest.fixture(scope="module")
def lib():
    return cb.load()


def code(rc, lib):
    assert rc != 0
    assert lib.cbh_last_error()
    return rc


def scores(data=P, type=0, rows=4, classes=100, rs=100, cs=1):
    return [data, type, rows, classes, rs, cs]


BAD_SCORES = [(dict(type=3), -4), (dict(type=-1), -4), (dict(classes=0), -2), (dict(classes=(1 << 24) + 1), -2),
              (dict(rows=1 << 31), -2), (dict(data=None), -5), (dict(data=P + 2), -5), (dict(type=1, data=P + 1), -5),
              (dict(rs=1 << 61), -2), (dict(cs=-(1 << 60)), -2)]


@pytest.mark.parametrize("bad,want", BAD_SCORES)
def test_scores_are_checked(lib, bad, want):
    s = scores(**bad)
    assert code(lib.cbh_top_classes(*s, 5, 1.0, P, P, P, None, 0, None), lib) == want
    assert code(lib.cbh_distill_gradients(*s, P, P, 5, None, 1.0, None, P, P, 100, 1, None, 0, None), lib) == want
    assert code(lib.cbh_sample_classes(*s, P, 1.0, None, 0, None, 1.0, None, 0.0, None, None, 0, P, P, None, 0, None), lib) == want


def test_top_arguments_are_checked(lib):
    def top(k=5, t=1.0, v=P, i=P, s=P, ws=None, size=0, **kw):
        return code(lib.cbh_top_classes(*scores(**kw), k, t, v, i, s, ws, size, None), lib)

    assert top(k=0) == -2 and top(k=101) == -2 and top(k=1025, classes=5000) == -2
    assert top(t=0.0) == -2 and top(t=-1.0) == -2 and top(t=float("nan")) == -2 and top(t=float("inf")) == -2
    assert top(v=None) == -5 and top(i=None) == -5 and top(s=None) == -5
    need = lib.cbh_top_classes_workspace(1, 200_000, 5)
    assert need > 0
    assert top(rows=1, classes=200_000) == -1
    assert top(rows=1, classes=200_000, ws=P, size=need - 1) == -1
    assert top(rows=1, classes=200_000, ws=P + 4, size=need) == -1


def test_distill_arguments_are_checked(lib):
    def distill(u=P, ix=P, k=5, t=1.0, loss=P, grad=P, grs=100, gcs=1, ws=None, size=0, **kw):
        return code(lib.cbh_distill_gradients(*scores(**kw), u, ix, k, None, t, None, loss, grad, grs, gcs, ws, size, None), lib)

    assert distill(k=0) == -2 and distill(k=1025) == -2
    assert distill(t=0.0) == -2 and distill(t=float("inf")) == -2 and distill(t=1e-320) == -2
    assert distill(u=None) == -5 and distill(ix=None) == -5
    assert distill(loss=None, grad=None) == -5
    assert distill(grad=P + 1) == -5
    assert distill(grs=1 << 61) == -2
    assert lib.cbh_distill_gradients_workspace(1, 200_000) > 0
    assert distill(rows=1, classes=200_000) == -1
    # a row longer than one workgroup takes, however many rows there are
    assert distill(rows=1000, classes=600_000) == -1


def test_sample_arguments_are_checked(lib):
    def sample(u=P, index=P, allowed=None, stride=0, ws=None, size=0, **kw):
        return code(lib.cbh_sample_classes(*scores(**kw), u, 1.0, None, 0, None, 1.0, None, 0.0, None, allowed, stride, index,
                                           P, ws, size, None), lib)

    assert sample(u=None) == -5 and sample(index=None) == -5
    assert sample(allowed=P, stride=3) == -2 and sample(allowed=P, stride=-3) == -2
    assert sample(allowed=P + 2) == -5
    need = lib.cbh_sample_classes_workspace(1, 200_000)
    assert need > 0 and lib.cbh_sample_classes_workspace(10 ** 9, 2048) == 0
    assert sample(rows=1, classes=200_000) == -1
    assert sample(rows=1, classes=200_000, ws=P, size=need - 1) == -1
    assert sample(rows=1, classes=200_000, ws=P + 4, size=need) == -1
    # the workspace does not grow with the rows beyond a chunk of them
    assert lib.cbh_sample_classes_workspace(2 ** 31 - 1, 200_000) < 128 << 20


def test_no_rows_are_no_work(lib):
    s = scores(rows=0, data=None)
    assert lib.cbh_top_classes(*s, 5, 1.0, None, None, None, None, 0, None) == 0
    assert lib.cbh_distill_gradients(*s, None, None, 5, None, 1.0, None, None, None, 0, 0, None, 0, None) == 0
    assert lib.cbh_sample_classes(*s, None, 1.0, None, 0, None, 1.0, None, 0.0, None, None, 0, None, None, None, 0, None) == 0


def test_the_functions_refuse_what_is_no_gpu_tensor():
    torch = pytest.importorskip("torch")
    x = torch.zeros(4, 10)
    u = torch.zeros(4, dtype=torch.float64)
    for f in (lambda: cb.top_classes(x, 3), lambda: cb.top_classes(np.zeros((4, 10)), 3), lambda: cb.top_classes(x.double(), 3),
              lambda: cb.distill_gradients(x, x, x), lambda: cb.sample_classes(x, u)):
        with pytest.raises((ValueError, RuntimeError)):
            f()


def test_the_plain_gradient_is_that_of_the_plain_loss():
    g = np.random.default_rng(0)
    for rest in (True, False):
        x = g.standard_normal((3, 12))
        u, ix, lse = O.top(g.standard_normal((3, 12)), 4, 1.5)
        base = lse if rest else None
        _, grad, _ = O.distill(x, u, ix, base, 1.5, None)
        for j in range(12):
            d = np.zeros((1, 12))
            d[0, j] = 1e-5
            up, dn = (O.distill(x + s * d, u, ix, base, 1.5, None)[0] for s in (1, -1))
            np.testing.assert_allclose((up - dn) / 2e-5, grad[:, j], atol=1e-8)


def test_the_plain_draw_has_its_frequencies():
    """Even steps of u hit every class as often as its kept mass says."""
    g = np.random.default_rng(1)
    x = g.standard_normal((1, 9))
    o, = O.sample(x, None, [1.0], [6], [0.8], [0.0], None)
    order = np.argsort(-x[0])
    kept = np.flatnonzero(o["kept"])
    assert set(kept) == set(order[:kept.size]) and 1 <= kept.size <= 6
    at = np.searchsorted(o["cum"], (np.arange(20000) + 0.5) / 20000 * o["cum"][-1], side="right")
    np.testing.assert_allclose(np.bincount(at, minlength=9) / 20000, o["kept"] / o["kept"].sum(), atol=1e-4)
