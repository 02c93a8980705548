"""Refusals of log probabilities, looked-up rows, their gradients and AdamW steps: typed errors before any device
call (no GPU needed); and the plain implementations that the GPU tests compare with, checked against each other."""
import ctypes as C

import numpy as np
import pytest

import catboost_rs_amd as cb
from catboost_rs_amd.adamw import _Settings, _Tensor
from tests import class_scores_oracle as O
from tests import student_oracle as S
from tests.test_class_scores_checks import BAD_SCORES, P, code, scores


@pytest.fixture(scope="module")
def lib():
    return cb.load()


def logprobs(lib, given=P, count=2, t=1.0, allowed=None, stride=0, k=3, lp=P, ent=P, st=P, tl=P, ti=P, ws=None, size=0, **kw):
    return code(lib.cbh_class_logprobs(*scores(**kw), given, count, t, allowed, stride, k, lp, ent, st, tl, ti, ws, size, None), lib)


def gradients(lib, given=P, count=2, g=P, h=P, st=P, t=1.0, allowed=None, stride=0, grad=P, grs=100, gcs=1, **kw):
    return code(lib.cbh_logprob_gradients(*scores(**kw), given, count, g, h, st, t, allowed, stride, grad, grs, gcs, None), lib)


@pytest.mark.parametrize("bad,want", BAD_SCORES)
def test_scores_are_checked(lib, bad, want):
    assert logprobs(lib, **bad) == want and gradients(lib, **bad) == want


def test_logprob_arguments_are_checked(lib):
    for f in (logprobs, gradients):
        assert f(lib, given=None) == -5 and f(lib, count=1025) == -2
        for t in (0.0, -1.0, float("nan"), float("inf"), 1e-320):
            assert f(lib, t=t) == -2
        assert f(lib, allowed=P + 2) == -5 and f(lib, allowed=P, stride=3) == -2 and f(lib, allowed=P, stride=-4) == -2
    assert logprobs(lib, k=101) == -2 and logprobs(lib, k=1025, classes=5000) == -2
    assert logprobs(lib, tl=None) == -5 and logprobs(lib, ti=None) == -5
    need = lib.cbh_class_logprobs_workspace(1, 200_000, 3)
    assert need > 0 and lib.cbh_class_logprobs_workspace(1 << 30, 32, 3) == 0
    for ws, size in ((None, 0), (P, need - 1), (P + 4, need)):
        assert logprobs(lib, rows=1, classes=200_000, ws=ws, size=size) == -1
    assert gradients(lib, g=None) == -5 and gradients(lib, st=None) == -5 and gradients(lib, grad=None) == -5
    assert gradients(lib, grad=P + 1) == -5 and gradients(lib, grs=1 << 61) == -2


def lookup(lib, table=P, type=0, entries=10, dim=4, rs=4, cs=1, index=P, rows=3, many=2, scale=1.0, out=P):
    return code(lib.cbh_lookup_rows(table, type, entries, dim, rs, cs, index, rows, many, scale, out, None), lib)


def table(lib, grad=P, type=0, entries=10, dim=4, rs=4, cs=1, index=P, rows=3, many=2, scale=1.0, out=P, out_type=0, ws=P, size=1 << 40):
    return code(lib.cbh_lookup_gradients(grad, type, rows, dim, rs, cs, index, many, entries, scale, out, out_type, ws, size, None), lib)


@pytest.mark.parametrize("f", [lookup, table])
def test_table_arguments_are_checked(lib, f):
    assert f(lib, type=3) == -4 and f(lib, entries=0) == -2 and f(lib, entries=1 << 31) == -2
    assert f(lib, dim=0) == -2 and f(lib, dim=(1 << 24) + 1) == -2 and f(lib, many=0) == -2
    assert f(lib, rows=1 << 31, many=1) == -2 and f(lib, rows=1 << 30, many=2) == -2
    assert f(lib, index=None) == -5 and f(lib, index=P + 2) == -5 and f(lib, out=None) == -5 and f(lib, out=P + 2) == -5
    assert f(lib, rs=1 << 61) == -2 and f(lib, cs=-(1 << 60)) == -2
    assert f(lib, scale=float("nan")) == -2 and f(lib, scale=float("inf")) == -2 and f(lib, scale=1e39) == -2


def test_table_workspace_is_checked(lib):
    assert lookup(lib, table=None) == -5 and table(lib, grad=None) == -5 and table(lib, out_type=5) == -4
    need = lib.cbh_lookup_gradients_workspace(3000, 2, 10, 4)
    assert need > 0 and lib.cbh_lookup_gradients_workspace(256, 2, 10, 4) == 0
    assert table(lib, rows=3000, size=need - 1) == -1
    assert table(lib, rows=3000, ws=None) == -1 and table(lib, rows=3000, ws=P + 8) == -1
    # what the entry refuses needs none
    assert lib.cbh_lookup_gradients_workspace(1 << 31, 1, 10, 4) == 0


def adamw(lib, count=1, tensor=None, **kw):
    base = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1)
    base.update(kw)
    t = dict(param=P, grad=2 * P, exp_avg=3 * P, exp_avg_sq=4 * P, exp_avg_scale=5 * P, exp_avg_sq_scale=6 * P, n=16)
    rows = [dict(t, **x) for x in (tensor if isinstance(tensor, list) else [tensor or {}])]
    a = (_Tensor * len(rows))(*(_Tensor(**r) for r in rows))
    return code(lib.cbh_adamw_step(a, len(rows), C.byref(_Settings(**base)), None), lib)


def test_adamw_arguments_are_checked(lib):
    assert code(lib.cbh_adamw_step(None, 1, C.byref(_Settings(step=1)), None), lib) == -5
    assert code(lib.cbh_adamw_step(None, 0, None, None), lib) == -5
    assert adamw(lib, state=2) == -4
    for b in (-0.1, 1.0, float("nan")):
        assert adamw(lib, beta1=b) == -2 and adamw(lib, beta2=b) == -2
    for x in (float("nan"), float("inf")):
        assert adamw(lib, lr=x) == -2 and adamw(lib, eps=x) == -2 and adamw(lib, weight_decay=x) == -2
    assert adamw(lib, eps=-1.0) == -2 and adamw(lib, step=0) == -2
    assert adamw(lib, step_device=P + 4) == -5 and adamw(lib, lr_device=P + 2) == -5
    assert adamw(lib, grad_scale=P + 2) == -5 and adamw(lib, skip=P + 2) == -5
    for name in ("param", "grad", "exp_avg", "exp_avg_sq"):
        assert adamw(lib, tensor={name: None}) == -5 and adamw(lib, tensor={name: 9 * P + 1}) == -5
    assert adamw(lib, state=1, tensor=dict(exp_avg_scale=None)) == -5
    assert adamw(lib, state=1, tensor=dict(exp_avg_sq_scale=6 * P + 2)) == -5
    assert adamw(lib, tensor=dict(param_type=3)) == -4 and adamw(lib, tensor=dict(grad_type=-1)) == -4
    assert adamw(lib, tensor=dict(copy=7 * P, copy_type=3)) == -4 and adamw(lib, tensor=dict(copy=7 * P + 2)) == -5
    assert adamw(lib, tensor=dict(n=(1 << 40) + 1)) == -2


def test_adamw_refuses_the_same_memory_twice(lib):
    far = {k: 100 * P + i * P for i, k in enumerate(("param", "exp_avg", "exp_avg_sq"))}
    assert adamw(lib, tensor=[{}, {}]) == -5                              # a tensor twice
    assert adamw(lib, tensor=[{}, dict(far, param=P + 60)]) == -5         # the last value of one
    assert adamw(lib, tensor=[{}, dict(far, exp_avg=3 * P)]) == -5
    assert adamw(lib, tensor=dict(copy=P + 32)) == -5
    assert adamw(lib, state=1, tensor=dict(exp_avg_scale=6 * P)) == -5


def test_adamw_refuses_a_gradient_that_it_would_write_over(lib):
    far = {k: 100 * P + i * P for i, k in enumerate(("param", "exp_avg", "exp_avg_sq"))}
    for grad in (P, P + 60, P - 60, 3 * P, 4 * P + 4, 100 * P + 32):
        assert adamw(lib, tensor=[dict(grad=grad), far]) == -5
    assert adamw(lib, tensor=dict(copy=7 * P, grad=7 * P)) == -5
    assert adamw(lib, state=1, tensor=dict(grad=6 * P)) == -5


def test_no_work_is_no_error(lib):
    s = scores(rows=0, data=None)
    assert lib.cbh_class_logprobs(*s, None, 1, 1.0, None, 0, 3, None, None, None, None, None, None, 0, None) == 0
    assert lib.cbh_logprob_gradients(*s, None, 1, None, None, None, 1.0, None, 0, None, 0, 0, None) == 0
    assert lib.cbh_lookup_rows(P, 0, 10, 4, 4, 1, None, 0, 2, 1.0, None, None) == 0
    assert lib.cbh_adamw_step(None, 0, C.byref(_Settings(step=1)), None) == 0
    assert lib.cbh_adamw_step((_Tensor * 1)(_Tensor()), 1, C.byref(_Settings(step=1)), None) == 0


def test_the_functions_refuse_what_is_no_gpu_tensor():
    torch = pytest.importorskip("torch")
    x, i = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int32)
    for f in (lambda: cb.class_logprobs(x, i), lambda: cb.logprob_gradients(x, i, x[:, 0], x[:, :3]), lambda: cb.lookup_rows(x, i),
              lambda: cb.lookup_gradients(x, i, 5), lambda: cb.AdamW([x]), lambda: cb.AdamW([np.zeros(3)])):
        with pytest.raises((ValueError, RuntimeError)):
            f()


# ---- the plain implementations -----------------------------------------------------------------
def test_the_plain_log_probabilities_are_those_of_a_softmax():
    g = np.random.default_rng(0)
    x, given = g.standard_normal((4, 9)) * 3, g.integers(-1, 9, (4, 3))
    free = g.random((4, 9)) < 0.7
    free[:, 2] = True
    lp, ent, st, top, index = S.logprobs(x, given, 1.5, 4, free)
    for r in range(4):
        p = np.where(free[r], np.exp(x[r] / 1.5), 0)
        p /= p.sum()
        with np.errstate(divide="ignore"):
            want = np.where(given[r] >= 0, np.log(p[given[r]]), 0)
        np.testing.assert_allclose(lp[r], want, rtol=1e-12)
        np.testing.assert_allclose(ent[r], -(p[p > 0] * np.log(p[p > 0])).sum(), rtol=1e-12)
        best = np.argsort(-p, kind="stable")[:4]
        assert np.array_equal(index[r], np.where(p[best] > 0, best, -1))


@pytest.mark.parametrize("entropy", [False, True])
def test_the_plain_gradient_is_that_of_the_plain_forward_pass(entropy):
    g = np.random.default_rng(1)
    x, given = g.standard_normal((3, 8)), np.array([[1, 1, -1], [7, 0, 99], [3, 4, 3]])
    up, h = g.standard_normal((3, 3)), g.standard_normal(3) if entropy else None
    free = np.ones((3, 8), bool)
    free[1, 5] = free[2, 0] = False

    def value(x):
        lp, ent, *_ = S.logprobs(x, given, 0.7, 0, free)
        return (lp * up).sum(1) + (ent * h if entropy else 0.0)

    grad, _ = S.logprob_gradients(x, given, up, h, 0.7, free)
    for j in range(8):
        d = np.zeros((1, 8))
        d[0, j] = 1e-5
        np.testing.assert_allclose((value(x + d) - value(x - d)) / 2e-5, grad[:, j], atol=1e-8)


def test_the_plain_table_gradient_is_that_of_the_plain_lookup():
    g = np.random.default_rng(2)
    table, index, up = g.standard_normal((5, 3)), g.integers(-1, 6, (7, 4)), g.standard_normal((7, 3))
    grad, _, count = S.table_gradient(up, index, 5, 0.5)
    assert count.sum() == ((index >= 0) & (index < 5)).sum()
    for v in range(5):
        for c in range(3):
            d = np.zeros((5, 3))
            d[v, c] = 1e-5
            num = ((S.lookup(table + d, index, 0.5)[0] - S.lookup(table - d, index, 0.5)[0]) * up).sum() / 2e-5
            np.testing.assert_allclose(num, grad[v, c], atol=1e-8)


def test_the_plain_step_in_32_bits_is_that_in_64():
    g = np.random.default_rng(3)
    p, gr, m = g.standard_normal((3, 1000)).astype(np.float32)
    v = g.random(1000).astype(np.float32)
    for step in (1, 2, 1000, 10 ** 6):
        a, b = S.adamw_f32(p, gr, m, v, step), S.adamw(p, gr, m, v, step)
        for x, y in zip(a, b):
            np.testing.assert_allclose(x, y, rtol=3e-5, atol=3e-6)


def test_the_plain_codes_are_the_values_next_to_what_they_hold():
    g = np.random.default_rng(4)
    x = (g.standard_normal(3000) * np.exp(g.uniform(-12, 3, 3000))).astype(np.float32)
    x[:300] = 0
    x[700] = 448.0
    low, high = S.random_bits(3000, 7, 3, 1)
    c, s = S.encode(x, low, False)
    assert s[0] == 0 and (c[:256] == 0).all()
    y = S.decode(c, s)
    each = np.repeat(s, 256)[:3000]
    with np.errstate(all="ignore"):
        q = np.abs(x) / each
    step = np.where(each > 0, each * np.maximum(2.0 ** -9, 2.0 ** (np.floor(np.log2(np.maximum(q, 1e-30))) - 3)), 0)
    assert (np.abs(x - y) <= step).all() and (np.sign(y) * np.sign(x) >= 0).all()
    largest = np.abs(np.pad(x, (0, -3000 % 256))).reshape(-1, 256).max(1)
    assert ((largest[2:] / s[2:] > 224) & (largest[2:] / s[2:] <= 448)).all()
    assert (S.encode(np.abs(x), low, True)[0][x != 0] > 0).all()


def test_random_bits_are_even():
    """16 bits of 2^20 values each: every one of the upper 8 bits' values as often as another within 5 of its standard
    deviations, and rounding by them keeps the mean."""
    for step, number in ((1, 0), (2, 0), (1, 1)):
        for bits in S.random_bits(1 << 20, 3, step, number):
            n = np.bincount(bits >> 8, minlength=256)
            assert np.abs(n - 4096).max() < 5 * 64
    x = np.full(1 << 16, 1.03, np.float32)
    x[::256] = 1.75   # (scale 2^-8 for every block)
    y = S.decode(*S.encode(x, S.random_bits(1 << 16, 3, 1, 0)[0], False))
    free = x != 1.75
    # steps of 1/8 taken with probability 0.24: a standard deviation of 0.0534 a value
    assert abs(y[free].mean() - 1.03) < 5 * 0.0534 / 256 and set(np.unique(y[free])) == {1.0, 1.125}


def test_masked_scores_match_the_class_score_oracle():
    g = np.random.default_rng(5)
    x = O.scores(g, 6, 50, "masked").astype(np.float64)
    _, ent, st, top, index = S.logprobs(x, np.zeros((6, 1), int), 1.0, 5)
    lse = O.log_sum_exp(x)
    with np.errstate(invalid="ignore"):
        np.testing.assert_allclose(np.where(np.isneginf(lse), 0, st[:, 0] + st[:, 1] - lse), 0, atol=1e-9)
    assert st[0, 0] == -np.inf and ent[0] == 0 and (index[0] == -1).all()
