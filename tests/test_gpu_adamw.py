"""AdamW steps (cbh_adamw_step) on device buffers: bit for bit the plain f32 implementation, whose every operation rounds
as the device's does, which in turn meets the formula in 64 bits.

Bars of the latter: m and v are sums of two products (five roundings with those of the betas); the step is m's
times three roundings more, over a root (half of v's relative error, one rounding) and a sum; p two more.
"""
import ctypes as C

import numpy as np
import pytest

import catboost_rs_amd as cb
from catboost_rs_amd.adamw import _Settings, _Tensor
from tests import class_scores_oracle as O
from tests import student_oracle as S
from tests.device_buffers import Buffers
from tests.test_gpu_class_scores import TYPE

pytestmark = pytest.mark.gpu

SIZES = [1, 3, 4, 255, 256, 257, 1000, 4095, 4096, 4097, 70001]


def tensors(g, sizes, kind, grad_kind, small):
    out = []
    for n in sizes:
        p = O.round_to(g.standard_normal(n).astype(np.float32), kind)
        gr = O.round_to((g.standard_normal(n) * np.exp(g.uniform(-6, 1, n))).astype(np.float32), grad_kind)
        gr[g.random(n) < 0.1] = 0
        m, v = (g.standard_normal(n) * 0.1).astype(np.float32), (g.random(n) ** 4).astype(np.float32)
        v[g.random(n) < 0.1] = 0
        m[v == 0] = 0
        t = dict(p=p, g=gr)
        if small:
            t["m"], t["ms"] = S.encode(m, np.zeros(n, np.uint32), False)
            t["v"], t["vs"] = S.encode(np.sqrt(v), np.zeros(n, np.uint32), True)
        else:
            t["m"], t["v"] = m, v
        out.append(t)
    return out


def step(ts, kind, grad_kind, small, number=0, copy=None, skip=0, odd=False, on_device=False, **settings):
    """One step on copies of the tensors; what they are then."""
    L = cb.load()
    new = []
    pad = 1 if odd else 0   # (tensors that start behind an element, and 8-bit states behind a byte)
    with Buffers() as b:
        def put(a):
            return b.put(np.concatenate([np.zeros(pad, a.dtype), a])) + pad * a.itemsize, a

        recs, kept = (_Tensor * len(ts))(), []
        for i, t in enumerate(ts):
            r, n = recs[i], len(t["p"])
            ptr = {}
            for name, a in (("p", O.to_bits(t["p"], kind)), ("g", O.to_bits(t["g"], grad_kind)), ("m", t["m"]), ("v", t["v"])):
                ptr[name], _ = put(a)
            if small:
                ptr["ms"], ptr["vs"] = b.put(t["ms"]), b.put(t["vs"])
            if copy:
                ptr["c"] = b.put(O.to_bits(np.full(n, 9, np.float32), copy))
            r.param, r.grad, r.exp_avg, r.exp_avg_sq, r.n = ptr["p"], ptr["g"], ptr["m"], ptr["v"], n
            r.exp_avg_scale, r.exp_avg_sq_scale, r.copy = ptr.get("ms"), ptr.get("vs"), ptr.get("c")
            r.param_type, r.grad_type, r.copy_type, r.number = TYPE[kind], TYPE[grad_kind], TYPE[copy or "f32"], number + i
            kept.append(ptr)
        s = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, step=1, seed=0)
        s.update(settings)
        if s.get("grad_scale") is not None:
            s["grad_scale"] = b.put(np.array([s["grad_scale"]], np.float32))
        if on_device:
            s["step_device"], s["lr_device"] = b.put(np.array([s["step"]], np.int64)), b.put(np.array([s["lr"]], np.float32))
            s["step"], s["lr"] = 0, 123.0
        s["skip"] = b.put(np.array([skip], np.int32))
        cb._check(L.cbh_adamw_step(recs, len(ts), C.byref(_Settings(state=int(small), **s)), None))
        for t, ptr in zip(ts, kept):
            u = {"g": t["g"]}
            u["p"] = O.from_bits(b.get(ptr["p"] - pad * (4 if kind == "f32" else 2))[pad:], kind)
            b.get(ptr["g"] - pad * (4 if grad_kind == "f32" else 2))
            size = 1 if small else 4
            u["m"], u["v"] = (b.get(ptr[x] - pad * size)[pad:] for x in "mv")
            if small:
                u["ms"], u["vs"] = b.get(ptr["ms"]), b.get(ptr["vs"])
            if copy:
                u["c"] = O.from_bits(b.get(ptr["c"]), copy)
            new.append(u)
    return new


def expected(t, small, seed=0, number=0, **kw):
    if small:
        m, v = S.decode(t["m"], t["ms"]), np.square(S.decode(t["v"], t["vs"]))
    else:
        m, v = t["m"], t["v"]
    p, m, v, root = S.adamw_f32(t["p"], t["g"], m, v, **kw)
    if not small:
        return dict(p=p, m=m, v=v)
    low, high = S.random_bits(len(p), seed, kw["step"], number)
    (cm, sm), (cv, sv) = S.encode(m, low, False), S.encode(root, high, True)
    return dict(p=p, m=cm, ms=sm, v=cv, vs=sv)


def check(new, ts, kind, small, copy=None, number=0, **kw):
    for i, (u, t) in enumerate(zip(new, ts)):
        e = expected(t, small, number=number + i, **kw)
        for name in e:
            want = O.round_to(e[name], kind) if name == "p" else e[name]
            if want.dtype == np.uint8:   # (0x7F and 0xFF are both NaN)
                got, want = (np.where(c & 0x7F == 0x7F, 0x7F, c) for c in (u[name], want))
                assert np.array_equal(got, want), (i, len(t["p"]), name)
                continue
            assert np.array_equal(u[name], want, equal_nan=u[name].dtype.kind == "f"), (i, len(t["p"]), name)
        if copy:
            assert np.array_equal(u["c"], O.round_to(e["p"], copy), equal_nan=True), (i, "copy")


@pytest.mark.parametrize("small", [False, True])
@pytest.mark.parametrize("grad_kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_types_and_sizes(kind, grad_kind, small):
    g = np.random.default_rng(1)
    ts = tensors(g, SIZES, kind, grad_kind, small)
    for n in (1, 2, 1000):
        check(step(ts, kind, grad_kind, small, step=n, seed=5), ts, kind, small, step=n, seed=5)
    check(step(ts, kind, grad_kind, small, step=3, odd=True), ts, kind, small, step=3)


@pytest.mark.parametrize("small", [False, True])
def test_settings(small):
    g = np.random.default_rng(2)
    ts = tensors(g, [1000, 5, 300], "f32", "bf16", small)
    for kw in (dict(lr=0.0), dict(beta1=0.0), dict(beta2=0.0), dict(beta1=0.0, beta2=0.0), dict(weight_decay=0.0), dict(weight_decay=-0.5),
               dict(eps=0.0), dict(eps=1.0), dict(grad_scale=0.125), dict(grad_scale=0.0), dict(seed=0xFFFFFFFF), dict(lr=-1e-2)):
        n = dict(step=7, **kw)
        check(step(ts, "f32", "bf16", small, number=3, **n), ts, "f32", small, number=3, **n)
    # the step and the rate from the device (a rate in f32)
    rate = float(np.float32(3e-4))
    for n in (1, 999, 123456):
        check(step(ts, "f32", "bf16", small, step=n, lr=rate, on_device=True), ts, "f32", small, step=n, lr=rate)
    # copies in 16 bits
    for copy in ("bf16", "f16", "f32"):
        check(step(ts, "f32", "bf16", small, step=2, copy=copy), ts, "f32", small, copy=copy, step=2)


@pytest.mark.parametrize("small", [False, True])
def test_a_step_held_back_changes_nothing(small):
    ts = tensors(np.random.default_rng(3), [700, 4], "bf16", "f32", small)
    for u, t in zip(step(ts, "bf16", "f32", small, skip=1, copy="f16"), ts):
        assert all(np.array_equal(u[name], t[name]) for name in t) and (u["c"] == 9).all()


@pytest.mark.parametrize("small", [False, True])
def test_many_tensors(small):
    """More than a launch takes, of different sizes, empty ones among them, some without alignment."""
    g = np.random.default_rng(4)
    ts = tensors(g, [int(n) for n in np.exp(g.uniform(0, 8, 101))], "f32", "f32", small)
    ts[50] = {k: v[:0] for k, v in ts[50].items()}
    check(step(ts, "f32", "f32", small, step=4, seed=9), ts, "f32", small, step=4, seed=9)


@pytest.mark.parametrize("small", [False, True])
def test_nan_infinity_and_the_ends_of_f32(small):
    g = np.random.default_rng(5)
    t, = tensors(g, [1500], "f32", "f32", small)
    t["g"][:8] = np.nan, np.inf, -np.inf, 3e38, -3e38, 1e-45, 1e-38, -1e-30
    t["g"][300] = 2e19      # (its square is near the largest f32)
    t["g"][600:900] = 0
    for name in ("m", "v"):
        t[name][512:1100] = 0   # blocks of nothing
    if small:
        t["ms"][2:4] = t["vs"][2:4] = 0
    new = step([t], "f32", "f32", small, step=2)
    check(new, [t], "f32", small, step=2)
    if small:
        u = new[0]
        assert (u["m"][:3] & 0x7F == 0x7F).all() and (u["v"][:3] & 0x7F == 0x7F).all()
        assert (u["m"][8:256] & 0x7F != 0x7F).all() and np.isfinite(u["ms"]).all() and np.isfinite(u["vs"]).all()


def test_the_step_meets_the_formula():
    g = np.random.default_rng(6)
    ts = tensors(g, [5000], "f32", "f32", False)
    t, = ts
    for n in (1, 10, 5000):
        u, = step(ts, "f32", "f32", False, step=n)
        p, m, v = S.adamw(t["p"], t["g"], t["m"], t["v"], n)
        h = 2.0 ** -24
        sm = 0.9 * np.abs(t["m"]) + 0.1 * np.abs(t["g"])
        denom = np.sqrt(v / (1 - 0.999 ** n)) + 1e-8
        rate = 1e-3 / (1 - 0.9 ** n)
        assert (np.abs(u["m"] - m) <= 5 * h * sm + 1e-45).all()
        assert (np.abs(u["v"] - v) <= 6 * h * v + 1e-44).all()
        tol = rate / denom * (5 * h * sm + 10 * h * np.abs(m)) + 3 * h * np.abs(t["p"]) + h * np.abs(p)
        assert (np.abs(u["p"] - p) <= tol + 1e-44).all(), n


def test_states_in_8_bits_follow():
    """A second moment that changes by less than half a code's step a step is followed: after 3000 steps at beta2 = 0.999
    with gradients of one size, its root is that size, from a tenth of it."""
    n = 1 << 12
    t = dict(p=np.zeros(n, np.float32), g=np.full(n, 0.5, np.float32))
    t["g"][::256] = 2.0     # (so that the block's scale is not the others')
    t["m"], t["ms"] = S.encode(np.zeros(n, np.float32), np.zeros(n, np.uint32), False)
    t["v"], t["vs"] = S.encode(t["g"] * np.float32(0.1), np.zeros(n, np.uint32), True)
    L = cb.load()
    with Buffers() as b:
        ptr = {k: b.put(a) for k, a in t.items()}
        r = (_Tensor * 1)(_Tensor(param=ptr["p"], grad=ptr["g"], exp_avg=ptr["m"], exp_avg_sq=ptr["v"], exp_avg_scale=ptr["ms"],
                                  exp_avg_sq_scale=ptr["vs"], n=n))
        for i in range(3000):
            s = _Settings(lr=0.0, beta1=0.9, beta2=0.999, eps=1e-8, step=i + 1, seed=1, state=1)
            cb._check(L.cbh_adamw_step(r, 1, C.byref(s), None))
        root, m = S.decode(b.get(ptr["v"]), b.get(ptr["vs"])), S.decode(b.get(ptr["m"]), b.get(ptr["ms"]))
    free = t["g"] == 0.5
    # v is 0.25 (1 - 0.99 * 0.999^3000) = 0.2377; a value wanders by steps of 1/8 of its root at most: the mean of 4080 values of a standard
    # deviation below 2 steps of 0.03125 lies within 5 * 0.001 of it, and the codes' own rounding of the square within
    # a step's half
    assert abs(np.sqrt(np.mean(root[free].astype(np.float64) ** 2)) - np.sqrt(0.2377)) < 0.02
    assert abs(m[free].mean() - 0.5) < 0.01
