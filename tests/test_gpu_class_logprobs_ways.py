"""Log probabilities of many long rows, by every way that the library's rule chooses between: workgroups of one wave or
of four, and the largest classes by groups of 32, by vectors, or over the whole row.

Rows repeat a few that are hard (ties, NaN, infinities, equal scores): those are compared with the plain implementation
in 64 bits, with the bars of test_gpu_class_logprobs, and all others with them, bit for bit.
"""
import numpy as np
import pytest

import catboost_rs_amd as cb
from tests import class_scores_oracle as O
from tests import student_oracle as S
from tests.device_buffers import Buffers
from tests.test_gpu_class_logprobs import close, words
from tests.test_gpu_class_scores import TYPE, reach, workspace

# rows, classes, k
SHAPES = [(2100, 2500, 0), (2100, 8192, 5), (2100, 2500, 20), (2050, 6000, 150), (2048, 10000, 300), (2100, 2500, 700),
          (600, 20000, 0), (600, 20000, 20), (600, 20000, 150), (520, 40000, 300), (300, 2500, 20), (300, 6000, 150),
          (300, 10000, 300), (300, 2500, 700), (515, 65536, 1000), (1030, 140001, 0)]
KINDS = ["f32", "f16", "bf16"]


def way(rows, n, k, kind):
    """The rule of the library: waves of a workgroup, how the largest are found, and the list that they are kept in."""
    parts = -(-n // (64 * 2048))
    if rows < 512 and n >= 2 * 8192:
        parts = max(parts, min(-(-512 // rows), n // 8192))
    seg = (-(-n // parts) + 31) // 32 * 32
    parts = -(-n // seg)
    shortest, vec = n - seg * (parts - 1), 4 if kind == "f32" else 8
    waves = 1 if rows * parts >= 2048 and (k == 0 or seg <= 16384) else 4
    kept = 256 if k <= 128 else 512 if k <= 256 else 2048
    if k == 0:
        return waves, "none", 0
    if 4 * k <= shortest // 32:
        return waves, "groups", kept
    if 4 * k <= shortest // vec and 4 * (2048 // vec) * -(-seg // 2048) <= 65536:
        return waves, "vectors", kept
    return waves, "whole", 0


def test_every_way_has_a_shape():
    ways = {(w, how, kept) for w in (1, 4) for how in ("groups", "vectors") for kept in (256, 512, 2048)}
    ways |= {(w, how, 0) for w in (1, 4) for how in ("none", "whole")}
    ways -= {(1, "groups", 512), (1, "groups", 2048)}   # (rows that long are not by one wave)
    for kind in KINDS:
        assert {way(*shape, kind) for shape in SHAPES} == ways


def hard_rows(g, n):
    x = np.concatenate([O.scores(g, 1, n, kind) for kind in ("normal", "ties", "equal", "rising", "sharp", "normal", "normal")] +
                       [O.scores(g, 3, n, "masked")])
    x[5, [n // 2, n - 1]] = np.nan, -np.nan
    x[6, g.integers(0, n, 3)] = np.inf
    return x


def run(base, given, t, k, kind, rows, order, allowed):
    """The library's answers on `rows` rows that repeat those of `base`."""
    L = cb.load()
    repeat = np.arange(rows) % len(base)
    bits = O.to_bits(base, kind)
    n, m = base.shape[1], given.shape[1]
    with Buffers() as b:
        block = np.ascontiguousarray(bits.T)[:, repeat] if order == "classes" else bits[repeat]
        rs, cs = (1, rows) if order == "classes" else (n, 1)
        x = b.put(block, fill=0xFF)
        mask = (None, 0) if allowed is None else (b.put(words(allowed)[repeat], fill=0xFF), -(-n // 32))
        out = [b.out((rows, m), np.float32), b.out(rows, np.float32), b.out((rows, 3), np.float32),
               b.out((rows, k), np.float32), b.out((rows, k), np.int32)]
        ws = workspace(b, L.cbh_class_logprobs_workspace(rows, n, k))
        cb._check(L.cbh_class_logprobs(x, TYPE[kind], rows, n, rs, cs, b.put(given[repeat].astype(np.int32)), m, t, *mask, k,
                                       *out, *ws, None))
        if ws[0]:
            b.get(ws[0])
        return [b.get(p) for p in out], repeat


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_ways(rows, n, k, kind):
    g = np.random.default_rng(n + k)
    base, t = hard_rows(g, n), 1.25
    given = g.integers(-1, n, (len(base), 3))
    free = g.random(base.shape) < 0.6
    free[-1] = False
    for order in ("rows", "classes") if rows * n <= 13_000_000 else ("rows",):
        for allowed in (None, free):
            tag = (order, allowed is not None)
            got, repeat = run(base, given, t, k, kind, rows, order, allowed)
            for a in got:
                assert np.array_equal(a, a[repeat], equal_nan=a.dtype.kind == "f"), tag
            lp, ent, st, top, index = (a[:len(base)] for a in got)
            h = O.round_to(base, kind)
            elp, eent, est, etop, eindex = S.logprobs(h, given, t, k, allowed)
            assert np.array_equal(index, eindex), tag
            z = (n / 64 + 16 + reach(S.masked(h, allowed), t)) * 2.0 ** -23
            e = np.nan_to_num(est[:, 2]) * 2 * z

            def rounded(want):
                return np.abs(np.where(np.isfinite(want), want, 0)) * 2.0 ** -24

            close(lp, elp, z + rounded(elp), (tag, "logprob"))
            close(top, etop, z + rounded(etop), (tag, "top"))
            close(ent, eent, z + e + rounded(eent), (tag, "entropy"))
            close(st[:, 0], est[:, 0], 0.0, (tag, "largest"))
            close(st[:, 1], est[:, 1], z + rounded(est[:, 1]), (tag, "log z"))
            close(st[:, 2], est[:, 2], e + rounded(est[:, 2]), (tag, "far"))
