"""Looked-up rows of long lists on both sides of the rule that holds entries in LDS: whole rows, 64 bytes of them, less of
rows that are no whole vectors, and from the caches.  Bars: test_gpu_lookup."""
import numpy as np
import pytest

from tests import class_scores_oracle as O
from tests import student_oracle as S
from tests.test_gpu_lookup import bar, indices, run_lookup

# rows, list, entries, dim
SHAPES = [(33000, 40, 5150, 13), (33000, 40, 5150, 5), (33000, 40, 5150, 16), (160000, 9, 5400, 3), (330000, 8, 10239, 2),
          (330000, 8, 10240, 2), (8300, 81, 2570, 24), (8300, 81, 2570, 30), (8200, 80, 2559, 64), (9000, 41, 1290, 70), (1000, 40, 90, 511),
          (33000, 40, 5150, 520), (41500, 33, 5300, 150), (170000, 8, 5200, 70)]


def way(rows, many, entries, dim, kind):
    """Vectors of every entry that are held in LDS, and those of a row; 0 held: from the caches."""
    vec = 4 if kind == "f32" else 8
    lanes = 1
    while lanes < 64 and lanes * vec < dim:
        lanes *= 2
    held = lanes
    while held > 1 and (entries + 1) * held * 16 > 163840:
        held //= 2
    share = 1 if dim % vec == 0 else 64 if many >= 32 and (vec == 8 or held >= 2) else 8 if vec == 8 else 2
    fits = many >= 8 and rows * many >= 256 * entries and (entries + 1) * held * 16 <= 163840
    large = many >= 32 and entries * dim * (16 // vec) > 8 << 20
    return (held if fits and (held >= 4 or lanes <= held * share or large) else 0), lanes


def test_both_sides_have_shapes():
    for kind in ("f32", "bf16"):
        ways = {way(*shape, kind) for shape in SHAPES}
        held = {h for h, _ in ways}
        assert {0, 1, 4} <= held and max(held) >= 16
        assert any(0 < h < lanes for h, lanes in ways) and any(0 < h == lanes for h, lanes in ways)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,many,entries,dim", SHAPES)
def test_lookup_ways(rows, many, entries, dim, kind):
    g = np.random.default_rng(entries + dim)
    table, index = O.scores(g, entries, dim, "normal"), indices(g, rows, many, entries, "even")
    for order, scale in (("rows", 1.0), ("padded", 0.1)):
        got = run_lookup(table, index, scale, kind, order)
        some = np.concatenate([np.arange(300), rows - 1 - np.arange(300)])   # (rows from both ends)
        want, size = S.lookup(O.round_to(table, kind), index[some], scale)
        assert (np.abs(got[some] - want) <= bar(want, size, many, kind)).all(), (order, scale)
        # all rows: the sum of a list of one entry repeated, and of nothing, in every place
        one = np.where(np.arange(many)[None] < 2, np.arange(rows)[:, None] % (entries + 1) - 1, -1).astype(np.int32)
        got = run_lookup(table, one, 0.5, kind, order)
        v = np.concatenate([np.zeros((1, dim), np.float32), O.round_to(table, kind)])
        assert np.array_equal(got, v[one[:, 0] + 1]), (order, "repeated")
