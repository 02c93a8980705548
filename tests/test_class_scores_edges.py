"""Refusals of the operators on class scores at the ends of their arguments (no GPU needed)."""
import pytest

import catboost_rs_amd as cb

P = 4096   # an aligned address that no call here may reach


@pytest.fixture(scope="module")
def lib():
    return cb.load()


@pytest.mark.parametrize("t,taken", [(1e-45, False), (1e-40, False), (4e-39, False), (9e-39, False), (1e-38, True), (1e-30, True),
                                     (1e30, True), (1e36, True), (1.1e36, False), (2e38, False), (1e45, False),
                                     (1e300, False)])
def test_temperatures_whose_arithmetic_leaves_f32_are_refused(lib, t, taken):
    """1 / t and the scores' differences are f32: below 1e-38 1 / t is infinite (every row was NaN), above 1e36 a difference
    of scores may be where its quotient by t is not (and from 2e45 on 1 / t is 0: NaN beside -inf)."""
    for rows in (0, 4):   # (no rows: a temperature that is taken does nothing)
        if rows and taken:
            continue
        top = lib.cbh_top_classes(P, 0, rows, 100, 100, 1, 5, t, P, P, P, None, 0, None)
        distill = lib.cbh_distill_gradients(P, 0, rows, 100, 100, 1, P, P, 5, None, t, None, P, P, 100, 1, None, 0, None)
        assert top == distill == (0 if taken else -2)
        assert taken or b"1e-38" in lib.cbh_last_error()
