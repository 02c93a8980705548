"""Workspace sizes of the operators on class scores at the ends of their arguments' types: a number, whatever is asked (in a
process of its own: a division by zero would end it)."""
import os
import subprocess
import sys

import pytest

SIZES = [0, 1, 2048, 2049, (1 << 24) - 1, 1 << 24, (1 << 24) + 1, (1 << 32) - 131072, (1 << 32) - 131071, (1 << 32) - 1]
ROWS = [0, 1, 511, 512, 1000, (1 << 31) - 1, 1 << 31, (1 << 64) - 1]
CALLS = {"cbh_top_classes_workspace": (1, 1024), "cbh_distill_gradients_workspace": (), "cbh_sample_classes_workspace": (),
         "cbh_class_logprobs_workspace": (0, 1024)}


@pytest.mark.parametrize("name", CALLS)
def test_workspaces_of_any_size(name):
    tail = CALLS[name] or (None,)
    code = f"""
import catboost_rs_amd as cb
f = cb.load().{name}
for rows in {ROWS}:
    for classes in {SIZES}:
        for k in {tail}:
            assert f(*([rows, classes] + ([] if k is None else [k]))) >= 0
print("done")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == "done", (r.returncode, r.stderr[-500:])
