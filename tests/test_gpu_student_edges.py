"""AdamW and log probabilities over torch tensors where a program does the unusual (in a process of its own: torch is imported first there)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_torch_front_end_edges():
    pytest.importorskip("torch")
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-u", os.path.join(here, "torch_student_edges.py")], cwd=os.path.dirname(here),
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    print(r.stdout)
    assert r.returncode == 0, r.stdout[-3000:]
    assert r.stdout.rstrip().endswith("all checks passed")
