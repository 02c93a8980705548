"""The operators on class scores over torch tensors at the ends of their arguments: run by
tests/test_gpu_class_scores_edges.py in a process of its own, or by hand (python tests/torch_class_scores_edges.py,
on a GPU)."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import catboost_rs_amd as cb  # noqa: E402


def refused(f, *a, **kw):
    try:
        f(*a, **kw)
    except cb.CbhError:
        return True
    return False


def check_sizes_beyond_32_bits():
    """Numbers that 32 bits would cut off are refused, or mean what they say (expanded tensors take no memory)."""
    one = torch.zeros(1, 1, device="cuda")
    u = torch.zeros(1, dtype=torch.float64, device="cuda")
    v, i = torch.zeros(1, 3, device="cuda"), torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    for n in ((1 << 24) + 1, (1 << 32) + 5):
        x = one.expand(1, n)
        assert refused(cb.top_classes, x, 5) and refused(cb.distill_gradients, x, v, i) and refused(cb.sample_classes, x, u)
    x = torch.randn(6, 40, device="cuda")
    for k in ((1 << 32) + 1, 1 << 40, -(1 << 32) + 3):
        assert refused(cb.top_classes, x, k)
    u = torch.full((6,), 0.999, dtype=torch.float64, device="cuda")
    all_classes = cb.sample_classes(x, u)
    for k in (40, (1 << 32) + 1, 1 << 40):
        for a, b in zip(all_classes, cb.sample_classes(x, u, top_k=k)):
            assert torch.equal(a, b), k


if __name__ == "__main__":
    for name, f in list(globals().items()):
        if name.startswith("check_"):
            print(name, flush=True)
            f()
            torch.cuda.synchronize()
    print("all checks passed")
