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


def check_scores_of_a_model():
    """Scores that require a gradient: nothing is recorded, and backward(grad) gives the model's."""
    inputs = torch.randn(50, 8, device="cuda")
    v, i, s = cb.top_classes(torch.randn(50, 12, device="cuda"), 3, temperature=2.0)
    weight = torch.randn(8, 12, device="cuda", requires_grad=True)
    scores = inputs @ weight
    loss, grad = cb.distill_gradients(scores, v, i, top_lse=s, temperature=2.0)
    assert not loss.requires_grad and not grad.requires_grad
    scores.backward(grad)
    torch.testing.assert_close(weight.grad, inputs.t() @ grad, rtol=1e-5, atol=1e-5)
    # against autograd through the formulas
    leaf = scores.detach().double().requires_grad_()
    lp = torch.log_softmax(leaf / 2.0, 1)
    q = torch.exp(v.double() / 2.0 - s.double()[:, None])
    rest = 1 - q.sum(1)
    others = torch.logsumexp(lp.scatter(1, i.long(), float("-inf")), 1)
    want = 4.0 * ((q * (torch.log(q) - lp.gather(1, i.long()))).sum(1) + rest * (torch.log(rest) - others))
    want.sum().backward()
    # (12 classes: f32 exponentials of |d| <= 20, off by 62 roundings, and the roundings of sums)
    assert (grad - leaf.grad).abs().max().item() <= 2.0 * 100 * 2.0 ** -24
    assert (loss - want).abs().max().item() <= 4.0 * 300 * 2.0 ** -24


if __name__ == "__main__":
    for name, f in list(globals().items()):
        if name.startswith("check_"):
            print(name, flush=True)
            f()
            torch.cuda.synchronize()
    print("all checks passed")
