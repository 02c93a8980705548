"""The operators on class scores over torch tensors: run by tests/test_gpu_class_scores.py in a
process of its own, or by hand (python tests/torch_class_scores.py, on a GPU)."""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import catboost_rs_amd as cb  # noqa: E402
from tests import class_scores_oracle as O  # noqa: E402

KIND = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}


def case(rows, n, dtype, seed=0, spread=2.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = (torch.randn(rows, n, generator=g, device="cuda") * spread).to(dtype)
    return x, x.float().cpu().numpy(), torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)


def check_types_and_layouts():
    for dtype in KIND:
        for rows, n in ((4, 1000), (257, 10), (3, 40001)):
            x, h, u = case(rows, n, dtype, n)
            for y in (x, x.t().contiguous().t(), torch.nn.functional.pad(x, (3, 4))[:, 3:3 + n]):
                k = min(n, 5)
                v, i, s = cb.top_classes(y, k, temperature=2.0)
                ev, ei, es = O.top(h, k, 2.0)
                assert np.array_equal(i.cpu().numpy(), ei) and np.array_equal(v.cpu().numpy(), ev.astype(np.float32))
                np.testing.assert_allclose(s.cpu().numpy(), es, rtol=2e-5)
                loss, grad = cb.distill_gradients(y, v, i, top_lse=s, temperature=2.0)
                assert grad.dtype == dtype and grad.shape == y.shape and loss.dtype == torch.float32
                el, eg, _ = O.distill(h, v.cpu().numpy(), ei, s.cpu().numpy(), 2.0, None)
                np.testing.assert_allclose(loss.cpu().numpy(), el, atol=4 * (n / 64 + 64) * 2.0 ** -23 * 3)
                np.testing.assert_allclose(grad.float().cpu().numpy(), eg, atol=2e-4, rtol=2.0 ** -7)
                j, lp = cb.sample_classes(y, u, temperature=0.9, top_k=40, top_p=0.9)
                f = np.ones(rows)
                O.check_sample(j.cpu().numpy(), lp.cpu().numpy(), O.sample(h, None, f * 0.9, f * 40, f * 0.9, f * 0, None),
                               u.cpu().numpy(), n)


def check_a_lists_own_student_has_no_loss():
    """A student whose scores are the teacher's has loss 0 and gradient 0, listed in part or in whole."""
    x, _, _ = case(5, 3001, torch.float32, 3)
    for k in (7, 1000):
        v, i, s = cb.top_classes(x, k)
        loss, grad = cb.distill_gradients(x, v, i, top_lse=s)
        assert loss.abs().max().item() < 1e-4 and grad.abs().max().item() < 1e-5


def check_other_streams():
    x, h, u = case(64, 50021, torch.float32, 4)
    want = cb.sample_classes(x, u, top_p=0.9), cb.top_classes(x, 20)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 1.0
        got = cb.sample_classes(y, u, top_p=0.9), cb.top_classes(y, 20)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want, got):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def check_graph_replays():
    """Captured once, replayed with new inputs and eager work between the replays."""
    for rows, n in ((2, 70001), (40, 2000), (300, 10)):
        x, _, u = case(rows, n, torch.bfloat16, 5)
        k = min(n, 9)

        def step():
            v, i, s = cb.top_classes(x, k)
            loss, grad = cb.distill_gradients(x, v.flip(1), i, top_lse=s)
            j, lp = cb.sample_classes(x, u, top_k=50, top_p=0.9)
            w, wl = cb.sample_classes(x, u, top_p=0.95)
            return v, i, s, loss, grad, j, lp, w, wl

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for seed in range(4):
            y, _, r = case(rows, n, torch.bfloat16, 50 + seed)
            x.copy_(y)
            u.copy_(r)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, step()):
                assert torch.equal(a, b), (rows, n, seed)


def check_no_rows():
    x = torch.empty(0, 7, device="cuda")
    v, i, s = cb.top_classes(x, 3)
    assert v.shape == (0, 3) and i.shape == (0, 3) and s.shape == (0,)
    loss, grad = cb.distill_gradients(x, v, i, top_lse=s)
    assert loss.shape == (0,) and grad.shape == (0, 7)
    j, lp = cb.sample_classes(x, torch.empty(0, device="cuda", dtype=torch.float64))
    assert j.shape == (0,) and lp.shape == (0,)


def check_far_rows():
    """Offsets past 32 bits: the last rows of a matrix of more than 2^32 elements."""
    rows, n = 70001, 65536
    x = torch.zeros(rows, n, dtype=torch.float16, device="cuda")
    at = torch.arange(rows, device="cuda") * 7919 % n
    x[torch.arange(rows, device="cuda"), at] = 20.0
    v, i, s = cb.top_classes(x, 1)
    assert torch.equal(i[:, 0].long(), at) and bool((v == 20).all())
    j, lp = cb.sample_classes(x, torch.full((rows,), 0.5, device="cuda", dtype=torch.float64), top_p=0.5)
    assert torch.equal(j.long(), at)
    loss, grad = cb.distill_gradients(x, v, i)
    assert bool((loss < 1e-3).all()) and bool((grad[-1] != 0).any()) and grad[-1].abs().max().item() < 1e-3


def check_refusals():
    x, _, u = case(4, 100, torch.float32, 6)
    v, i, s = cb.top_classes(x, 5)

    def refuses(error, f, *a, **kw):
        try:
            f(*a, **kw)
        except error:
            return
        raise AssertionError((f.__name__, a and getattr(a[0], "shape", a[0]), kw))

    refuses(ValueError, cb.top_classes, x.cpu(), 5)
    refuses(ValueError, cb.top_classes, x.double(), 5)
    refuses(ValueError, cb.top_classes, x[0], 5)
    refuses(cb.CbhError, cb.top_classes, x, 0)
    refuses(cb.CbhError, cb.top_classes, x, 101)
    refuses(cb.CbhError, cb.top_classes, x, 5, temperature=0.0)
    refuses(cb.CbhError, cb.top_classes, x[:, :0], 1)
    refuses(ValueError, cb.distill_gradients, x, v, i.long())
    refuses(ValueError, cb.distill_gradients, x, v[:3], i[:3])
    refuses(ValueError, cb.distill_gradients, x, v, i, top_lse=s[:2])
    refuses(ValueError, cb.distill_gradients, x, v, i, weight=s.cpu())
    refuses(cb.CbhError, cb.distill_gradients, x, v, i, temperature=float("nan"))
    refuses(ValueError, cb.sample_classes, x, u.float())
    refuses(ValueError, cb.sample_classes, x, u, allowed=torch.zeros(4, 3, dtype=torch.int32, device="cuda"))
    refuses(ValueError, cb.sample_classes, x, u, top_k=torch.zeros(4, device="cuda"))


def check_example():
    """The example trains a teacher, distils it and draws answers."""
    from examples import distill_classes
    losses, agree, drawn = distill_classes.main(rows=4000, steps=40)
    assert losses[-1] < 0.5 * losses[0] and agree > 0.5 and drawn.shape == (4000,)
    assert 0 <= int(drawn.min()) and int(drawn.max()) < 10


def check_split_settings():
    """Settings a row and one setting for all rows draw the same, over more rows than one pass of the long path takes."""
    x, _, u = case(700, 9001, torch.bfloat16, 8)
    full = torch.full((700,), 1.0, device="cuda")
    for k, p in ((0, 1.0), (0, 0.875), (40, 0.875), (3000, 1.0)):
        one = cb.sample_classes(x, u, top_k=k, top_p=p)
        row = cb.sample_classes(x, u, temperature=full, top_k=(full * k).int(), top_p=full * p, min_p=full * 0)
        for a, b in zip(one, row):
            assert torch.equal(a, b), (k, p)


if __name__ == "__main__":
    for name, f in list(globals().items()):
        if name.startswith("check_"):
            print(name, flush=True)
            f()
            torch.cuda.synchronize()
    print("all checks passed")
