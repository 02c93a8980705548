"""AdamW over torch tensors where a program does the unusual: run by tests/test_gpu_student_edges.py in a process of its
own, or by hand (python tests/torch_student_edges.py, on a GPU)."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import catboost_rs_amd as cb  # noqa: E402

DEVICE = "cuda"


def refuses(error, f):
    try:
        f()
    except error:
        return
    raise AssertionError(f"no {error}")


def check_version_counters():
    """What a step writes counts as written for autograd: a graph that holds the old weights is refused in its backward
    pass, as after torch's own updates."""
    for state in ("f32", "f8"):
        p, q = (torch.nn.Parameter(torch.ones(300, device=DEVICE)) for _ in range(2))
        copy = torch.zeros(300, device=DEVICE, dtype=torch.bfloat16, requires_grad=True)
        opt = cb.AdamW([p, q], state=state, copies=[copy, None])
        grad = torch.ones(300, device=DEVICE)

        def written(i):
            names = ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if state == "f8" else ())
            return [(p, q)[i]] + [getattr(opt, name)[i] for name in names] + ([copy] if i == 0 else [])

        old, other = (p * p * p).sum(), (q * q).sum()
        low = (copy * copy).sum()
        before = [[t._version for t in written(i)] for i in (0, 1)]
        opt.step([grad, None])
        assert all(t._version > v for t, v in zip(written(0), before[0])), state
        assert [t._version for t in written(1)] == before[1], state   # (no gradient: nothing of it is written)
        refuses(RuntimeError, old.backward)
        refuses(RuntimeError, low.backward)
        other.backward()
        assert bool((q.grad == 2).all())
        # a step that is refused writes nothing
        before = [t._version for i in (0, 1) for t in written(i)]
        refuses(cb.CbhError, lambda: opt.step([grad, grad], lr=float("nan")))
        assert [t._version for i in (0, 1) for t in written(i)] == before
        # weights of one block of memory
        flat = torch.ones(600, device=DEVICE)
        parts = [flat[:300], flat[300:]]
        opt = cb.AdamW(parts, state=state)
        leaf = torch.ones(600, device=DEVICE, requires_grad=True)
        loss = (leaf * flat).sum()
        opt.step([grad, grad])
        refuses(RuntimeError, loss.backward)


def check_inference_tensors():
    """Tensors made in inference mode, which have no such counter."""
    with torch.inference_mode():
        p, grad = torch.ones(30, device=DEVICE), torch.ones(30, device=DEVICE)
        opt = cb.AdamW([p], lr=0.5, weight_decay=0.0)
        opt.step([grad])
    opt.step([grad])
    assert opt.steps == 2 and bool((p < 0.5).all())


def check_a_captured_step_counts_on_the_device():
    """A number of steps would be a constant of the graph: refused, and nothing is changed."""
    p, grad = torch.ones(30, device=DEVICE), torch.ones(30, device=DEVICE)
    opt = cb.AdamW([p])
    opt.step([grad])
    before = p.clone()
    graph = torch.cuda.CUDAGraph()

    def capture():
        with torch.cuda.graph(graph):
            opt.step([grad])

    refuses(RuntimeError, capture)
    torch.cuda.synchronize()
    assert opt.steps == 1 and torch.equal(p, before)
    opt.step([grad])
    assert opt.steps == 2 and not torch.equal(p, before)


if __name__ == "__main__":
    for name, f in list(globals().items()):
        if name.startswith("check_"):
            print(name, flush=True)
            f()
            torch.cuda.synchronize()
    print("all checks passed")
