"""AdamW and log probabilities over torch tensors where a program does the unusual: run by tests/test_gpu_student_edges.py in a process of its
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


def check_weights_that_change_in_place():
    """A weight that becomes a shorter or another type's view of its own memory is refused, and nothing is written."""
    whole = torch.ones(300, device=DEVICE)
    p = torch.nn.Parameter(whole)
    opt = cb.AdamW([p], lr=0.5)
    grad = torch.ones(300, device=DEVICE)
    at = p.data_ptr()
    for bad in (whole[:200], whole.view(torch.float16)[:300], whole.view(torch.bfloat16)[:300], whole.view(30, 10)):
        p.data = bad
        assert p.data_ptr() == at
        for g in (grad, torch.ones(bad.shape, device=DEVICE)):
            refuses(ValueError, lambda: opt.step([g]))
    p.data = whole
    assert bool((whole == 1).all()) and opt.steps == 0
    opt.step([grad])
    assert opt.steps == 1 and bool((whole < 1).all())


def check_states_and_copies_that_move():
    """What a state's or a copy's memory became is what the next step goes on with."""
    for state in ("f32", "f8"):
        g = torch.Generator(device=DEVICE).manual_seed(3)
        first = torch.randn(700, generator=g, device=DEVICE)
        a, b = first.clone(), first.clone()
        copy = torch.zeros(700, device=DEVICE, dtype=torch.bfloat16)
        one, two = cb.AdamW([a], state=state, lr=0.1), cb.AdamW([b], state=state, lr=0.1, copies=[copy])
        names = ["exp_avg", "exp_avg_sq"] + (["exp_avg_scale", "exp_avg_sq_scale"] if state == "f8" else [])
        bits = torch.uint8 if state == "f8" else torch.int32

        def step():
            grad = torch.randn(700, generator=g, device=DEVICE)
            one.step([grad])
            two.step([grad])
            assert torch.equal(a, b) and torch.equal(two.copies[0], b.bfloat16())
            for name in names:
                x, y = getattr(one, name)[0], getattr(two, name)[0]
                kind = torch.int32 if x.dtype == torch.float32 else bits
                assert torch.equal(x.view(kind), y.view(kind)), (state, name)

        step()
        for name in names:
            # other memory
            old = getattr(two, name)[0].data
            before = old.clone()
            getattr(two, name)[0].data = old.clone()
            step()
            assert torch.equal(old.view(torch.uint8), before.view(torch.uint8)), (state, name)
            refuses(AttributeError, lambda: getattr(two, name).append(old))   # (the tuples stay)
            refuses(AttributeError, lambda: setattr(two, name, [old]))
            # memory given up for a while
            x = getattr(two, name)[0]
            saved, storage = x.clone(), x.untyped_storage()
            size = storage.size()
            storage.resize_(0)
            refuses(cb.CbhError, lambda: two.step([first]))
            other = torch.full((4000,), 7.0, device=DEVICE)   # (perhaps where it was)
            refuses(cb.CbhError, lambda: two.step([first]))
            assert bool((other == 7).all())
            storage.resize_(size)
            x.copy_(saved)
            step()
            # what does not fit is refused, and put right again
            good = x.data
            for bad in (good[:-1].clone(), good.to(torch.float64), torch.cat([good, good])[::2]):
                x.data = bad
                refuses(ValueError, lambda: two.step([first]))
            x.data = good
            step()
        two.copies[0].data = torch.zeros(700, device=DEVICE, dtype=torch.bfloat16)
        step()
        assert one.steps == two.steps


def check_weights_of_16_bits():
    """Steps of 16-bit weights through the handle, bit for bit the plain implementation's, and far larger than a rounding."""
    import numpy as np

    from tests import class_scores_oracle as O
    from tests import student_oracle as S
    from tests.test_gpu_adamw import expected

    for dtype, kind in ((torch.bfloat16, "bf16"), (torch.float16, "f16")):
        for small in (False, True):
            g = torch.Generator(device=DEVICE).manual_seed(7)
            params = [torch.randn(shape, generator=g, device=DEVICE).to(dtype) for shape in ((300, 3), (1,), (257,))]
            opt = cb.AdamW(params, lr=0.25, state="f8" if small else "f32", seed=11)
            held = [dict(p=p.float().cpu().numpy().reshape(-1), m=np.zeros(p.numel(), np.uint8 if small else np.float32)) for p in params]
            for t in held:
                t["v"] = t["m"].copy()
                t["ms"] = t["vs"] = np.zeros(-(-len(t["p"]) // S.BLOCK), np.float32)
            for n in range(1, 6):
                grads = [torch.randn(p.shape, generator=g, device=DEVICE).to(dtype) for p in params]
                before = [p.clone() for p in params]
                opt.step(grads)
                for i, (t, q, p) in enumerate(zip(held, grads, params)):
                    e = expected(dict(t, g=q.float().cpu().numpy().reshape(-1)), small, seed=11, number=i, step=n, lr=0.25)
                    held[i] = dict(t, **dict(e, p=O.round_to(e["p"], kind)))
                    assert np.array_equal(p.float().cpu().numpy().reshape(-1), held[i]["p"]), (kind, small, n, i)
                assert (params[0] != before[0]).float().mean().item() > 0.9, (kind, small, n)


def check_lists_of_no_classes():
    """Nothing given: the entropy's derivative alone, as with entries that are none; and a step without any gradient."""
    for dtype in (torch.float32, torch.bfloat16):
        for rows, n in ((300, 7), (300, 30), (40, 900), (5, 5000)):
            g = torch.Generator(device=DEVICE).manual_seed(n)
            x = torch.randn(rows, n, generator=g, device=DEVICE).to(dtype)
            none, no = torch.empty(rows, 0, dtype=torch.int32, device=DEVICE), torch.full((rows, 1), -1, dtype=torch.int32, device=DEVICE)
            up, h = torch.empty(rows, 0, device=DEVICE), torch.randn(rows, generator=g, device=DEVICE)
            for y in (x, x.t().contiguous().t()):
                got = cb.class_logprobs(y, none, k=2)
                assert got.logprob.shape == (rows, 0) and torch.equal(got.stats, cb.class_logprobs(y, no, k=2).stats)
                a = cb.logprob_gradients(y, none, up, got.stats, entropy_grad=h)
                b = cb.logprob_gradients(y, no, torch.ones(rows, 1, device=DEVICE), got.stats, entropy_grad=h)
                assert torch.equal(a, b) and bool((a != 0).any())
                assert bool((cb.logprob_gradients(y, none, up, got.stats) == 0).all())
    p = torch.ones(30, device=DEVICE)
    opt = cb.AdamW([p])
    opt.step([None])
    assert opt.steps == 1 and bool((p == 1).all()) and p._version == 0


if __name__ == "__main__":
    for name, f in list(globals().items()):
        if name.startswith("check_"):
            print(name, flush=True)
            f()
            torch.cuda.synchronize()
    print("all checks passed")
