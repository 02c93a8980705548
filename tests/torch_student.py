"""Log probabilities, looked-up rows, their gradients and AdamW over torch tensors: run by tests/test_gpu_student.py in a
process of its own, or by hand (python tests/torch_student.py, on a GPU)."""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import catboost_rs_amd as cb  # noqa: E402
from tests import student_oracle as S  # noqa: E402

DEVICE = "cuda"


def scores(rows, n, dtype, seed=0, spread=2.0):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    x = (torch.randn(rows, n, generator=g, device=DEVICE) * spread).to(dtype)
    return x, torch.randint(-1, n, (rows, 2), generator=g, device=DEVICE).int()


def check_types_and_layouts():
    for dtype, half in ((torch.float32, 2.0 ** -24), (torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -8)):
        for rows, n in ((4, 1000), (257, 10), (3, 40001)):
            x, given = scores(rows, n, dtype, n)
            h, c = x.double().cpu().numpy(), given.cpu().numpy()
            for y in (x, x.t().contiguous().t(), torch.nn.functional.pad(x, (3, 4))[:, 3:3 + n]):
                got = cb.class_logprobs(y, given, temperature=2.0, k=3)
                lp, ent, st, top, index = S.logprobs(h, c, 2.0, 3)
                tol = (n / 64 + 40) * 2.0 ** -23
                assert np.array_equal(got.top_index.cpu().numpy(), index)
                for a, b in ((got.logprob, lp), (got.entropy, ent), (got.stats, st), (got.top_logprob, top)):
                    assert np.abs(a.cpu().numpy() - b).max() <= tol * 8
                # one class a row, and none
                one = cb.class_logprobs(y, given[:, 0], temperature=2.0)
                assert one.logprob.shape == (rows,) and torch.equal(one.logprob, got.logprob[:, 0])
                assert one.top_index is None and one.top_logprob is None
                assert cb.class_logprobs(y, temperature=2.0).logprob is None
                g = torch.ones_like(got.logprob)
                grad = cb.logprob_gradients(y, given, g, got.stats, entropy_grad=got.entropy, temperature=2.0)
                assert grad.dtype == dtype and grad.shape == y.shape
                want, size = S.logprob_gradients(h, c, np.ones(c.shape), ent, 2.0)
                assert (np.abs(grad.double().cpu().numpy() - want) <= size * 80 * 2.0 ** -23 + np.abs(want) * half * 1.01 + 2.0 ** -25).all()


def check_a_draws_own_log_probability():
    """What sample_classes says of its draw over allowed classes is what class_logprobs says of it."""
    x, _ = scores(300, 5000, torch.bfloat16, 2)
    g = torch.Generator(device=DEVICE).manual_seed(1)
    allowed = torch.randint(-2**31, 2**31, (300, 157), generator=g, device=DEVICE).int()
    u = torch.rand(300, generator=g, device=DEVICE, dtype=torch.float64)
    for mask in (None, allowed, allowed[:1]):
        j, lp = cb.sample_classes(x, u, temperature=0.8, top_p=0.9, allowed=mask)
        again = cb.class_logprobs(x, j, temperature=0.8, allowed=mask)
        assert (again.logprob - lp).abs().max().item() < 1e-4


def check_lookup():
    g = torch.Generator(device=DEVICE).manual_seed(3)
    table = torch.randn(500, 24, generator=g, device=DEVICE)
    index = torch.randint(-1, 500, (70, 6), generator=g, device=DEVICE).int()
    want = torch.where((index >= 0)[:, :, None], table.double()[index.long().clamp(min=0)], 0.0).sum(1) * 0.5
    for t in (table, table.t().contiguous().t(), table[:, None].expand(-1, 3, -1)[:, 1]):
        assert (cb.lookup_rows(t, index, scale=0.5) - want).abs().max().item() < 1e-5
    assert torch.equal(cb.lookup_rows(table, index[:, 0].clamp(min=0)), table[index[:, 0].long().clamp(min=0)])
    # the gradient, of a sum over all (an expanded one among them)
    up = torch.randn(70, 24, generator=g, device=DEVICE)
    for u in (up, up.t().contiguous().t(), torch.ones(1, 1, device=DEVICE).expand(70, 24)):
        leaf = table.double().requires_grad_()
        rows = torch.where((index >= 0)[:, :, None], leaf[index.long().clamp(min=0)], 0.0).sum(1) * 0.5
        rows.backward(u.double())
        got = cb.lookup_gradients(u, index, 500, scale=0.5)
        assert (got - leaf.grad).abs().max().item() < 1e-5
    half = cb.lookup_gradients(up.half(), index, 500)
    assert half.dtype == torch.float16
    assert cb.lookup_gradients(up.half(), index, 500, dtype=torch.float32).dtype == torch.float32


def check_adamw():
    """A handle over tensors of several types: the same steps as the plain form's, through .grad and lists, with copies."""
    for state in ("f32", "f8"):
        g = torch.Generator(device=DEVICE).manual_seed(4)
        params = [torch.randn(s, generator=g, device=DEVICE) for s in ((30, 7), (1000,), (1,), (0, 3))]
        params.append(torch.randn(11, 5, generator=g, device=DEVICE).bfloat16())
        want = [p.double().cpu().numpy().reshape(-1) for p in params]
        m, v = [np.zeros_like(w) for w in want], [np.zeros_like(w) for w in want]
        copies = [torch.empty_like(params[0], dtype=torch.bfloat16), None, None, None, None]
        opt = cb.AdamW(params, lr=0.01, state=state, copies=copies, seed=3)
        for n in range(1, 4):
            grads = [torch.randn(p.shape, generator=g, device=DEVICE) for p in params]
            grads[1] = grads[1].half()
            grads[0] = grads[0].t().contiguous().t()
            if n == 2:
                grads[2] = None
            if n == 3:
                for p, q in zip(params, grads):
                    p.grad = q.to(p.dtype)
                opt.step()
                grads = [p.grad for p in params]
            else:
                opt.step(grads)
            for i, q in enumerate(grads):
                if q is not None:
                    want[i], m[i], v[i] = S.adamw(want[i], q.double().cpu().numpy().reshape(-1), m[i], v[i], n, lr=0.01)
        assert opt.steps == 3
        for i, (p, w) in enumerate(zip(params, want)):
            # f32 states: rounding; 8 bits: each step goes off by a sixteenth of its size at most, twice over
            tol = 1e-6 if state == "f32" else 0.03 * 0.5
            tol += 0.0 if p.dtype == torch.float32 else 3 * 2.0 ** -8 * 4
            assert not w.size or np.abs(p.double().cpu().numpy().reshape(-1) - w).max() < tol, (state, i)
        assert torch.equal(copies[0], params[0].bfloat16())
        # the states of one handle go on in another
        more = dict(exp_avg=opt.exp_avg, exp_avg_sq=opt.exp_avg_sq, exp_avg_scale=opt.exp_avg_scale, exp_avg_sq_scale=opt.exp_avg_sq_scale)
        again = cb.AdamW([p.clone() for p in params], lr=0.01, state=state, steps=3, seed=3,
                         **{k: None if a is None else [x.clone() for x in a] for k, a in more.items()})
        opt.step(grads)
        again.step(grads)
        assert all(torch.equal(a, b) for a, b in zip(opt.params, again.params))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(opt.exp_avg_sq, again.exp_avg_sq))


def check_steps_on_the_device():
    """A step counter and a rate on the GPU give the steps of a number, and a step held back is not counted."""
    for state in ("f32", "f8"):
        g = torch.Generator(device=DEVICE).manual_seed(5)
        a = [torch.randn(777, generator=g, device=DEVICE)]
        b = [a[0].clone()]
        one = cb.AdamW(a, state=state, seed=1)
        two = cb.AdamW(b, state=state, seed=1, steps=torch.zeros(1, dtype=torch.int64, device=DEVICE))
        rate = torch.full((1,), 0.5, device=DEVICE)
        skip = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        for i in range(5):
            grad = torch.randn(777, generator=g, device=DEVICE)
            skip.fill_(i == 2)
            two.step([grad], lr=rate, skip=skip)
            if i != 2:
                one.step([grad], lr=0.5)
        assert two.steps.item() == 4 and one.steps == 4 and torch.equal(a[0], b[0])


def everything(x, given, table, index, opt):
    """A training step of all of them: rows looked up are scores, beside x; their loss, its gradient, the table's, its
    update."""
    y = (x.float() + cb.lookup_rows(table, index, 0.5).float()).to(x.dtype)
    got = cb.class_logprobs(y, given, k=3)
    g = -torch.ones_like(got.logprob) / len(given)
    grad = cb.logprob_gradients(y, given, g, got.stats, entropy_grad=torch.full_like(got.entropy, -0.01))
    tg = cb.lookup_gradients(grad, index, table.shape[0], 0.5, dtype=torch.float32)
    if opt is not None:
        opt.step([tg])
    return (*got, grad, tg)


def inputs(rows, n, seed, many=3):
    x, given = scores(rows, n, torch.bfloat16, seed)
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return x, given, torch.randint(-1, 300, (rows, many), generator=g, device=DEVICE).int()


def check_other_streams():
    x, given, index = inputs(64, 5003, 6)
    table = torch.randn(300, 5003, device=DEVICE)
    want = everything(x, given, table, index, None)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = everything(x * 1.0, given, table, index, None)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def check_graph_replays():
    """Captured once with the optimizer's step, replayed with new inputs and eager work between the replays."""
    for rows, n in ((2, 70001), (40, 2000), (300, 10), (700, 33)):
        for state in ("f32", "f8"):
            x, given, index = inputs(rows, n, 7)
            tables = [torch.randn(300, n, generator=torch.Generator(device=DEVICE).manual_seed(8), device=DEVICE) for _ in range(2)]
            opts = [cb.AdamW([t], state=state, steps=torch.zeros(1, dtype=torch.int64, device=DEVICE)) for t in tables]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                everything(x, given, tables[0], index, opts[0])
            torch.cuda.current_stream().wait_stream(side)
            everything(x, given, tables[1], index, opts[1])
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = everything(x, given, tables[0], index, opts[0])
            for seed in range(4):
                for a, b in zip((x, given, index), inputs(rows, n, 50 + seed)):
                    a.copy_(b)
                graph.replay()
                torch.cuda.synchronize()
                for a, b in zip(out, everything(x, given, tables[1], index, opts[1])):
                    assert torch.equal(a, b), (rows, n, seed, state)
                assert torch.equal(*tables), (rows, n, seed, state)
            assert opts[0].steps.item() == 5


def check_graphs_of_tables():
    """Every way of the sort, and the tables held in LDS beyond what a launch has without asking, captured and replayed."""
    g = torch.Generator(device=DEVICE).manual_seed(11)
    for rows, many, entries, dim in ((300, 1, 50, 9), (900, 3, 5000, 30), (30000, 1, 300, 16), (20000, 2, 90000, 8), (8000, 40, 1280, 64),
                                     (33000, 40, 1280, 64)):
        table, up = torch.randn(entries, dim, generator=g, device=DEVICE), torch.randn(rows, dim, generator=g, device=DEVICE)
        index = torch.randint(-1, entries, (rows, many), generator=g, device=DEVICE).int()

        def step():
            return cb.lookup_rows(table, index, 0.5), cb.lookup_gradients(up, index, entries)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        with torch.cuda.graph(other):
            out2 = step()
        for seed in range(3):
            for x in (table, up):
                x.copy_(torch.randn(x.shape, generator=g, device=DEVICE))
            index.copy_(torch.randint(-1, entries, (rows, many), generator=g, device=DEVICE))
            graph.replay()
            other.replay()
            torch.cuda.synchronize()
            for a, b, c in zip(out, out2, step()):
                assert torch.equal(a, c) and torch.equal(b, c), (rows, many, entries, seed)


def check_weights_that_move():
    """A weight whose memory is replaced between steps is found again; one that changes its type or shape is refused."""
    p = torch.nn.Parameter(torch.ones(300, device=DEVICE))
    opt = cb.AdamW([p], lr=0.5, weight_decay=0.0)
    grad = torch.ones(300, device=DEVICE)
    opt.step([grad])
    old = p.data
    p.data = p.data.clone()
    before = old.clone()
    opt.step([grad])
    assert torch.equal(old, before) and not torch.equal(p.data, before)
    for bad in (p.data.half(), p.data[:200].clone(), p.data.cpu()):
        keep, p.data = p.data, bad
        try:
            opt.step([torch.ones_like(bad, device=DEVICE)] if bad.numel() != 300 else [grad])
        except ValueError:
            p.data = keep
            continue
        raise AssertionError(bad.dtype)
    opt.step([grad])
    assert opt.steps == 3


def check_no_rows():
    x, i = torch.empty(0, 7, device=DEVICE), torch.empty(0, 2, device=DEVICE, dtype=torch.int32)
    got = cb.class_logprobs(x, i, k=3)
    assert got.logprob.shape == (0, 2) and got.stats.shape == (0, 3) and got.top_index.shape == (0, 3)
    assert cb.logprob_gradients(x, i, got.logprob, got.stats).shape == (0, 7)
    table = torch.randn(5, 7, device=DEVICE)
    assert cb.lookup_rows(table, i).shape == (0, 7)
    grad = cb.lookup_gradients(x, i, 5)
    assert grad.shape == (5, 7) and bool((grad == 0).all())
    cb.AdamW([]).step([])


def check_steps_that_are_refused():
    """Nothing of a step that is refused is done: neither weights nor a counter on the GPU."""
    p, grad = torch.ones(20, 20, device=DEVICE), torch.ones(20, 20, device=DEVICE)
    for skip in (None, torch.zeros(1, dtype=torch.int32, device=DEVICE), torch.ones(1, dtype=torch.int32, device=DEVICE)):
        opt = cb.AdamW([p], steps=torch.full((1,), 4, dtype=torch.int64, device=DEVICE))
        tries = [(cb.CbhError, lambda: opt.step([grad], lr=float("nan"), skip=skip))]
        good = opt.steps
        for steps in (good.cpu(), good.int(), good.repeat(2)):
            tries.append((ValueError, lambda steps=steps: (setattr(opt, "steps", steps), opt.step([grad], skip=skip))))
        whole = p.data
        tries.append((ValueError, lambda: (setattr(opt, "steps", good), setattr(p, "data", whole.t()), opt.step([grad], skip=skip))))
        for error, f in tries:
            try:
                f()
            except error:
                pass
            else:
                raise AssertionError("a step was not refused")
        p.data = whole
        assert good.item() == 4 and bool((p == 1).all()) and bool((opt.exp_avg[0] == 0).all())


def check_far_rows():
    """Offsets past 32 bits: the last rows of matrices of more than 2^32 elements."""
    rows, n = 70001, 65536
    x = torch.zeros(rows, n, dtype=torch.float16, device=DEVICE)
    at = torch.arange(rows, device=DEVICE) * 7919 % n
    x[torch.arange(rows, device=DEVICE), at] = 20.0
    got = cb.class_logprobs(x, at.int(), k=1)
    assert torch.equal(got.top_index[:, 0].long(), at) and got.logprob.abs().max().item() < 1e-3
    grad = cb.logprob_gradients(x, at.int(), torch.full((rows,), 64.0, device=DEVICE), got.stats)
    want = 64 * (1 - torch.exp(got.logprob.double()))
    assert (grad.gather(1, at[:, None])[:, 0].double() - want).abs().max().item() < 1e-4
    assert bool((grad[-1] != 0).any())
    del grad
    # (entries of a table of more than 2^32 elements, and its gradient)
    index = torch.tensor([rows - 1, 0, rows - 1, 65537], dtype=torch.int32, device=DEVICE)
    out = cb.lookup_rows(x, index)
    assert torch.equal(out, x[index.long()])
    tg = cb.lookup_gradients(out, index, rows)
    assert torch.equal(tg[-1], out[0] + out[2]) and torch.equal(tg[65537], out[3])
    assert torch.count_nonzero(tg.sum(1, dtype=torch.float32)).item() == 3


def check_large_optimizer():
    """A tensor of more than 2^32 values in 16 bits with states in 8."""
    n = (1 << 32) + 1000
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEVICE)
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device=DEVICE)
    g[-1] = -0.5
    opt = cb.AdamW([p], lr=0.125, weight_decay=0.0, state="f8")
    opt.step([g])
    assert torch.equal(p[:5], p[-7:-2]) and abs(p[0].item() + 0.125) < 1e-3 and abs(p[-1].item() - 0.125) < 1e-3
    assert p[1 << 32].item() == p[0].item() and bool((p[::1 << 20] == p[0]).all())


def check_refusals():
    x, given = scores(4, 100, torch.float32, 9)
    got = cb.class_logprobs(x, given)
    table, index = torch.randn(9, 4, device=DEVICE), torch.zeros(4, 2, dtype=torch.int32, device=DEVICE)

    def refuses(error, f, *a, **kw):
        try:
            f(*a, **kw)
        except error:
            return
        raise AssertionError((f, a and getattr(a[0], "shape", a[0]), kw))

    refuses(ValueError, cb.class_logprobs, x.cpu(), given)
    refuses(ValueError, cb.class_logprobs, x.double(), given)
    refuses(ValueError, cb.class_logprobs, x[0], given)
    refuses(ValueError, cb.class_logprobs, x, given.long())
    refuses(ValueError, cb.class_logprobs, x, given[:3])
    refuses(ValueError, cb.class_logprobs, x, given.cpu())
    refuses(ValueError, cb.class_logprobs, x, given, allowed=torch.zeros(4, 3, dtype=torch.int32, device=DEVICE))
    refuses(cb.CbhError, cb.class_logprobs, x, given, k=101)
    refuses(cb.CbhError, cb.class_logprobs, x, given, k=-1)
    refuses(cb.CbhError, cb.class_logprobs, x, given, temperature=0.0)
    refuses(cb.CbhError, cb.class_logprobs, x[:, :0], given)
    refuses(cb.CbhError, cb.class_logprobs, x, torch.zeros(4, 1025, dtype=torch.int32, device=DEVICE))
    refuses(ValueError, cb.logprob_gradients, x, given, got.logprob[:, 0], got.stats)
    refuses(ValueError, cb.logprob_gradients, x, given, got.logprob, got.stats[:, :2])
    refuses(ValueError, cb.logprob_gradients, x, given, got.logprob, got.stats, entropy_grad=got.logprob)
    refuses(ValueError, cb.logprob_gradients, x, None, got.logprob, got.stats)
    refuses(cb.CbhError, cb.logprob_gradients, x, given, got.logprob, got.stats, temperature=float("nan"))
    refuses(ValueError, cb.lookup_rows, table, index.long())
    refuses(ValueError, cb.lookup_rows, table.double(), index)
    refuses(ValueError, cb.lookup_rows, table[0], index)
    refuses(ValueError, cb.lookup_rows, table, index[None])
    refuses(cb.CbhError, cb.lookup_rows, table, index[:, :0])
    refuses(cb.CbhError, cb.lookup_rows, table[:0], index)
    refuses(cb.CbhError, cb.lookup_rows, table, index, scale=float("inf"))
    refuses(ValueError, cb.lookup_gradients, table, index, 9)          # rows of index and gradient differ
    refuses(ValueError, cb.lookup_gradients, table[:4], index, 9, dtype=torch.float64)
    refuses(cb.CbhError, cb.lookup_gradients, table[:4], index, 0)
    refuses(cb.CbhError, cb.lookup_gradients, table[:4], index, 1 << 31)
    refuses(ValueError, cb.AdamW, [table.double()])
    refuses(ValueError, cb.AdamW, [table.t()])
    refuses(ValueError, cb.AdamW, [table.cpu()])
    refuses(ValueError, cb.AdamW, [table], state="8")
    refuses(ValueError, cb.AdamW, [table], steps=-1)
    refuses(ValueError, cb.AdamW, [table], exp_avg=[table[:3]])
    refuses(ValueError, cb.AdamW, [table], exp_avg_scale=[table])
    refuses(ValueError, cb.AdamW, [table], copies=[table[:3]])
    opt = cb.AdamW([table])
    refuses(ValueError, opt.step, [])
    refuses(ValueError, opt.step, [table[:3]])
    refuses(ValueError, opt.step, [table.double()])
    refuses(ValueError, opt.step, [table], grad_scale=table)
    refuses(ValueError, opt.step, [table], skip=torch.zeros(1, device=DEVICE))
    refuses(ValueError, opt.step, [table], grad_scale=0.5)
    refuses(ValueError, opt.step, [table], skip=1)
    refuses(ValueError, opt.step, [table.cpu()])
    refuses(cb.CbhError, opt.step, [table])   # (the weight as its own gradient)
    refuses(ValueError, opt.step, [[1.0]])
    refuses(TypeError, opt.step, table[0, 0])
    refuses(cb.CbhError, opt.step, [table], lr=float("nan"))
    refuses(cb.CbhError, cb.AdamW([table, table]).step, [table, table])
    assert opt.steps == 0


def check_example():
    """The additive student runs, and its gradient is that of its loss (a plain one in 64 bits, by autograd)."""
    from examples import additive_student as A
    losses, held = A.main(rows=2000, steps=3)
    assert len(losses) == 3 and all(np.isfinite(losses)) and bool(torch.isfinite(held).all())
    x, y = A.table(500, 5, 7)
    index, entries = A.binned(x, 9)
    held = torch.randn(entries, 7, generator=torch.Generator(device=DEVICE).manual_seed(9), device=DEVICE)
    index, label = torch.from_numpy(index).cuda(), torch.from_numpy(y.astype(np.int32)).cuda()
    loss, grad = A.loss_and_gradient(held, index, label)
    leaf = held.double().requires_grad_()
    logp = torch.log_softmax(leaf[index.long()].sum(1), 1)
    plain = -(logp.gather(1, label.long()[:, None]).mean() - 0.01 * (logp.exp() * logp).sum(1).mean())
    plain.backward()
    # scores are sums of five f32 values of up to 4; a gradient is a sum of up to 500 of them, each a p to 40 roundings, over 500 rows
    assert abs(loss.item() - plain.item()) < 1e-5
    assert (grad - leaf.grad).abs().max().item() < 500 / 500 * 60 * 2.0 ** -23


if __name__ == "__main__":
    for name, f in list(globals().items()):
        if name.startswith("check_"):
            print(name, flush=True)
            f()
            torch.cuda.synchronize()
            torch.cuda.empty_cache()
    print("all checks passed")
