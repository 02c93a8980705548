"""The operators on class scores as cases that can be timed and compared: the top classes of a
row with its log-sum-exp, distillation from a teacher's top classes (loss and gradient), and
classes drawn from given random numbers.

Scores are [rows][classes].  Three orders of memory occur: ``rows`` (a row's classes next to
each other), ``padded`` (rows further apart than their classes) and ``classes`` (a class's rows
next to each other: the layout of a session's approximant and of ``apply_oblivious``).  Inputs
are synthetic, made from the seed alone: normal scores whose spread differs from row to row, so
that some rows are sure of an answer and others are not.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one small request to a model with a thousand classes: the launches are the whole cost
        dict(name="top request", kind="top", rows=4, classes=1000, type="f32", order="rows", k=5, temperature=1.0),
        # rows of odd length, so that none but the first starts at an aligned address; a warm teacher
        dict(name="top ragged", kind="top", rows=777, classes=50021, type="f32", order="rows", k=20, temperature=2.0),
        # a teacher's pass over a batch: what is kept of its scores for a student
        dict(name="top teacher", kind="top", rows=4096, classes=65536, type="bf16", order="rows", k=64, temperature=1.0),
        # a handful of rows: the gradient of one small step
        dict(name="distill request", kind="distill", rows=8, classes=32768, type="f16", order="rows", k=16,
             temperature=1.0, rest=True, weights=False),
        # ten classes and a million rows, class-major with weights: the scores of a boosted model in training
        dict(name="distill boosted", kind="distill", rows=1_000_000, classes=10, type="f32", order="classes", k=3,
             temperature=1.5, rest=True, weights=True),
        # a teacher that gave its listed scores alone, odd rows in a wider buffer
        dict(name="distill listed", kind="distill", rows=1500, classes=100003, type="f32", order="padded", k=20,
             temperature=2.0, rest=False, weights=True),
        # a large batch over many classes
        dict(name="distill batch", kind="distill", rows=4096, classes=65536, type="bf16", order="rows", k=64,
             temperature=1.0, rest=True, weights=False),
        # one answer being drawn, class by class of a long list
        dict(name="sample request", kind="sample", rows=1, classes=131072, type="bf16", order="rows", how="both",
             spread=2.5, mask="none"),
        # a served batch: each row has settings of its own, and a list of what it may answer
        dict(name="sample batch", kind="sample", rows=256, classes=131072, type="f32", order="rows", how="mixed",
             spread=2.5, mask="rows"),
        # draws from the whole distribution, odd rows
        dict(name="sample whole", kind="sample", rows=512, classes=65537, type="bf16", order="rows", how="whole",
             spread=2.0, mask="none"),
        # unsure rows: the nucleus holds tens of thousands of classes
        dict(name="sample unsure", kind="sample", rows=64, classes=200001, type="f16", order="padded", how="nucleus",
             spread=0.7, mask="shared"),
        # answers of a boosted model for a million rows of a generated table
        dict(name="sample boosted", kind="sample", rows=1_000_000, classes=10, type="f32", order="classes",
             how="nucleus", spread=1.5, mask="none"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["top", "distill", "distill", "sample", "sample"])
    most = 30_000_000 if kind == "sample" else 200_000_000
    classes = _log(rng, 2, 40) if rng.random() < 0.3 else _log(rng, 40, 260_000)
    rows = _log(rng, 1, min(1_000_000, most // classes))
    order = rng.choice(["rows", "classes"]) if classes <= 40 else rng.choice(["rows", "rows", "padded"])
    case = dict(kind=kind, rows=rows, classes=classes, type=rng.choice(["f32", "f16", "bf16"]), order=order)
    if kind == "sample":
        return dict(case, how=rng.choice(["mixed", "mixed", "both", "nucleus", "whole", "greedy"]),
                    spread=round(rng.uniform(0.5, 4.0), 2), mask=rng.choice(["none", "none", "shared", "rows"]))
    k = min(classes, _log(rng, 1, 256))
    case.update(k=k, temperature=rng.choice([1.0, 1.0, 1.5, 2.0, 4.0]))
    if kind == "distill":
        case.update(rest=rng.random() < 0.7, weights=rng.random() < 0.5)
    return case


# ---- inputs -------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1_000_003 + 29)
    return g


def _laid(x, case):
    """`x` [rows][classes] f32 in the case's type and order of memory."""
    rows, classes = x.shape
    x = x.to(_TYPES[case["type"]])
    if case["order"] == "classes":
        return x.t().contiguous().t()
    if case["order"] == "padded":
        wide = torch.zeros(rows, classes + 13, dtype=x.dtype, device="cuda")
        wide[:, 5:5 + classes] = x
        return wide[:, 5:5 + classes]
    return x


def _scores(case, g, spread):
    rows, classes = case["rows"], case["classes"]
    sigma = spread * (0.5 + torch.rand(rows, 1, generator=g, device="cuda"))
    return torch.randn(rows, classes, generator=g, device="cuda") * sigma


def prepare(case, seed):
    g = _generator(seed)
    rows, classes = case["rows"], case["classes"]
    state = dict(case)
    if case["kind"] == "top":
        state["scores"] = _laid(_scores(case, g, 2.5), case)
    elif case["kind"] == "distill":
        teacher = _scores(case, g, 2.5)
        state["scores"] = _laid(teacher * 0.7 + torch.randn(rows, classes, generator=g, device="cuda"), case)
        top = torch.topk(teacher, case["k"], dim=1)
        state["top_scores"], state["top_index"] = top.values, top.indices.int()
        lse = torch.empty(rows, device="cuda")
        step = max(1, 50_000_000 // classes)
        for a in range(0, rows, step):   # by blocks of rows, for the memory
            lse[a:a + step] = torch.logsumexp(teacher[a:a + step].double() / case["temperature"], 1).float()
        state["top_lse"] = lse if case["rest"] else None
        state["weight"] = None
        if case["weights"]:   # a tenth of the rows is left out
            w = torch.rand(rows, generator=g, device="cuda") + 0.5
            state["weight"] = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.1, torch.zeros_like(w), w)
    else:
        state["scores"] = _laid(_scores(case, g, case["spread"]), case)
        state["uniform"] = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
        how = case["how"]
        state.update(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, allowed=None)
        if how == "both":
            state.update(temperature=0.8, top_k=min(50, classes), top_p=0.95)
        elif how == "nucleus":
            state.update(top_p=0.9)
        elif how == "greedy":
            state.update(temperature=0.0)
        elif how == "mixed":
            def pick(values, dtype):
                values = torch.tensor(values, dtype=dtype, device="cuda")
                return values[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]
            state.update(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3], torch.float32),
                         top_k=pick([0, 0, 1, 20, 50, 300, 5000], torch.int32),
                         top_p=pick([1.0, 1.0, 0.95, 0.8, 0.5], torch.float32),
                         min_p=pick([0.0, 0.0, 0.02, 0.1], torch.float32))
        if case["mask"] != "none":
            words = (classes + 31) // 32
            n = rows if case["mask"] == "rows" else 1
            shape = (n, words)
            a = torch.randint(-2**31, 2**31, shape, generator=g, device="cuda")
            b = torch.randint(-2**31, 2**31, shape, generator=g, device="cuda")
            state["allowed"] = (a | b).int()
    return state


# ---- plain forms --------------------------------------------------------------------------
def _plain_top(s):
    x = s["scores"].float()
    values, index = torch.sort(x, dim=1, descending=True, stable=True)   # ties: the lowest class first
    t = x / s["temperature"]
    m = t.amax(1, keepdim=True)
    lse = torch.log(torch.exp(t - m).sum(1)) + m[:, 0]
    k = s["k"]
    return {"values": values[:, :k].contiguous(), "index": index[:, :k].int(), "lse": lse}


def _plain_distill(s):
    x, t = s["scores"], s["temperature"]
    z = x.float() / t
    listed = s["top_index"].long()
    lz = z - z.amax(1, keepdim=True)
    lz = lz - torch.log(torch.exp(lz).sum(1, keepdim=True))
    p = torch.exp(lz)
    u = s["top_scores"].double() / t
    if s["top_lse"] is not None:
        logq = u - s["top_lse"].double()[:, None]
    else:
        logq = u - u.amax(1, keepdim=True)
        logq = logq - torch.log(torch.exp(logq).sum(1, keepdim=True))
    q = torch.exp(logq)
    kl = (q * (logq - lz.gather(1, listed).double())).sum(1)
    if s["top_lse"] is not None and s["k"] < s["classes"]:
        rest = (1 - q.sum(1)).clamp(min=0)
        other = p.scatter(1, listed, 0.0)
        mass = other.sum(1)
        kl = kl + torch.where(rest > 0, rest * (torch.log(rest) - torch.log(mass.double())), torch.zeros_like(rest))
        whole = (q.sum(1) + rest).float()[:, None]
        grad = p * whole - other * (rest.float() / mass)[:, None]
    else:
        grad = p * q.sum(1).float()[:, None]
    grad = grad.scatter_add(1, listed, -q.float())
    if s["weight"] is not None:
        w = s["weight"]
        kl, grad = torch.where(w != 0, kl * w, 0.0), torch.where(w[:, None] != 0, grad * w[:, None], 0.0)
    return {"loss": (kl * t * t).float(), "grad": (grad * t).to(x.dtype)}


def _column(v, dtype):
    return v.to(dtype)[:, None] if isinstance(v, torch.Tensor) else torch.full((1, 1), v, dtype=dtype, device="cuda")


def _plain_sample(s):
    x = s["scores"].double()
    classes = s["classes"]
    if s["allowed"] is not None:
        j = torch.arange(classes, device="cuda")
        bits = (s["allowed"][:, j >> 5] >> (j & 31)) & 1
        x = torch.where(bits != 0, x, float("-inf"))
    t, k = _column(s["temperature"], torch.float64), _column(s["top_k"], torch.int64)
    top_p, min_p = _column(s["top_p"], torch.float64), _column(s["min_p"], torch.float64)
    greedy = t <= 0
    t = torch.where(greedy, 1.0, t)
    m = x.amax(1, keepdim=True)
    w = torch.where(x == m, 1.0, torch.exp((x - m) / t))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    rank = torch.arange(classes, device="cuda")[None]
    keep = ((rank < torch.where((k > 0) & (k < classes), k, classes)) & ~(greedy & (rank > 0))).repeat(
        x.shape[0] if t.shape[0] == k.shape[0] == 1 else 1, 1)
    mass = torch.cumsum(ranked * keep, 1)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
    keep &= (before < top_p * mass[:, -1:]) | (top_p >= 1) | (rank == 0)
    keep &= (ranked >= min_p) | (rank == 0)
    kept = torch.zeros_like(keep).scatter(1, order, keep) & (w > 0)
    mass = torch.cumsum(w * kept, 1)
    last = classes - 1 - torch.argmax(kept.flip(1).int(), 1)
    index = torch.minimum((mass <= s["uniform"][:, None] * mass[:, -1:]).sum(1), last)
    logprob = ((x.gather(1, index[:, None]) - m) / t)[:, 0] - torch.log(w.sum(1))
    logprob = torch.where(greedy.expand(x.shape[0], 1)[:, 0], 0.0, logprob)
    empty = m[:, 0] == float("-inf")   # a row that may answer nothing
    return {"index": torch.where(empty, -1, index).int(), "logprob": torch.where(empty, float("-inf"), logprob).float()}


def run(state):
    kind = state["kind"]
    if own:
        import catboost_rs_amd as cb
        if kind == "top":
            values, index, lse = cb.top_classes(state["scores"], state["k"], temperature=state["temperature"])
            return {"values": values, "index": index, "lse": lse}
        if kind == "distill":
            loss, grad = cb.distill_gradients(state["scores"], state["top_scores"], state["top_index"],
                                              top_lse=state["top_lse"], temperature=state["temperature"],
                                              weight=state["weight"])
            return {"loss": loss, "grad": grad}
        index, logprob = cb.sample_classes(state["scores"], state["uniform"], temperature=state["temperature"],
                                           top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"],
                                           allowed=state["allowed"])
        return {"index": index, "logprob": logprob}
    return {"top": _plain_top, "distill": _plain_distill, "sample": _plain_sample}[kind](state)


def work(case):
    rows, classes, e = case["rows"], case["classes"], _BYTES[case["type"]]
    scores = rows * classes
    if case["kind"] == "top":
        return {"bytes": scores * e + rows * (8 * case["k"] + 4), "flops": 4 * scores}
    if case["kind"] == "distill":
        n = scores * e * 2 + rows * (8 * case["k"] + 4 + 4 * case["rest"] + 4 * case["weights"])
        return {"bytes": n, "flops": 8 * scores}
    words = (classes + 31) // 32 * 4
    n = scores * e + rows * (8 + 8 + (16 if case["how"] == "mixed" else 0))
    n += {"none": 0, "shared": words, "rows": rows * words}[case["mask"]]
    return {"bytes": n, "flops": 6 * scores}


# ---- the definitions, in 64 bits ----------------------------------------------------------
def _exact_top(s, a, b):
    x = s["scores"][a:b].double()
    return {"values": torch.topk(x, s["k"], dim=1).values, "index": None,
            "lse": torch.logsumexp(x / s["temperature"], 1)}


def _exact_distill(s, a, b):
    t = s["temperature"]
    z = s["scores"][a:b].double() / t
    listed = s["top_index"][a:b].long()
    free = torch.ones_like(z, dtype=torch.bool).scatter_(1, listed, False)
    total = torch.logsumexp(z, 1)
    u = s["top_scores"][a:b].double() / t
    base = s["top_lse"][a:b].double() if s["top_lse"] is not None else torch.logsumexp(u, 1)
    q = torch.exp(u - base[:, None])
    held = q.sum(1)
    loss = (torch.xlogy(q, q) - q * (z.gather(1, listed) - total[:, None])).sum(1)
    grad = torch.exp(z - total[:, None])
    if s["top_lse"] is not None and bool(free.any()):
        rest = (1 - held).clamp(min=0)
        others = torch.logsumexp(z.masked_fill(~free, float("-inf")), 1)
        loss += torch.xlogy(rest, rest) - rest * (others - total)
        share = torch.where(free, torch.exp(z - others[:, None]), 0.0)
        grad = grad * (held + rest)[:, None] - rest[:, None] * share
    else:
        grad *= held[:, None]
    grad.scatter_add_(1, listed, -q)
    w = s["weight"][a:b].double() if s["weight"] is not None else torch.ones_like(loss)
    return {"loss": w * loss * t * t, "grad": grad * (w * t)[:, None]}


def _exact_sample(s, a, b):
    x = s["scores"][a:b].double().cpu().numpy()
    rows, classes = x.shape
    if s["allowed"] is not None:
        words = s["allowed"] if s["allowed"].shape[0] == 1 else s["allowed"][a:b]
        bits = np.unpackbits(words.cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :classes]
        x = np.where(bits != 0, x, -np.inf)

    def column(name):
        v = s[name]
        v = v[a:b].double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(rows, float(v))
        return v[:, None]

    t, k, top_p, min_p, u = (column(n) for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
    with np.errstate(divide="ignore", invalid="ignore"):
        best = x.max(1, keepdims=True)
        z = np.where(x == best, 0.0, (x - best) / np.where(t > 0, t, 1.0))
        w = np.exp(z)
        by = np.argsort(-x, axis=1, kind="stable")
        sorted_w = np.take_along_axis(w, by, 1)
        place = np.arange(classes)[None]
        among = place < np.where(t <= 0, 1, np.where(k > 0, k, classes))
        held = np.add.accumulate(np.where(among, sorted_w, 0.0), axis=1)
        ahead = held - np.where(among, sorted_w, 0.0)
        stay = among & ((top_p >= 1) | (ahead < top_p * held[:, -1:])) & (sorted_w >= min_p)
        stay[:, 0] = True
        mask = np.zeros((rows, classes), bool)
        np.put_along_axis(mask, by, stay, 1)
        mask &= w > 0
        held = np.add.accumulate(np.where(mask, w, 0.0), axis=1)
        found = held > u * held[:, -1:]
        found[:, -1] |= ~found.any(1)
        at = found.argmax(1)
        logprob = np.take_along_axis(z, at[:, None], 1)[:, 0] - np.log(w.sum(1))
    logprob = np.where(best[:, 0] == -np.inf, -np.inf, np.where(t[:, 0] <= 0, 0.0, logprob))
    return {"index": None, "logprob": torch.from_numpy(logprob)}


def exact(case, seed):
    s = prepare(case, seed)
    one = {"top": _exact_top, "distill": _exact_distill, "sample": _exact_sample}[case["kind"]]
    step = max(1, (4_000_000 if case["kind"] == "sample" else 100_000_000) // case["classes"])
    parts = [one(s, a, min(case["rows"], a + step)) for a in range(0, case["rows"], step)]
    return {name: None if parts[0][name] is None else torch.cat([p[name] for p in parts]) for name in parts[0]}
