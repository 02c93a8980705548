"""The operators that train and score a student beside a boosted model, as cases that can be timed
and compared: log probabilities of given classes with entropy and alternatives, their gradient,
sums of looked-up rows of a table (bins, leaves, category buckets), the table's gradient, and an
AdamW step over many tensors with states in 32 or 8 bits.

Inputs are synthetic, made from the seed alone.  Scores are [rows][classes] in the three orders of
memory in which they occur: ``rows``, ``padded`` (rows further apart than their classes) and
``classes`` (a class's rows next to each other, as a boosted model gives them).
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_BLOCK = 256   # values of an 8-bit state that share a scale


def listed():
    return [
        # one answer being scored as it is served: its class and five alternatives
        dict(name="logprobs request", kind="logprobs", rows=1, classes=131072, type="bf16", order="rows", given=1, k=5,
             temperature=1.0, mask="none"),
        # answers with several classes each and a list of what may be answered, odd rows in a wider buffer
        dict(name="logprobs ragged", kind="logprobs", rows=777, classes=50021, type="f32", order="padded", given=4, k=20,
             temperature=1.5, mask="shared"),
        # the loss of a large training batch
        dict(name="logprobs batch", kind="logprobs", rows=4096, classes=65536, type="bf16", order="rows", given=1, k=0,
             temperature=1.0, mask="none"),
        # a million rows of a boosted model's scores against their labels
        dict(name="logprobs boosted", kind="logprobs", rows=1_000_000, classes=10, type="f32", order="classes", given=1, k=3,
             temperature=1.0, mask="none"),
        # the gradient of one small step
        dict(name="gradients request", kind="gradients", rows=8, classes=32768, type="f16", order="rows", given=1,
             temperature=1.0, mask="none", entropy=False),
        # the gradient of a large batch, with a reward for entropy
        dict(name="gradients batch", kind="gradients", rows=4096, classes=65536, type="bf16", order="rows", given=1,
             temperature=1.0, mask="none", entropy=True),
        # category buckets of a few rows being answered
        dict(name="lookup request", kind="lookup", rows=32, list=1, entries=50021, dim=256, type="bf16", scale=16.0),
        # the leaves that forty trees of 32 give a large table's rows, summed as vectors
        dict(name="lookup leaves", kind="lookup", rows=200_000, list=40, entries=1280, dim=64, type="f32", scale=0.1),
        # the gradient of those leaves' vectors: few entries, each in many rows
        dict(name="table leaves", kind="table", rows=65536, list=40, entries=1280, dim=64, type="f32", out="f32", scale=0.1),
        # the gradient of category buckets, frequent and rare ones, some absent
        dict(name="table categories", kind="table", rows=262144, list=1, entries=50021, dim=256, type="bf16", out="f32",
             scale=16.0),
        # the weights of a network of many small tensors, one step
        dict(name="adamw many", kind="adamw", tensors=150, values=4_000_000, type="f32", grad="f32", state="f32", flags=False),
        # a large model's step with states in 8 bits and 16-bit gradients, scaled and perhaps skipped
        dict(name="adamw large", kind="adamw", tensors=12, values=60_000_000, type="f32", grad="bf16", state="f8", flags=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs", "gradients", "lookup", "table", "table", "adamw", "adamw"])
    kinds = ["f32", "f16", "bf16"]
    if kind in ("logprobs", "gradients"):
        classes = _log(rng, 2, 40) if rng.random() < 0.3 else _log(rng, 40, 260_000)
        rows = _log(rng, 1, min(1_000_000, 130_000_000 // classes))
        case = dict(kind=kind, rows=rows, classes=classes, type=rng.choice(kinds),
                    order=rng.choice(["rows", "classes"]) if classes <= 40 else rng.choice(["rows", "rows", "padded"]),
                    given=_log(rng, 1, 12), temperature=rng.choice([1.0, 1.0, 0.7, 1.5, 2.0]),
                    mask=rng.choice(["none", "none", "shared", "rows"]))
        if kind == "logprobs":
            return dict(case, k=rng.choice([0, 1, min(classes, _log(rng, 1, 256))]))
        return dict(case, entropy=rng.random() < 0.5)
    if kind == "adamw":
        state = rng.choice(["f32", "f8"])
        tensors, values = _log(rng, 1, 150 if state == "f32" else 24), _log(rng, 1000, 38_000_000)
        return dict(kind=kind, tensors=tensors, values=max(values, tensors), type=rng.choice(["f32", "f32", "bf16", "f16"]),
                    grad=rng.choice(kinds), state=state, flags=rng.random() < 0.4)
    entries, dim = _log(rng, 16, 300_000), _log(rng, 1, 1024)
    many = 1 if rng.random() < 0.6 else _log(rng, 2, 100)
    entries = min(entries, 30_000_000 // dim)
    rows = _log(rng, 1, min(2_000_000 // many, 60_000_000 // (dim * many)))
    case = dict(kind=kind, rows=rows, list=many, entries=entries, dim=dim, type=rng.choice(kinds),
                scale=rng.choice([1.0, 0.1, 16.0]))
    return case if kind == "lookup" else dict(case, out=rng.choice(["f32", case["type"]]))


# ---- inputs -------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1_000_003 + 71)
    return g


def _laid(x, order):
    """`x` [rows][columns] in an order of memory."""
    if order == "classes":
        return x.t().contiguous().t()
    if order == "padded":
        wide = torch.zeros(x.shape[0], x.shape[1] + 13, dtype=x.dtype, device="cuda")
        wide[:, 5:5 + x.shape[1]] = x
        return wide[:, 5:5 + x.shape[1]]
    return x


def _prepare_scores(case, g, state):
    rows, classes, t = case["rows"], case["classes"], case["temperature"]
    sigma = 2.0 * (0.5 + torch.rand(rows, 1, generator=g, device="cuda"))
    x = torch.randn(rows, classes, generator=g, device="cuda") * sigma
    state["scores"] = _laid(x.to(_TYPES[case["type"]]), case["order"])
    # given classes: those that score high for the most part, as labels do of a model that has learnt
    some = torch.randint(0, classes, (rows, case["given"], 8), generator=g, device="cuda")
    best = x.gather(1, some.flatten(1)).view_as(some).argmax(2, keepdim=True)
    given = some.gather(2, best)[:, :, 0]
    given = torch.where(torch.rand(given.shape, generator=g, device="cuda") < 0.02, -1, given)   # no entry
    state["given"] = given.int()
    state["allowed"] = None
    if case["mask"] != "none":   # three quarters of the classes, the same for every row or not
        shape = (rows if case["mask"] == "rows" else 1, (classes + 31) // 32)
        a = torch.randint(-2**31, 2**31, shape, generator=g, device="cuda")
        state["allowed"] = (a | torch.randint(-2**31, 2**31, shape, generator=g, device="cuda")).int()
    if case["kind"] == "gradients":
        state["logprob_grad"] = -torch.rand(given.shape, generator=g, device="cuda") / rows
        state["entropy_grad"] = -0.01 * torch.rand(rows, generator=g, device="cuda") / rows if case["entropy"] else None
        step = max(1, 50_000_000 // classes)   # by blocks of rows, for the memory
        state["stats"] = torch.cat([_statistics(dict(state, scores=state["scores"][a:a + step], allowed=_some(state, a, a + step)))[1]
                                    for a in range(0, rows, step)])


def _some(state, a, b):
    """The lists of allowed classes of rows a .. b."""
    allowed = state["allowed"]
    return allowed if allowed is None or allowed.shape[0] == 1 else allowed[a:b]


def _tokens(case, g):
    """Entries [rows][list]: with one a row, buckets from frequent to rare; with more, a leaf of every tree, uneven."""
    rows, many, entries = case["rows"], case["list"], case["entries"]
    u = torch.rand(rows, many, generator=g, device="cuda", dtype=torch.float64)
    if many == 1:
        index = torch.pow(float(entries + 1), u) - 1
    else:
        leaves = max(1, entries // many)
        index = torch.floor(u * u * leaves) + leaves * torch.arange(many, device="cuda")
    index = index.long().clamp(0, entries - 1)
    return torch.where(torch.rand(rows, many, generator=g, device="cuda") < 0.01, -1, index).int()   # no entry


def _sizes(case):
    """Sizes of a model's tensors: a few large ones, many small ones, odd for the most part."""
    n, total = case["tensors"], case["values"]
    share = [1.0 / (i + 1) ** 1.3 for i in range(n)]
    whole = sum(share)
    return [max(1, int(total * s / whole)) for s in share]


def _prepare_adamw(case, g, state):
    sizes, starts, at = _sizes(case), [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // _BLOCK) * _BLOCK
    state["sizes"], state["steps"], state["seed"] = sizes, 1000, 12345
    state["flat"] = flat = {}

    def views(name, x, blocks=False):
        flat[name] = x
        return [x[a // _BLOCK:(a + n + _BLOCK - 1) // _BLOCK] if blocks else x[a:a + n] for a, n in zip(starts, sizes)]

    used = torch.zeros(at, dtype=torch.bool, device="cuda")
    for a, n in zip(starts, sizes):
        used[a:a + n] = True

    def normal(scale):
        return torch.where(used, torch.randn(at, generator=g, device="cuda") * scale, torch.zeros((), device="cuda"))

    state["params"] = views("params", normal(0.05).to(_TYPES[case["type"]]))
    scale = 1024.0 if case["flags"] else 1.0
    grads = normal(1e-3 * scale).to(_TYPES[case["grad"]])
    state["grads"] = [grads[a:a + n] for a, n in zip(starts, sizes)]
    m, root = normal(3e-4), normal(1e-3).abs() + 1e-4 * used
    if case["state"] == "f32":
        state["exp_avg"], state["exp_avg_sq"] = views("exp_avg", m), views("exp_avg_sq", root * root)
        state["exp_avg_scale"] = state["exp_avg_sq_scale"] = None
    else:
        for name, x in (("exp_avg", m), ("exp_avg_sq", root)):
            s = _block_scale(x.view(-1, _BLOCK).abs().amax(1))
            q = x.view(-1, _BLOCK) / torch.where(s > 0, s, 1.0)[:, None]
            state[name] = views(name, q.to(torch.float8_e4m3fn).flatten())
            state[name + "_scale"] = views(name + "_scale", s, True)
    state["grad_scale"] = torch.full((1,), 1 / scale, device="cuda") if case["flags"] else None
    state["skip"] = torch.zeros(1, dtype=torch.int32, device="cuda") if case["flags"] else None
    if own:   # the handle that a program keeps beside its weights
        import catboost_rs_amd as cb
        state["optimizer"] = cb.AdamW(state["params"], lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01,
                                      state=case["state"], exp_avg=state["exp_avg"], exp_avg_sq=state["exp_avg_sq"],
                                      exp_avg_scale=state["exp_avg_scale"], exp_avg_sq_scale=state["exp_avg_sq_scale"],
                                      steps=state["steps"], seed=state["seed"])


def prepare(case, seed):
    g, state, kind = _generator(seed), dict(case), case["kind"]
    if kind in ("logprobs", "gradients"):
        _prepare_scores(case, g, state)
    elif kind == "adamw":
        _prepare_adamw(case, g, state)
    else:
        state["index"] = _tokens(case, g)
        if kind == "lookup":
            state["table"] = (torch.randn(case["entries"], case["dim"], generator=g, device="cuda") * 0.05).to(_TYPES[case["type"]])
        else:
            state["grad"] = (torch.randn(case["rows"], case["dim"], generator=g, device="cuda") * 0.1).to(_TYPES[case["type"]])
    return state


# ---- plain forms --------------------------------------------------------------------------
def _masked(s):
    """Scores in 32 bits, -inf where a class is not allowed."""
    x = s["scores"].float()
    if s["allowed"] is not None:
        j = torch.arange(s["classes"], device="cuda")
        x = torch.where((s["allowed"][:, j >> 5] >> (j & 31)) & 1 != 0, x, float("-inf"))
    return x


def _statistics(s):
    """The distances d of a row's scores from the largest, and its statistics [m, log Z, E]: -inf, -inf and 0 of a
    row that allows nothing."""
    x = _masked(s)
    m = x.amax(1, keepdim=True)
    d = (x - torch.where(m > float("-inf"), m, 0.0)) / s["temperature"]
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    far = torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True)
    return d, torch.cat([m, torch.log(z), torch.where(z > 0, -far / z, 0.0)], 1)


def _plain_logprobs(s):
    d, stats = _statistics(s)
    given = s["given"].long()
    some = (given >= 0) & (given < s["classes"])
    log_z = torch.where(stats[:, 1:2] > float("-inf"), stats[:, 1:2], 0.0)   # (a row that allows nothing: d is -inf)
    logprob = torch.where(some, d.gather(1, torch.where(some, given, 0)) - log_z, 0.0)
    out = {"logprob": logprob, "entropy": log_z[:, 0] + stats[:, 2], "stats": stats}
    if s["k"]:
        values, index = torch.sort(d, dim=1, descending=True, stable=True)   # ties: the lowest class first
        values, index = values[:, :s["k"]], index[:, :s["k"]]
        out["top_logprob"] = values - log_z
        out["top_index"] = torch.where(values > float("-inf"), index, -1).int()
    return out


def _plain_gradients(s):
    m, log_z, far = s["stats"][:, :, None].unbind(1)
    some = m > float("-inf")   # (a row that allows nothing)
    d = (_masked(s) - torch.where(some, m, 0.0)) / s["temperature"]
    p = torch.exp(d - torch.where(some, log_z, 0.0))
    given = s["given"].long()
    some = (given >= 0) & (given < s["classes"])
    g = torch.where(some, s["logprob_grad"], 0.0)
    factor = g.sum(1, keepdim=True)
    if s["entropy_grad"] is not None:
        factor = factor + s["entropy_grad"][:, None] * torch.where(p > 0, d + far, 0.0)
    grad = (-p * factor).scatter_add_(1, torch.where(some, given, 0), g)
    if s["allowed"] is not None:
        grad = torch.where(d > float("-inf"), grad, 0.0)
    return {"grad": (grad / s["temperature"]).to(s["scores"].dtype)}


def _plain_lookup(s):
    index, table = s["index"].long(), s["table"]
    some = (index >= 0) & (index < s["entries"])
    rows = table[torch.where(some, index, 0)].float()
    return {"out": (torch.where(some[:, :, None], rows, 0.0).sum(1) * s["scale"]).to(table.dtype)}


def _plain_table(s):
    index, grad = s["index"].long(), s["grad"]
    some = (index >= 0) & (index < s["entries"])
    # an entry may stand in a large part of the rows: sums of parts of them in 32 bits, and over the parts in 64
    entries, dim = s["entries"], s["dim"]
    parts = max(1, min(64, some.numel() // (256 * entries), 2**26 // (entries * dim)))
    part = torch.arange(s["rows"], device="cuda")[:, None] * parts // s["rows"]
    at = torch.where(some, index, entries) + part * (entries + 1)
    total = torch.zeros(parts * (entries + 1), dim, device="cuda")
    rows = grad.float()[:, None].expand(-1, s["list"], -1).reshape(-1, dim)
    total.index_add_(0, at.flatten(), rows)
    total = total.view(parts, entries + 1, dim)[:, :-1].sum(0, dtype=torch.float64)
    return {"grad": (total * s["scale"]).to(_TYPES[s["out"]])}


def _block_scale(largest):
    """The power of two by which a block's values are divided: the largest then lies in (224, 448]."""
    bits = largest.view(torch.int32)
    e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()
    return torch.where(largest < 2.0 ** -100, 0.0, (e << 23).view(torch.float32))


def _mixed(x):
    """The low 32 bits of x, well mixed."""
    x = (x ^ (x >> 16)) * 0x5851F42D & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * 0x4C957F2D & 0xFFFFFFFF
    return x ^ (x >> 16)


def _to_8_bits(x, random, least):
    """Codes (e4m3) and scales of `x`, each value rounded to one of its two neighbours by 16 random bits;
    `least`: a value above 0 is not held as 0."""
    n = x.numel()
    blocks = torch.nn.functional.pad(x, (0, -n % _BLOCK)).view(-1, _BLOCK)
    scale = _block_scale(blocks.abs().amax(1))
    y = (blocks.abs() * torch.where(scale > 0, 1 / scale, 0.0)[:, None]).flatten()[:n]
    normal = (y.view(torch.int32) + (random << 4) >> 20) - (120 << 3)
    small = (y * 512 + random.float() * 2.0 ** -16).int()
    code = torch.where(y < 2.0 ** -6, small, normal)
    if least:
        code = torch.where(x > 0, code.clamp(min=1), code)
    code = torch.where(y > 0, code, 0) | torch.where(x < 0, 128, 0)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), scale


def _from_8_bits(code, scale):
    n = code.numel()
    return code.float() * scale.repeat_interleave(_BLOCK)[:n]


def _plain_step(s, i, factors):
    """One tensor's step, in place."""
    decay, rate, root_correction = factors
    p, g = s["params"][i], s["grads"][i].float()
    if s["grad_scale"] is not None:
        g = g * s["grad_scale"]
    small = s["state"] == "f8"
    if small:
        m = _from_8_bits(s["exp_avg"][i], s["exp_avg_scale"][i])
        v = torch.square(_from_8_bits(s["exp_avg_sq"][i], s["exp_avg_sq_scale"][i]))
    else:
        m, v = s["exp_avg"][i], s["exp_avg_sq"][i]
    m = m * 0.9 + g * (1 - 0.9)
    v = v * 0.999 + g * g * (1 - 0.999)
    root = torch.sqrt(v)
    new = p.float() * decay - m * rate / (root * root_correction + 1e-8)
    go = True if s["skip"] is None else s["skip"] == 0

    def keep(old, x):
        old.copy_(x if go is True else torch.where(go, x, old.float()))

    keep(p, new)
    if small:
        key = _mixed(s["seed"] ^ _mixed(s["steps"] & 0xFFFFFFFF)) + i * 0x9E3779B9
        bits = _mixed((torch.arange(p.numel(), device="cuda") + key) & 0xFFFFFFFF)
        for name, x, random, least in (("exp_avg", m, bits & 0xFFFF, False), ("exp_avg_sq", root, bits >> 16, True)):
            code, scale = _to_8_bits(x, random.int(), least)
            keep(s[name][i], code.float())   # (whole codes: nothing is rounded again)
            keep(s[name + "_scale"][i], scale)
    else:
        keep(s["exp_avg"][i], m)
        keep(s["exp_avg_sq"][i], v)


def _plain_adamw(s):
    s["steps"] += 1
    factors = (1 - 1e-3 * 0.01, 1e-3 / (1 - 0.9 ** s["steps"]), 1 / math.sqrt(1 - 0.999 ** s["steps"]))
    for i in range(len(s["params"])):   # a model's tensors are separate ones
        _plain_step(s, i, factors)
    return s["flat"]


def run(state):
    kind = state["kind"]
    if own:
        import catboost_rs_amd as cb
        if kind == "logprobs":
            got = cb.class_logprobs(state["scores"], state["given"], temperature=state["temperature"], k=state["k"],
                                    allowed=state["allowed"])
            out = {"logprob": got.logprob, "entropy": got.entropy, "stats": got.stats}
            if state["k"]:
                out.update(top_logprob=got.top_logprob, top_index=got.top_index)
            return out
        if kind == "gradients":
            return {"grad": cb.logprob_gradients(state["scores"], state["given"], state["logprob_grad"], state["stats"],
                                                 entropy_grad=state["entropy_grad"], temperature=state["temperature"],
                                                 allowed=state["allowed"])}
        if kind == "lookup":
            return {"out": cb.lookup_rows(state["table"], state["index"], scale=state["scale"])}
        if kind == "table":
            return {"grad": cb.lookup_gradients(state["grad"], state["index"], state["entries"], scale=state["scale"],
                                                dtype=_TYPES[state["out"]])}
        state["optimizer"].step(state["grads"], grad_scale=state["grad_scale"], skip=state["skip"])
        return state["flat"]
    return {"logprobs": _plain_logprobs, "gradients": _plain_gradients, "lookup": _plain_lookup, "table": _plain_table,
            "adamw": _plain_adamw}[kind](state)


def work(case):
    kind = case["kind"]
    if kind in ("logprobs", "gradients"):
        rows, classes, e = case["rows"], case["classes"], _BYTES[case["type"]]
        words = (classes + 31) // 32 * 4
        n = rows * classes * e + {"none": 0, "shared": words, "rows": rows * words}[case["mask"]]
        if kind == "logprobs":
            return {"bytes": n + rows * (8 * case["given"] + 16 + 8 * case["k"]), "flops": 6 * rows * classes}
        n += rows * classes * e + rows * (8 * case["given"] + 12 + 4 * case["entropy"])
        return {"bytes": n, "flops": (8 if case["entropy"] else 5) * rows * classes}
    if kind == "adamw":
        values = sum(_sizes(case))
        a = 2 * _BYTES[case["type"]] + _BYTES[case["grad"]] + (16 if case["state"] == "f32" else 4 + 16 / _BLOCK)
        return {"bytes": values * a, "flops": 15 * values}
    rows, many, entries, dim = case["rows"], case["list"], case["entries"], case["dim"]
    e = _BYTES[case["type"]]
    n = rows * many * 4 + rows * dim * e
    if kind == "lookup":
        n += min(entries, rows * many) * dim * e
    else:
        n += entries * dim * _BYTES[case["out"]]
    return {"bytes": n, "flops": rows * many * dim}


# ---- the definitions, in 64 bits ----------------------------------------------------------
def _allowed(s, a, b):
    bits = _some(s, a, b)
    if bits is None:
        return None
    word = torch.arange(32, device="cuda")
    return ((bits[:, :, None] >> word) & 1).flatten(1)[:, :s["classes"]] != 0


def _exact_scores(s, a, b):
    z = s["scores"][a:b].double() / s["temperature"]
    free = _allowed(s, a, b)
    if free is not None:
        z = z.masked_fill(~free, float("-inf"))
    lse = torch.logsumexp(z, 1, keepdim=True)
    logp = torch.where(lse > float("-inf"), z - lse, float("-inf"))   # (a row that allows nothing)
    p = torch.exp(logp)
    entropy = -torch.nan_to_num(p * logp, nan=0.0).sum(1, keepdim=True)
    given = s["given"][a:b].long()
    some = (given >= 0) & (given < s["classes"])
    at = torch.where(some, given, 0)
    if s["kind"] == "logprobs":
        best = z.amax(1, keepdim=True)
        log_z = torch.where(best > float("-inf"), lse - best, best)
        out = {"logprob": torch.where(some, logp.gather(1, at), 0.0), "entropy": entropy[:, 0],
               "stats": torch.cat([best * s["temperature"], log_z, torch.where(log_z > float("-inf"), entropy - log_z, 0.0)], 1)}
        if s["k"]:
            out["top_logprob"], out["top_index"] = torch.topk(logp, s["k"], dim=1).values, None
        return out
    g = torch.where(some, s["logprob_grad"][a:b].double(), 0.0)
    grad = torch.zeros_like(z).scatter_add_(1, at, g) - p * g.sum(1, keepdim=True)
    if s["entropy_grad"] is not None:
        grad -= s["entropy_grad"][a:b, None].double() * torch.nan_to_num(p * (logp + entropy), nan=0.0)
    if free is not None:
        grad = grad.masked_fill(~free, 0.0)
    return {"grad": grad / s["temperature"]}


def _exact_lookup(s):
    index = s["index"].long()
    pad = torch.where((index < 0) | (index >= s["entries"]), s["entries"], index)
    table = torch.nn.functional.pad(s["table"].double(), (0, 0, 0, 1))
    out = torch.zeros(s["rows"], s["dim"], dtype=torch.float64, device="cuda")
    for i in range(s["list"]):
        out += table[pad[:, i]]
    return {"out": out * s["scale"]}


def _exact_table(s):
    index = s["index"].long()
    pad = torch.where((index < 0) | (index >= s["entries"]), s["entries"], index)
    total = torch.zeros(s["entries"] + 1, s["dim"], dtype=torch.float64, device="cuda")
    for i in range(s["list"]):   # sorted, and sums as differences of running ones: by blocks of columns, for the memory
        by = torch.argsort(pad[:, i], stable=True)
        ends = torch.bincount(pad[:, i], minlength=s["entries"] + 1).cumsum(0)
        for c in range(0, s["dim"], 64):
            running = torch.nn.functional.pad(s["grad"][by, c:c + 64].double().cumsum(0), (0, 0, 1, 0))
            upto = running[ends]
            total[:, c:c + 64] += upto - torch.cat([running[:1], upto[:-1]])
    return {"grad": total[:-1] * s["scale"]}


def _exact_adamw(s):
    t, small = s["steps"] + 1, s["state"] == "f8"
    p, kept = s["flat"]["params"].double(), {name: s["flat"][name].double() for name in ("exp_avg", "exp_avg_sq")}
    if small:
        for name in kept:
            kept[name] = (kept[name].view(-1, _BLOCK) * s["flat"][name + "_scale"].double()[:, None]).flatten()
        kept["exp_avg_sq"] = kept["exp_avg_sq"] ** 2
    g, at = torch.zeros_like(p), 0
    for x in s["grads"]:
        g[at:at + x.numel()] = x.double() * (1.0 if s["grad_scale"] is None else s["grad_scale"].double())
        at += -(-x.numel() // _BLOCK) * _BLOCK
    m = 0.9 * kept["exp_avg"] + 0.1 * g
    v = 0.999 * kept["exp_avg_sq"] + 0.001 * g ** 2
    step = (m / (1 - 0.9 ** t)) / (torch.sqrt(v / (1 - 0.999 ** t)) + 1e-8)
    out = {"params": p - 1e-3 * (step + 0.01 * p), "exp_avg": m, "exp_avg_sq": v}
    # (what 8 bits hold goes by random bits: no value of its own)
    return dict(out, exp_avg=None, exp_avg_sq=None, exp_avg_scale=None, exp_avg_sq_scale=None) if small else out


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("logprobs", "gradients"):
        step = max(1, 60_000_000 // case["classes"])
        parts = [_exact_scores(s, a, min(case["rows"], a + step)) for a in range(0, case["rows"], step)]
        return {name: None if parts[0][name] is None else torch.cat([p[name] for p in parts]) for name in parts[0]}
    return {"lookup": _exact_lookup, "table": _exact_table, "adamw": _exact_adamw}[kind](s)
