"""Plain 64-bit implementations of the operators on class scores, and scores to try them on."""
import numpy as np

LOWEST = float(np.finfo(np.float32).min)


def round_to(x, kind):
    """f32 values as the type holds them (still f32)."""
    x = np.asarray(x, np.float32)
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    if kind == "bf16":
        return from_bits(to_bits(x, kind), kind)
    return x


def to_bits(x, kind):
    """The array whose bytes are the scores of this type."""
    x = np.asarray(x, np.float32)
    if kind == "f32":
        return x
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32)
    r = ((b.astype(np.uint64) + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, kind):
    if kind == "bf16":
        return (b.astype(np.uint32) << 16).view(np.float32)
    return b.astype(np.float32)


def half_step(kind):
    return {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]


def smallest(kind):
    """What a result below the type's normal range may be off by."""
    return {"f32": 2.0 ** -125, "f16": 2.0 ** -25, "bf16": 2.0 ** -125}[kind]


def log_sum_exp(z):
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = z.max(1, keepdims=True)
        d = np.where(np.isneginf(z), 0.0, np.exp(np.where(z == m, 0.0, z - m)))
        return np.where(np.isposinf(m[:, 0]), np.inf, np.where(np.isneginf(m[:, 0]), -np.inf, m[:, 0] + np.log(d.sum(1))))


def top(x, k, t):
    x = x.astype(np.float64)
    by = np.argsort(np.where(np.isnan(x), -np.inf, -x), axis=1, kind="stable")
    nan_first = np.argsort(~np.isnan(np.take_along_axis(x, by, 1)), axis=1, kind="stable")
    by = np.take_along_axis(by, nan_first, 1)[:, :k]
    return np.take_along_axis(x, by, 1), by, log_sum_exp(x / t)


def distill(x, u, ix, base, t, weight):
    """Loss and gradient of every row, row by row; and the part of the gradient that is a softmax
    probability (what its rounding counts against)."""
    rows, n = x.shape
    loss, grad, size = np.zeros(rows), np.zeros((rows, n)), np.zeros((rows, n))
    with np.errstate(all="ignore"):
        for r in range(rows):
            w = 1.0 if weight is None else float(weight[r])
            if w == 0:
                continue
            z = x[r].astype(np.float64) / t
            ok = (ix[r] >= 0) & (ix[r] < n)
            at, lu = ix[r][ok].astype(int), u[r][ok].astype(np.float64) / t
            m = z.max()
            if np.isnan(z).any() or m == np.inf:
                loss[r], grad[r] = np.nan, np.nan
                continue
            p = np.zeros(n) if m == -np.inf else np.exp(z - m) / np.exp(z - m).sum()
            # log q and log p as differences from the largest first: a log-sum-exp next to the lowest
            # f32 would lose the logarithm
            if base is not None:
                lq = lu - float(base[r])
            elif at.size:
                lq = (lu - lu.max()) - np.log(np.exp(lu - lu.max()).sum())
            else:
                lq = lu
            q = np.exp(lq)
            free = np.ones(n, bool)
            free[at] = False
            rest = max(0.0, 1.0 - q.sum()) if base is not None and free.any() else 0.0
            others = p[free].sum()
            pos = q > 0
            lp = np.log(p[at]) if m == -np.inf else (z[at] - m) - np.log(np.exp(z - m).sum())
            loss[r] = (q[pos] * (lq[pos] - lp[pos])).sum()
            if rest > 0:
                loss[r] += rest * (np.log(rest) - np.log(others))
            g = p * (q.sum() + rest)
            size[r] = w * t * g
            if others > 0:
                share = rest * p / others
                size[r] = np.where(free, w * t * np.abs(g - share), size[r])
                g = np.where(free, g - share, g)
            g[at] -= q
            loss[r] *= w * t * t
            grad[r] = w * t * g
    return loss, grad, size


def sample(x, u, t, k, p, min_p, allowed):
    """Per row: the kept masses' running sums in class order, the order's first class, the log
    probabilities, and whether the row is empty or greedy."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if allowed is not None:
        x = np.where(allowed, x, -np.inf)
    n = x.shape[1]
    out = []
    with np.errstate(all="ignore"):
        for r in range(x.shape[0]):
            m = x[r].max()
            if m == -np.inf:
                out.append(dict(empty=True))
                continue
            first = int(np.argmax(x[r]))
            if not t[r] > 0:
                out.append(dict(empty=False, greedy=True, first=first))
                continue
            w = np.where(x[r] == m, 1.0, np.exp((x[r] - m) / t[r]))
            w = np.where(np.isneginf(x[r]), 0.0, w)
            order = np.argsort(-x[r], kind="stable")
            s = w[order]
            place = np.arange(n)
            stay = place < (k[r] if k[r] > 0 else n)
            mass = np.cumsum(np.where(stay, s, 0.0))
            if p[r] < 1:
                stay &= np.concatenate([[0.0], mass[:-1]]) < p[r] * mass[-1]
            stay &= ~(s < min_p[r])
            stay[0] = True
            kept = np.zeros(n)
            kept[order] = np.where(stay, s, 0.0)
            lp = np.where(x[r] == m, 0.0, (x[r] - m) / t[r]) - np.log(w.sum())
            out.append(dict(empty=False, greedy=False, first=first, kept=kept, cum=np.cumsum(kept), logprob=lp))
    return out


def check_sample(index, logprob, want, u, n, tag=""):
    """The drawn classes are those of the running sums; a draw within rounding (of n sums in 64 bits and n
    masses of 2^-52 of the largest) of a border may fall on either side of it."""
    for r, o in enumerate(want):
        if o["empty"]:
            assert index[r] == -1 and logprob[r] == -np.inf, (tag, r, index[r], logprob[r])
            continue
        if o["greedy"]:
            assert index[r] == o["first"] and logprob[r] == 0, (tag, r, index[r], o["first"])
            continue
        j, cum = int(index[r]), o["cum"]
        assert 0 <= j < n and o["kept"][j] > 0, (tag, r, j)
        target, eps = u[r] * cum[-1], cum[-1] * 2.0 ** -52 * (n + 8) + n * 2.0 ** -44 * 2.0 ** -8
        assert (cum[j - 1] if j else 0.0) <= target + eps and target <= cum[j] + eps, (tag, r, j, target, cum[max(j - 1, 0):j + 1])
        assert abs(logprob[r] - o["logprob"][j]) <= 2.0 ** -22 * (1 + abs(o["logprob"][j])), (tag, r)


def scores(g, rows, n, kind):
    """Scores [rows][n] f32 of one of several kinds."""
    if kind == "normal":
        return (g.standard_normal((rows, n)) * (0.5 + 3 * g.random((rows, 1)))).astype(np.float32)
    if kind == "ties":
        return g.integers(-3, 4, (rows, n)).astype(np.float32) * 0.5
    if kind == "equal":
        return np.full((rows, n), 1.5, np.float32)
    if kind == "rising":
        return np.linspace(-9, 9, n, dtype=np.float32)[None] * np.linspace(0.5, 1, rows, dtype=np.float32)[:, None]
    x = scores(g, rows, n, "normal")
    if kind == "masked":        # -inf and the type's lowest value in places, a row of each alone
        x[g.random((rows, n)) < 0.4] = -np.inf
        x[g.random((rows, n)) < 0.2] = LOWEST
        x[0] = -np.inf
        if rows > 1:
            x[1] = LOWEST
        return x
    if kind == "sharp":         # one class far above the others
        x[np.arange(rows), g.integers(0, n, rows)] += 60
        return x
    raise ValueError(kind)
