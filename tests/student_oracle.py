"""Plain 64-bit implementations of log probabilities and their gradient, looked-up rows and the table's
gradient, and AdamW steps; the 8-bit states' codes in numpy's f32, whose every operation rounds as the
device's does."""
import numpy as np

BLOCK = 256


# ---- class scores ---------------------------------------------------------------------------
def masked(x, allowed):
    x = np.asarray(x, np.float64)
    return x if allowed is None else np.where(allowed, x, -np.inf)


def row_stats(x, t, allowed=None):
    """d [rows][n], m, log Z and E of every row; rows of -inf alone: -inf, -inf, 0; rows with NaN or +inf: NaN."""
    x = masked(x, allowed)
    with np.errstate(all="ignore"):
        m = x.max(1)
        d = (x - np.where(np.isneginf(m), 0.0, m)[:, None]) / t
        e = np.exp(d)
        z = e.sum(1)
        far = -np.where(e > 0, e * d, np.where(np.isnan(e), np.nan, 0.0)).sum(1) / np.where(z == 0, 1.0, z)
        log_z = np.log(z)
    return d, np.where(np.isnan(z), np.nan, m), log_z, np.where(np.isnan(z), np.nan, far)


def logprobs(x, given, t, k, allowed=None):
    """logprob, entropy, stats, top_logprob, top_index."""
    rows, n = x.shape
    d, m, log_z, far = row_stats(x, t, allowed)
    base = np.where(np.isneginf(log_z), 0.0, log_z)
    ok = (given >= 0) & (given < n)
    with np.errstate(all="ignore"):
        lp = np.where(ok, np.take_along_axis(d, np.where(ok, given, 0), 1) - base[:, None], 0.0)
        x = masked(x, allowed)
        key = np.where(np.isnan(x), np.inf, x)
        if np.isnan(x).any():
            order = np.lexsort((np.broadcast_to(np.arange(n), x.shape), -key, ~np.isnan(x)), axis=1)[:, :k]
        else:
            order = np.argsort(-key, axis=1, kind="stable")[:, :k]
        top = np.take_along_axis(d, order, 1) - base[:, None]
        top = np.where(np.isnan(log_z)[:, None], np.nan, top)
        lp = np.where(np.isnan(log_z)[:, None] & ok, np.nan, lp)
    index = np.where(np.isneginf(np.take_along_axis(x, order, 1)), -1, order)
    return lp, base + far, np.stack([m, log_z, far], 1), top, index


def logprob_gradients(x, given, g, h, t, allowed=None):
    """The gradient, and for every value the size that its rounding errors count against."""
    rows, n = x.shape
    d, m, log_z, far = row_stats(x, t, allowed)
    ok = (given >= 0) & (given < n)
    g = np.where(ok, g, 0.0).astype(np.float64)
    h = np.zeros(rows) if h is None else np.asarray(h, np.float64)
    with np.errstate(all="ignore"):
        p = np.where(np.isneginf(log_z)[:, None], 0.0, np.exp(d - log_z[:, None]))
        near = np.where(p > 0, d, np.where(np.isnan(p), np.nan, 0.0))
        whole = g.sum(1)[:, None] + h[:, None] * (near + far[:, None])
        grad = -p * whole
        size = p * (np.abs(g).sum(1)[:, None] + np.abs(h)[:, None] * (np.abs(near) + np.abs(far)[:, None]))
    np.add.at(grad, (np.arange(rows)[:, None].repeat(given.shape[1], 1)[ok], given[ok]), g[ok])
    zero = (g == 0).all(1) & (h == 0)
    free = np.ones((rows, n), bool) if allowed is None else np.broadcast_to(allowed, (rows, n))
    grad = np.where(free & ~zero[:, None], grad, 0.0) / t
    return grad, np.where(zero[:, None], 0.0, size) / t


# ---- tables ---------------------------------------------------------------------------------
def lookup(table, index, scale):
    """Sums, and the sums of sizes."""
    entries = table.shape[0]
    ok = (index >= 0) & (index < entries)
    rows = np.where(ok[:, :, None], table.astype(np.float64)[np.where(ok, index, 0)], 0.0)
    return rows.sum(1) * scale, np.abs(rows).sum(1) * abs(scale)


def table_gradient(grad, index, entries, scale):
    """Sums, the sums of sizes, and how often every entry occurs."""
    out, size = np.zeros((2, entries, grad.shape[1]))
    ok = (index >= 0) & (index < entries)
    place = np.broadcast_to(np.arange(len(index))[:, None], index.shape)[ok]
    np.add.at(out, index[ok], grad[place].astype(np.float64))
    np.add.at(size, index[ok], np.abs(grad[place]).astype(np.float64))
    return out * scale, size * abs(scale), np.bincount(index[ok], minlength=entries)


# ---- AdamW ----------------------------------------------------------------------------------
def mix(x):
    x = np.asarray(x, np.uint64)
    mask = np.uint64(0xFFFFFFFF)
    x = (x ^ (x >> np.uint64(16))) * np.uint64(0x5851F42D) & mask
    x = (x ^ (x >> np.uint64(15))) * np.uint64(0x4C957F2D) & mask
    return x ^ (x >> np.uint64(16))


def random_bits(n, seed, step, number):
    """The low and the high 16 bits of every value."""
    key = int(mix(seed ^ int(mix(step & 0xFFFFFFFF)))) + number * 0x9E3779B9 & 0xFFFFFFFF
    r = mix((np.arange(n, dtype=np.uint64) + np.uint64(key)) & np.uint64(0xFFFFFFFF))
    return (r & np.uint64(0xFFFF)).astype(np.uint32), (r >> np.uint64(16)).astype(np.uint32)


def code_values():
    """The 256 values of e4m3."""
    c = np.arange(256)
    e, f = c >> 3 & 15, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * 2.0 ** (e - 7.0))
    v = np.where(c & 0x7F == 0x7F, np.nan, v)
    return np.where(c & 0x80, -v, v).astype(np.float32)


def block_scale(largest):
    with np.errstate(all="ignore"):
        s = 2.0 ** np.ceil(np.log2(largest.astype(np.float64) / 448.0))
        # (the logarithm may round: the largest lies in (224, 448] of it)
        s = np.where(largest / s > 448, s * 2, np.where(largest / s <= 224, s / 2, s))
    return np.where(largest < 2.0 ** -100, 0.0, s).astype(np.float32)


def encode(x, random, least):
    """Codes and scales of f32 values."""
    n = len(x)
    a = np.where(np.isfinite(x), np.abs(x), 0).astype(np.float32)
    blocks = np.concatenate([a, np.zeros(-n % BLOCK, np.float32)]).reshape(-1, BLOCK)
    scale = block_scale(blocks.max(1)) if n else np.zeros(0, np.float32)
    with np.errstate(all="ignore"):
        each = np.repeat(scale, BLOCK)[:n]
        y = np.where(each > 0, a / np.where(each > 0, each, 1), 0).astype(np.float64)
        code = np.zeros(n, np.int64)
        table = code_values()[:0x7F].astype(np.float64)
        low = np.searchsorted(table, y, side="right") - 1
        low = np.minimum(low, 0x7E)
        step = np.where(low < 0x7E, table[np.minimum(low + 1, 0x7E)] - table[low], 1.0)
        # what is left of y as a fraction of the step, in the bits that f32 holds; up where it and u 2^-16 reach 1 together
        part = (y - table[low]) / step
        small = y < 2.0 ** -6
        up = np.where(small, np.floor((y * 512).astype(np.float32) + (random * np.float32(2.0 ** -16)).astype(np.float32)) - low,
                      part + random * 2.0 ** -16 >= 1)
        code = low + up.astype(np.int64)
    if least:
        code = np.where(x > 0, np.maximum(code, 1), code)
    code = np.where(y > 0, code, 0)
    code = np.where(np.isfinite(x), code, 0x7F)
    return (code | np.where(x < 0, 0x80, 0)).astype(np.uint8), scale


def decode(code, scale):
    return (code_values()[code] * np.repeat(scale, BLOCK)[:len(code)]).astype(np.float32)


def adamw_f32(p, g, m, v, step, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, grad_scale=None):
    """New p (f32, before its rounding), m, v and sqrt(v) in numpy's f32, in the device's order."""
    f = np.float32
    with np.errstate(all="ignore"):
        decay, rate = f(1.0 - lr * weight_decay), f(lr / (1.0 - beta1 ** step))
        correction = f(1.0 / np.sqrt(1.0 - beta2 ** step))
        p, g, m, v = (np.asarray(a, f) for a in (p, g, m, v))
        if grad_scale is not None:
            g = g * f(grad_scale)
        m = m * f(beta1) + g * f(1.0 - beta1)
        v = v * f(beta2) + g * g * f(1.0 - beta2)
        root = np.sqrt(v)
        p = p * decay - m * rate / (root * correction + f(eps))
    return p, m, v, root


def adamw(p, g, m, v, step, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01):
    """New p, m, v in 64 bits."""
    p, g, m, v = (np.asarray(a, np.float64) for a in (p, g, m, v))
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    p = p * (1 - lr * weight_decay) - lr * (m / (1 - beta1 ** step)) / (np.sqrt(v / (1 - beta2 ** step)) + eps)
    return p, m, v
