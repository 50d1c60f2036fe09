"""Plain 64-bit forms of the operators over a vocabulary, written row by row from their formulas, and bounds on what
32-bit arithmetic may differ from them."""
import numpy as np

import musapy_amd as ms
from tests.blocks_reference import ROUND, rounded, to_device, values

U = 2.0 ** -24  # half an ulp of f32, relative


def ids(x, dt="i64"):
    return ms.array(np.asarray(x), dtype=dt)


def draw(rng, shape, dt, scale=1.0):
    return rounded(rng.standard_normal(shape) * scale, dt)


def within(got, want, bound, dt, what=""):
    """|got - want| <= bound + the rounding of a stored result; infinities and NaN in the same places."""
    got = values(got) if not isinstance(got, np.ndarray) else got
    assert got.shape == want.shape, (what, got.shape, want.shape)
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)]), what
    rel, tiny = ROUND[dt]
    w = np.where(odd, 0.0, want)
    err = np.abs(np.where(odd, 0.0, got) - w)
    room = np.broadcast_to(bound, w.shape) + (np.abs(w) + bound) * rel + tiny
    room = np.where(odd, 0.0, room)
    bad = err > room
    if bad.any():
        at = tuple(int(i[0]) for i in np.nonzero(bad))
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size}, first at {at}: {got[at]!r}, not {want[at]!r} "
                             f"(off by {err[at]:.3g}, room {room[at]:.3g})")


# ---- embedding -------------------------------------------------------------------------------------------
def embedding(table, tokens, scale):
    out = np.zeros(tokens.shape + table.shape[1:])
    for at in np.ndindex(tokens.shape):
        if 0 <= tokens[at] < len(table):
            out[at] = table[tokens[at]] * scale
    return out


def embedding_grad(dy, tokens, rows, scale):
    """(sums, sums of the terms' absolute values times the number of roundings)"""
    out = np.zeros((rows, dy.shape[-1]))
    size, n = np.zeros_like(out), np.zeros(rows)
    dy = dy.reshape(-1, dy.shape[-1])
    for k, d in zip(tokens.reshape(-1), dy):
        if 0 <= k < rows:
            out[k] += d
            size[k] += np.abs(d)
            n[k] += 1
    return out * scale, U * (n[:, None] + 2) * size * abs(scale)


# ---- distillation -----------------------------------------------------------------------------------------
def softmax(x):
    e = np.exp(x - x.max())
    return e / e.sum()


def log_sum(x):
    """(m, log sum exp(x - m))"""
    return x.max(), np.log(np.exp(x - x.max()).sum())


def entries(index, teacher, width, temp):
    """(indices, probabilities) of the entries of a row that count"""
    keep = (index >= 0) & (index < width) & (teacher != -np.inf)
    if not keep.any():
        return index[:0], teacher[:0]
    return index[keep], softmax(teacher[keep] / temp)


def uses(z, i, label, weight):
    return len(i) > 0 and weight > 0, label is not None and 0 <= label < len(z) and weight < 1


def distill(z, index, teacher, label, temp, weight):
    """One row: (loss, highest logit m, log sum exp((z - m) / T), log sum exp(z - m))"""
    i, p = entries(index, teacher, len(z), temp)
    soft, hard = uses(z, i, label, weight)
    loss, m, ls, ls1 = 0.0, 0.0, 0.0, 0.0
    with np.errstate(all="ignore"):
        if soft:
            m = z.max()
            ls = log_sum((z - m) / temp)[1]
            some = p > 0
            loss += weight * temp ** 2 * (p[some] * (np.log(p[some]) - ((z[i[some]] - m) / temp - ls))).sum()
        if hard:
            m, ls1 = log_sum(z)
            loss += (1 - weight) * (m - z[label] + ls1)
    return loss, m, ls, ls1


def distill_grad(dl, z, sums, index, teacher, label, temp, weight):
    """One row's gradient, from what the loss left."""
    g = np.zeros(len(z))
    i, p = entries(index, teacher, len(z), temp)
    soft, hard = uses(z, i, label, weight)
    if soft:
        q = np.exp((z - sums[0]) / temp - sums[1])
        np.subtract.at(q, i, p)
        g += weight * temp * q
    if hard:
        s = np.exp(z - sums[0] - sums[2])
        s[label] -= 1
        g += (1 - weight) * s
    return dl * g


def _spread(x):
    x = x[np.isfinite(x)]
    return float(x.max() - x.min()) if len(x) else 0.0


def log_sum_bound(z, temp):
    """Of log sum exp((z - m) / T): each term is off by 4 roundings of its exponent, at most the spread (terms further
    down weigh nothing: 30 at most counts), and two of its own; a thread adds V / 512 terms and rescales its sum some times, and
    the joins are ten more; the logarithm, at most some 12, is off by four roundings of its own."""
    return U * (8 * min(_spread(z) / temp, 30.0) + len(z) / 256 + 128 + 4 * np.log(len(z)))


def _teacher_bound(kept, temp, n):
    """Of p, relative: exponents and their roundings as above, a sum of n terms."""
    return U * (8 * min(_spread(kept) / temp, 30.0) + n + 16)


def distill_bound(z, index, teacher, label, temp, weight):
    """(loss, m, the two logarithms).  The loss is formed from differences: of the teacher's values to their highest, of the
    entries' logits to theirs, and of that to the row's; each part is off by some roundings of its own size."""
    i, p = entries(index, teacher, len(z), temp)
    soft, hard = uses(z, i, label, weight)
    ls, ls1 = log_sum_bound(z, temp), log_sum_bound(z, 1.0)
    m = z[np.isfinite(z)].max(initial=-np.inf)
    b = 0.0
    if soft:
        kept = teacher[(index >= 0) & (index < len(z)) & (teacher != -np.inf)]
        zi = z[i][np.isfinite(z[i])]
        r = zi.max(initial=-np.inf) if len(zi) else 0.0
        off = np.where(np.isfinite(z[i]), np.abs(z[i] - r), 0.0)
        size = (p * (np.abs(kept - kept.max()) + off)).sum() / temp
        rel = _teacher_bound(kept, temp, len(i))
        parts = size + np.log(len(p)) + abs(m - r) / temp + np.log(len(z))
        b += weight * temp ** 2 * (2 * rel * size + rel + ls + 12 * U * parts)
    if hard:
        zl = abs(m - z[label]) if np.isfinite(z[label]) else 0.0
        b += (1 - weight) * (ls1 + 4 * U * (zl + np.log(len(z))))
    return b, 0.0, ls, ls1


def distill_grad_bound(dl, z, sums, index, teacher, label, temp, weight):
    """exp((x - m) / T - l): four roundings of each part of the exponent, ten of factors; below f32's normal numbers nothing
    is promised but their size."""
    g = np.zeros(len(z))
    i, p = entries(index, teacher, len(z), temp)
    soft, hard = uses(z, i, label, weight)
    d = np.where(np.isfinite(z), sums[0] - z, 0.0)
    if soft:
        q = np.exp(-d / temp - sums[1]) * np.isfinite(z)
        g += weight * temp * (q * U * (4 * d / temp + 4 * sums[1] + 10) + 2.0 ** -125)
        kept = teacher[(index >= 0) & (index < len(z)) & (teacher != -np.inf)]
        np.add.at(g, i, weight * temp * p * (2 * _teacher_bound(kept, temp, len(index)) + 8 * U))
    if hard:
        s = np.exp(-d - sums[2]) * np.isfinite(z)
        # (or, at T = 2, the square of exp((x - m) / 2 - l): twice its relative error, and the constant's own)
        g += (1 - weight) * (s * U * (4 * d + 4 * sums[2] + 10 + (8 * sums[1] + 20 if temp == 2 else 0)) + 2.0 ** -125)
        g[label] += 4 * U * (1 - weight)
    return abs(dl) * g


# ---- logits --------------------------------------------------------------------------------------------------
def adjust(z, history=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, bias_index=None, allowed=None):
    """One row: (values, bound).  Every operation rounds once."""
    z = z.astype(np.float64).copy()
    size = np.abs(np.where(np.isfinite(z), z, 0.0))
    if history is not None:
        for v, c in zip(*np.unique(history, return_counts=True)):
            if not 0 <= v < len(z):
                continue
            z[v] = z[v] / repetition if z[v] > 0 else z[v] * repetition
            z[v] -= frequency * c + presence
            size[v] = max(size[v], size[v] * repetition, size[v] / repetition) + 2 * (abs(frequency) * c + abs(presence))
    if bias_index is not None:
        for v, b in zip(bias_index, bias):
            if 0 <= v < len(z):
                z[v] += b
                size[v] += 2 * abs(b) * len(bias)
    elif bias is not None:
        z += bias
        size += np.abs(bias)
    if allowed is not None:
        z[~allowed] = -np.inf
    return z, 4 * U * size


def pack(allowed):
    """Truth values (..., V) as 32-bit words (..., ceil(V / 32)), lowest bits first; bits behind the last column are set."""
    v = allowed.shape[-1]
    pad = np.ones(allowed.shape[:-1] + (-v % 32,), dtype=bool)
    b = np.concatenate([allowed, pad], -1).reshape(allowed.shape[:-1] + (-1, 32)).astype(np.uint32)
    return (b << np.arange(32, dtype=np.uint32)).sum(-1, dtype=np.uint32)


__all__ = ["to_device", "values", "rounded"]
