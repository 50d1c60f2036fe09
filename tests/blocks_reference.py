"""Plain 64-bit forms of the gated recurrent block's operators, written step by step from their formulas, and bounds
on what 32-bit arithmetic may differ from them."""
import numpy as np

import musapy_amd as ms

EPS = 2.0 ** -24  # half an ulp of f32, relative
# a stored result's rounding: half an ulp, relative, and the spacing of the smallest numbers
ROUND = {"f32": (2.0 ** -24, 2.0 ** -149), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -133)}


def rounded(x, dt):
    """`x` rounded to `dt`, as f64 values."""
    if dt == "f32":
        return x.astype(np.float32).astype(np.float64)
    if dt == "f16":
        return x.astype(np.float16).astype(np.float64)
    b = np.ascontiguousarray(x.astype(np.float32)).view(np.uint32).astype(np.uint64)
    b = ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32)
    return b.view(np.float32).astype(np.float64).reshape(np.shape(x))


def bf16_bits(x):
    return (np.ascontiguousarray(x.astype(np.float32)).view(np.uint32) >> 16).astype(np.uint16)


def to_device(x, dt):
    """A device array of the (already rounded) values."""
    x = np.asarray(x)
    if dt == "bool":
        return ms.array(x, dtype="bool")
    if dt == "bf16":
        return ms.array(bf16_bits(x).reshape(x.shape), dtype="bf16")
    return ms.array(x, dtype=dt)


def values(a):
    """A device array's values in f64."""
    h = a.numpy()
    if a.dtype == "bf16":
        return (h.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return h.astype(np.float64)


def sigmoid(g):
    e = np.exp(-np.abs(g))
    return np.where(g >= 0, 1 / (1 + e), e / (1 + e))


# ---- gated scan ------------------------------------------------------------------------------------
def factors(x, g, kind):
    """(a, b) of h[t] = a[t] h[t-1] + b[t]"""
    if kind == "decay":
        return np.broadcast_to(g, x.shape), x
    return np.broadcast_to(sigmoid(g), x.shape), sigmoid(-g) * x


def scan(x, g, h0, reset, axis, kind):
    a, b = factors(x, g, kind)
    cut = np.zeros(x.shape, bool) if reset is None else np.broadcast_to(reset, x.shape)
    a, b, cut = (np.moveaxis(v, axis, 0) for v in (a, b, cut))
    h = np.zeros(b.shape[1:]) if h0 is None else h0.astype(np.float64)
    out = np.empty(b.shape)
    for t in range(b.shape[0]):
        h = np.where(cut[t], 0.0, a[t] * np.where(cut[t], 0.0, h)) + b[t]
        out[t] = h
    return np.moveaxis(out, 0, axis), h


def scan_grad(dh, x, g, h, h0, reset, dstate, axis, kind):
    """(dx, dgate in g's shape, dh0)"""
    a, _ = factors(x, g, kind)
    cut = np.zeros(x.shape, bool) if reset is None else np.broadcast_to(reset, x.shape)
    a, cut, dh, hs, xs = (np.moveaxis(v, axis, 0) for v in (a, cut, dh, h, x))
    c = np.zeros(dh.shape[1:]) if dstate is None else dstate.astype(np.float64)
    G = np.empty(dh.shape)
    for t in range(dh.shape[0] - 1, -1, -1):
        G[t] = dh[t] + c
        c = np.where(cut[t], 0.0, a[t] * G[t])
    first = np.zeros(dh.shape[1:]) if h0 is None else h0
    before = np.where(cut, 0.0, np.concatenate([first[None], hs[:-1]])) if dh.shape[0] else hs
    if kind == "decay":
        dx, dg = G, G * before
    else:
        gm = np.moveaxis(np.broadcast_to(g, x.shape), axis, 0)
        dx, dg = sigmoid(-gm) * G, G * (before - xs) * a * sigmoid(-gm)
    dx, dg = np.moveaxis(dx, 0, axis), np.moveaxis(dg, 0, axis)
    return dx, unspread(dg, np.shape(g)), c


def unspread(v, shape):
    """Sums of `v` over the axes that `shape` was broadcast along."""
    full = (1,) * (v.ndim - len(shape)) + tuple(shape)
    axes = tuple(i for i in range(v.ndim) if full[i] == 1 and v.shape[i] != 1)
    return v.sum(axis=axes, keepdims=True).reshape(shape)


def scan_error(a, b, first, factor, term):
    """Bound on |computed h - h|: what flows from b[s] to h[t] is a product of t - s factors, each with a relative
    error of at most `factor`, of a b[s] with `term`, whatever the order in which they are multiplied and added."""
    a, b = np.abs(a), np.abs(b)
    H = np.abs(first)
    E = np.zeros(H.shape)
    out, mag = np.empty(b.shape), np.empty(b.shape)
    for t in range(b.shape[0]):
        E = a[t] * (E + factor * H) + term * b[t] + 2 * EPS * b[t]
        H = a[t] * H + b[t]
        out[t], mag[t] = E, H
    return out, mag


# ---- dropout ---------------------------------------------------------------------------------------
def philox4x32(counter, key, rounds=10):
    """Philox4x32 in Python's whole numbers: four words from a counter of four and a key of two."""
    c0, c1, c2, c3 = counter
    k0, k1 = key
    m = 0xFFFFFFFF
    for _ in range(rounds):
        p, q = 0xD2511F53 * c0, 0xCD9E8D57 * c2
        c0, c1, c2, c3 = (q >> 32) ^ c1 ^ k0, q & m, (p >> 32) ^ c3 ^ k1, p & m
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    return c0, c1, c2, c3


def kept(rows, width, p, seed, offset):
    """Which elements of (rows, width) dropout keeps."""
    m = 0xFFFFFFFF
    out = np.zeros((rows, -(-width // 8) * 8), bool)
    for r in range(rows):
        for b in range(out.shape[1] // 8):
            words = philox4x32((b, r, offset & m, offset >> 32), (seed & m, seed >> 32))
            out[r, 8 * b:8 * b + 8] = [h >= round(p * 65536) for w in words for h in (w & 0xFFFF, w >> 16)]
    return out[:, :width]


def keep_scale(p):
    n = round(p * 65536)
    return 0.0 if n == 65536 else 65536 / (65536 - n)


# ---- norms -----------------------------------------------------------------------------------------
def norm(v, kind, eps):
    """(normalised, 1 / deviation)"""
    if kind is None:
        return v, np.ones(v.shape[:-1] + (1,))
    if kind == "layer":
        v = v - v.mean(-1, keepdims=True)
    inv = 1 / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    return v * inv, inv


def norm_back(q, n, inv, kind):
    if kind is None:
        return q
    out = q - n * (q * n).mean(-1, keepdims=True)
    return inv * (out - q.mean(-1, keepdims=True) if kind == "layer" else out)


def act(g, kind):
    s = sigmoid(g)
    return (g * s, s * (1 + g * sigmoid(-g))) if kind == "silu" else (s, s * sigmoid(-g))


def block(x, residual, gate, w1, scale, w2, keep, o):
    """(r, y) of norm_residual; `keep`: 0, or the factor of what is kept; `o`: post, pre, gate_kind, eps"""
    n1, _ = norm(x, o["post"], o["eps"])
    v = n1 * w1 * (act(gate, o["gate_kind"])[0] if gate is not None else 1.0)
    r = residual + scale * np.where(keep == 0, 0.0, v * keep)
    return r, (norm(r, o["pre"], o["eps"])[0] * w2 if o["pre"] else None)


def block_grad(dr, dy, x, r, gate, w1, scale, w2, keep, o):
    """dict of the gradients of norm_residual, r as it was stored"""
    n1, inv1 = norm(x, o["post"], o["eps"])
    D = dr
    if o["pre"]:
        n2, inv2 = norm(r, o["pre"], o["eps"])
        D = D + norm_back(dy * w2, n2, inv2, o["pre"])
    a, slope = act(gate, o["gate_kind"]) if gate is not None else (1.0, 0.0)
    d = np.where(keep == 0, 0.0, n1 * w1 * a * keep)
    dv = np.where(keep == 0, 0.0, D * scale * keep)
    du = dv * a
    lead = tuple(range(x.ndim - 1))
    return {"dx": norm_back(du * w1, n1, inv1, o["post"]), "dresidual": D, "dgate": dv * n1 * w1 * slope,
            "dpost_weight": (du * n1).sum(lead), "dscale": (D * d).sum(lead),
            "dpre_weight": (dy * n2).sum(lead) if o["pre"] else None}
