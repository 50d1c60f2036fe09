"""The operators of a gated recurrent block: what is timed, on which inputs, and their plain forms.

A block of such a model runs, for every token: a norm, products that give the recurrence its inputs and gates, the
gated recurrence along the sequence, and, back on the residual stream, a norm of what came out, its gate, dropout and
a residual scale, with the next block's norm behind them.  The operators here are the ones between the products:

* ``gated_scan``           h[t] = g[t] h[t-1] + x[t]                            (kind "decay")
                           h[t] = s h[t-1] + (1 - s) x[t],  s = sigmoid(g[t])   (kind "blend")
                           h[-1] is the given state or 0; where ``reset`` is true, h[t-1] counts as 0 (packed sequences).
* ``gated_scan_grad``      its gradient: x, the gates and the first state.
* ``norm_residual``        u = norm(x) w_post,  v = u act(gate),  d = dropout(v),  r = residual + scale d,
                           y = norm(r) w_pre; either norm is "rms", "layer" or left out.
* ``norm_residual_grad``   its gradient, from x, r and what came back for r and y.
* ``dropout``              x / (1 - p) where kept, else 0, from a counter-based generator: no mask is stored.

Random bits: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with the
seed as its key.  The counter (c // 8, row, offset low, offset high) gives the eight 16-bit numbers of the columns
8 (c // 8) .. + 7 of a row, low halves first; column c is dropped where its number is below round(65536 p).
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # One token for each of 8 sequences that are being served: the state goes on by one step.
        {"name": "scan_step", "op": "scan", "layout": "seq", "batch": 8, "steps": 1, "width": 2048, "dtype": "bf16",
         "gates": "bf16", "kind": "blend", "reset": False, "state": True},
        # A training batch, channels innermost as the products leave them, gates as pre-activations.
        {"name": "scan_batch", "op": "scan", "layout": "seq", "batch": 8, "steps": 2048, "width": 4096, "dtype": "bf16",
         "gates": "bf16", "kind": "blend", "reset": False, "state": False},
        # One long row of packed documents: few channels, many steps, decays in 32 bits.
        {"name": "scan_packed", "op": "scan", "layout": "seq", "batch": 1, "steps": 65536, "width": 2048, "dtype": "bf16",
         "gates": "f32", "kind": "decay", "reset": True, "state": True},
        # Time innermost, as a convolution over time leaves it, with an odd length.
        {"name": "scan_time_last", "op": "scan", "layout": "time_last", "batch": 4, "steps": 5001, "width": 1500,
         "dtype": "f32", "gates": "f32", "kind": "decay", "reset": False, "state": False},
        # The training batch's gradient.
        {"name": "scan_grad_batch", "op": "scan_grad", "layout": "seq", "batch": 8, "steps": 2048, "width": 4096,
         "dtype": "bf16", "gates": "bf16", "kind": "blend", "reset": False, "state": False},
        # One decay for each head and step, shared by the head's channels, over packed rows of odd length.
        {"name": "scan_grad_heads", "op": "scan_grad", "layout": "heads", "batch": 2, "steps": 4099, "heads": 16,
         "width": 128, "dtype": "f16", "gates": "f32", "kind": "decay", "reset": True, "state": True},
        # The block's end for 16 sequences that are being served.
        {"name": "norm_step", "op": "norm", "rows": 16, "width": 4096, "dtype": "bf16", "stream": "bf16", "post": "rms",
         "pre": "rms", "gate": "silu", "p": 0.0},
        # The same in training, the residual stream in 32 bits, with dropout.
        {"name": "norm_batch", "op": "norm", "rows": 16384, "width": 4096, "dtype": "bf16", "stream": "f32", "post": "rms",
         "pre": "rms", "gate": "silu", "p": 0.1},
        {"name": "norm_grad_batch", "op": "norm_grad", "rows": 8192, "width": 4096, "dtype": "bf16", "stream": "bf16",
         "post": "rms", "pre": "rms", "gate": "silu", "p": 0.1},
        # An odd width in 32 bits, layer norms and a sigmoid gate.
        {"name": "norm_grad_odd", "op": "norm_grad", "rows": 5003, "width": 1111, "dtype": "f32", "stream": "f32",
         "post": "layer", "pre": "layer", "gate": "sigmoid", "p": 0.0},
        # Dropout of a training batch's activations, and of a slice of wider rows.
        {"name": "dropout_batch", "op": "dropout", "rows": 16384, "width": 4096, "dtype": "bf16", "p": 0.1, "pitch": 4096},
        {"name": "dropout_slice", "op": "dropout", "rows": 2047, "width": 999, "dtype": "f32", "p": 0.25, "pitch": 2048},
    ]


_MOST = 1.0e9  # bytes that a drawn case moves, at most


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["scan", "scan", "scan_grad", "scan_grad", "norm", "norm_grad", "dropout"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        c = {"op": op, "dtype": dtype}
        if op in ("scan", "scan_grad"):
            layout = rng.choice(["seq", "seq", "heads", "time_last"])
            c |= {"layout": layout, "batch": _log(rng, 1, 64),
                  "steps": _log(rng, 1, 65536), "width": _log(rng, 16, 8192),
                  "gates": rng.choice([dtype, "f32"]), "kind": rng.choice(["decay", "blend"]),
                  "reset": rng.random() < 0.4, "state": rng.random() < 0.5}
            if layout == "heads":
                c |= {"heads": _log(rng, 1, 64), "width": rng.choice([32, 64, 96, 128, 256, _log(rng, 16, 256)])}
        elif op in ("norm", "norm_grad"):
            c |= {"rows": _log(rng, 1, 65536), "width": rng.choice([_log(rng, 64, 16384), 8 * _log(rng, 8, 2048)]),
                  "stream": rng.choice([dtype, "f32"]), "post": rng.choice(["rms", "layer", "none"]),
                  "pre": rng.choice(["rms", "layer", "none"]), "gate": rng.choice(["silu", "sigmoid", "none"]),
                  "p": rng.choice([0.0, 0.0, 0.1, 0.2])}
        else:
            width = _log(rng, 64, 16384)
            c |= {"rows": _log(rng, 1, 65536), "width": width, "p": rng.choice([0.1, 0.2, 0.5]),
                  "pitch": width if rng.random() < 0.5 else width + rng.randrange(1, 64)}
        b = work(c)["bytes"]
        if 1e4 <= b <= _MOST:
            return c


# ---- shapes -------------------------------------------------------------------------------------
def _scan_shapes(c):
    """(x, gate, reset, state, time axis)"""
    b, t, w = c["batch"], c["steps"], c["width"]
    if c["layout"] == "seq":
        return (b, t, w), (b, t, w), (b, t, 1), (b, w), 1
    if c["layout"] == "heads":
        return (b, t, c["heads"], w), (b, t, c["heads"], 1), (b, t, 1, 1), (b, c["heads"], w), 1
    return (b, w, t), (b, w, t), (b, 1, t), (b, w), 2


def _threshold(p):
    return int(round(p * 65536))


def _tensors(c, seed):
    """The case's inputs, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[c["dtype"]]

    def normal(shape, dtype, mean=0.0, std=1.0):
        return torch.randn(shape, dtype=torch.float32, device="cuda", generator=g).mul_(std).add_(mean).to(dtype)

    def chance(shape, p):
        return torch.rand(shape, device="cuda", generator=g) < p

    t = {}
    if c["op"] in ("scan", "scan_grad"):
        xs, gs, rs, ss, axis = _scan_shapes(c)
        gt = _DT[c["gates"]]
        t["x"] = normal(xs, dt)
        # decays mostly near 1 and now and then a low one; pre-activations whose sigmoid is like that
        logits = normal(gs, torch.float32, 2.5, 1.5)
        t["gate"] = (torch.sigmoid(logits) if c["kind"] == "decay" else logits).to(gt)
        del logits
        if c["reset"]:
            t["reset"] = chance(rs, 1.0 / 300)
        if c["state"]:
            t["h0"] = normal(ss, torch.float32)
        if c["op"] == "scan_grad":
            t["h"] = normal(xs, dt)
            t["dh"] = normal(xs, dt)
            if c["state"]:
                t["dstate"] = normal(ss, torch.float32)
    elif c["op"] in ("norm", "norm_grad"):
        s, w, st = (c["rows"], c["width"]), (c["width"],), _DT[c["stream"]]
        t["x"] = normal(s, dt, 0.1)
        if c["gate"] != "none":
            t["gate"] = normal(s, dt)
        if c["post"] != "none":
            t["post_weight"] = normal(w, torch.float32, 1.0, 0.1)
        if c["pre"] != "none":
            t["pre_weight"] = normal(w, torch.float32, 1.0, 0.1)
        t["scale"] = normal(w, torch.float32, 0.5, 0.1)
        t["residual"] = normal(s, st, 0.0, 2.0)  # of the gradient: the stream behind the block
        if c["op"] == "norm_grad":
            t["dr"] = normal(s, st)
            if c["pre"] != "none":
                t["dy"] = normal(s, dt)
    else:
        t["x"] = normal((c["rows"], c["pitch"]), dt)[:, :c["width"]]
    return t


def prepare(case, seed):
    c = dict(case)
    t = _tensors(c, seed)
    state = {"case": c, "t": t, "seed": seed}
    if own:  # the arrays over these tensors, and those that take the results: a program keeps both
        import musapy_amd as ms

        dt = _DT[c["dtype"]]
        like = {k: v.shape for k, v in t.items()}
        f32 = torch.float32
        if c["op"] == "scan":
            outs = [(like["x"], dt), (_scan_shapes(c)[3], f32)]
        elif c["op"] == "scan_grad":
            outs = [(like["x"], dt), (like["gate"], _DT[c["gates"]])] + ([(like["h0"], f32)] if c["state"] else [])
        elif c["op"] == "norm":
            outs = [(like["x"], _DT[c["stream"]])] + ([(like["x"], dt)] if c["pre"] != "none" else [])
        elif c["op"] == "norm_grad":
            outs = [(like["x"], dt), (like["x"], _DT[c["stream"]])] + ([(like["x"], dt)] if "gate" in t else [])
            outs += [((c["width"],), f32)] * (1 + ("post_weight" in t) + ("pre_weight" in t))
        else:
            outs = [(like["x"], dt)]
        state["out_t"] = [torch.empty(s, dtype=d, device="cuda") for s, d in outs]
        state["ms"] = ms
        state["a"] = {k: ms.from_dlpack(v) for k, v in t.items()}
        state["out"] = [ms.from_dlpack(o) for o in state["out_t"]]
    return state


def run(state):
    c = state["case"]
    return (_run_own if own else _run_plain)(c, state)


def _run_own(c, state):
    ms, a, o = state["ms"], state["a"], state["out"]
    op = c["op"]
    if op == "scan":
        ms.gated_scan(a["x"], a["gate"], a.get("h0"), reset=a.get("reset"), axis=_scan_shapes(c)[4], kind=c["kind"],
                      out=o[0], state_out=o[1])
    elif op == "scan_grad":
        ms.gated_scan_grad(a["dh"], a["x"], a["gate"], a["h"], a.get("h0"), reset=a.get("reset"), dstate=a.get("dstate"),
                           axis=_scan_shapes(c)[4], kind=c["kind"], out=tuple(o) if c["state"] else (o[0], o[1], None))
    elif op == "norm":
        ms.norm_residual(a["x"], a["residual"], gate=a.get("gate"), post_weight=a.get("post_weight"), scale=a["scale"],
                         pre_weight=a.get("pre_weight"), out=tuple(o) if c["pre"] != "none" else (o[0], None),
                         **_norm_options(c, state["seed"]))
    elif op == "norm_grad":
        q = iter(o[2:])
        out = (o[0], o[1], next(q) if "gate" in a else None, next(q) if "post_weight" in a else None, next(q),
               next(q) if "pre_weight" in a else None)
        ms.norm_residual_grad(a["dr"], a.get("dy"), a["x"], a["residual"], gate=a.get("gate"),
                              post_weight=a.get("post_weight"), scale=a["scale"], pre_weight=a.get("pre_weight"), out=out,
                              **_norm_options(c, state["seed"]))
    else:
        ms.dropout(a["x"], c["p"], seed=state["seed"], offset=7, out=o[0])
    return state["out_t"]


def _norm_options(c, seed):
    return {"post": None if c["post"] == "none" else c["post"], "pre": None if c["pre"] == "none" else c["pre"],
            "gate_kind": "silu" if c["gate"] == "none" else c["gate"], "eps": 1e-5, "p": c["p"], "seed": seed, "offset": 3}


# ---- the plain forms ------------------------------------------------------------------------------
def _running(a, b, axis, first):
    """h[t] = a[t] h[t-1] + b[t] for all t at once: pairs (a, b) are composed over distances 1, 2, 4, ..."""
    steps, d = b.shape[axis], 1
    if first is not None:
        f = b.narrow(axis, 0, 1) + a.narrow(axis, 0, 1) * first.unsqueeze(axis)
        b = torch.cat([f, b.narrow(axis, 1, steps - 1)], axis)
    while d < steps:
        late, early = a.narrow(axis, d, steps - d), a.narrow(axis, 0, steps - d)
        b = torch.cat([b.narrow(axis, 0, d), late * b.narrow(axis, 0, steps - d) + b.narrow(axis, d, steps - d)], axis)
        if 2 * d < steps:
            a = torch.cat([a.narrow(axis, 0, d), late * early], axis)
        d *= 2
    return b


def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _kept(c, seed, offset, rows, width):
    """Truth values (rows, width): which elements dropout keeps."""
    m = 0xFFFFFFFF
    k0, k1 = seed & m, (seed >> 32) & m
    blocks = (width + 7) // 8
    x0 = torch.arange(blocks, device="cuda", dtype=torch.int64)[None, :].expand(rows, blocks)
    x1 = torch.arange(rows, device="cuda", dtype=torch.int64)[:, None].expand(rows, blocks)
    x2, x3 = torch.full_like(x0, offset & m), torch.full_like(x0, (offset >> 32) & m)
    for _ in range(10):  # the generator's ten rounds
        p, q = x0 * 0xD2511F53, x2 * 0xCD9E8D57  # the low 64 bits of each product: the sign bit is masked off below
        x0, x1, x2, x3 = ((q >> 32) & m) ^ x1 ^ k0, q & m, ((p >> 32) & m) ^ x3 ^ k1, p & m
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    words = torch.stack([x0, x1, x2, x3], -1)
    halves = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, blocks * 8)
    return halves[:, :width] >= _threshold(c["p"])


def _keep_scale(p):
    """1 / (1 - p) for the p that 16 bits hold."""
    return 65536.0 / (65536 - _threshold(p))


def _norm(x, kind, eps=1e-5):
    """(normalised x, 1 / its deviation)"""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r, r


def _norm_back(g, n, r, kind):
    """The gradient of the norm's input, from that of its output."""
    g2 = g - n * (g * n).mean(-1, keepdim=True)
    return r * (g2 - g.mean(-1, keepdim=True) if kind == "layer" else g2)


def _activation(g, kind):
    """(act(g), its derivative)"""
    s = _sigmoid(g)
    return (g * s, s * (1.0 + g * (1.0 - s))) if kind == "silu" else (s, s * (1.0 - s))


def _run_plain(c, state):
    t = state["t"]
    f = {k: v.float() for k, v in t.items() if k != "reset"}
    dt = _DT[c["dtype"]]
    op = c["op"]
    if op in ("scan", "scan_grad"):
        axis = _scan_shapes(c)[4]
        x, g = f["x"], f["gate"]
        blend = c["kind"] == "blend"
        a = _sigmoid(g) if blend else g
        cut = torch.where(t["reset"], torch.zeros((), device="cuda"), a) if c["reset"] else a
        steps = x.shape[axis]
        if op == "scan":
            h = _running(cut.expand_as(x), (1.0 - a) * x if blend else x, axis, f.get("h0"))
            return [h.to(dt), h.select(axis, steps - 1).clone()]
        first = f["h0"].unsqueeze(axis) if c["state"] else torch.zeros_like(x.narrow(axis, 0, 1))
        before = torch.cat([first, f["h"].narrow(axis, 0, steps - 1)], axis)
        if c["reset"]:
            before = torch.where(t["reset"], torch.zeros((), device="cuda"), before)
        # what flows into h[t] from later steps: q[t] = cut[t+1] (dh[t+1] + q[t+1]), run over reversed time
        back = cut.expand_as(x).flip(axis)
        late = f["dh"].flip(axis)
        if c["state"]:
            late = torch.cat([late.narrow(axis, 0, 1) + f["dstate"].unsqueeze(axis), late.narrow(axis, 1, steps - 1)], axis)
        flow = torch.cat([torch.zeros_like(late.narrow(axis, 0, 1)), back.narrow(axis, 0, steps - 1)], axis)
        total = _running(flow, late, axis, None).flip(axis)
        if blend:
            dx, dg = (1.0 - a) * total, total * (before - x) * a * (1.0 - a)
        else:
            dx, dg = total, total * before
        if c["layout"] == "heads":
            dg = dg.sum(-1, keepdim=True)
        out = [dx.to(dt), dg.to(_DT[c["gates"]])]
        if c["state"]:
            out.append((cut.narrow(axis, 0, 1) * total.narrow(axis, 0, 1)).squeeze(axis))
        return out
    if op == "dropout":
        keep = _kept(c, state["seed"], 7, c["rows"], c["width"])
        return [torch.where(keep, f["x"] * _keep_scale(c["p"]), torch.zeros((), device="cuda")).to(dt)]

    post, pre, gated = c["post"] != "none", c["pre"] != "none", c["gate"] != "none"
    x = f["x"]
    n1, r1 = _norm(x, c["post"]) if post else (x, None)
    u = n1 * f["post_weight"] if post else n1
    act, slope = _activation(f["gate"], c["gate"]) if gated else (None, None)
    v = u * act if gated else u
    keep = _kept(c, state["seed"], 3, c["rows"], c["width"]) if c["p"] else None
    zero = torch.zeros((), device="cuda")
    d = torch.where(keep, v * _keep_scale(c["p"]), zero) if c["p"] else v
    if op == "norm":
        r = f["residual"] + f["scale"] * d
        return [r.to(_DT[c["stream"]])] + ([(_norm(r, c["pre"])[0] * f["pre_weight"]).to(dt)] if pre else [])
    total = f["dr"]
    if pre:
        n2, r2 = _norm(f["residual"], c["pre"])
        total = total + _norm_back(f["dy"] * f["pre_weight"], n2, r2, c["pre"])
    dd = total * f["scale"]
    dv = torch.where(keep, dd * _keep_scale(c["p"]), zero) if c["p"] else dd
    du = dv * act if gated else dv
    dx = _norm_back(du * f["post_weight"], n1, r1, c["post"]) if post else du
    out = [dx.to(dt), total.to(_DT[c["stream"]])]
    if gated:
        out.append((dv * u * slope).to(dt))
    if post:
        out.append((du * n1).sum(0))
    out.append((total * d).sum(0))
    if pre:
        out.append((f["dy"] * n2).sum(0))
    return out


# ---- what the path cannot do without -----------------------------------------------------------------
def work(case):
    """Each input read once, each output written once; a few operations for each element."""
    c, op = case, case["op"]
    es = _SIZE[c["dtype"]]
    if op in ("scan", "scan_grad"):
        shapes = _scan_shapes(c)[:4]
        n, ng, nr, ns = (math.prod(s) for s in shapes)
        gs = _SIZE[c["gates"]]
        resets = nr if c["reset"] else 0
        if op == "scan":
            return {"bytes": 2 * n * es + ng * gs + resets + 4 * ns * (2 if c["state"] else 1),
                    "flops": n * (8 if c["kind"] == "blend" else 2)}
        arrays = 4 if c["kind"] == "blend" else 3  # dh, h and dx; blend reads x too
        return {"bytes": arrays * n * es + 2 * ng * gs + resets + (12 * ns if c["state"] else 0),
                "flops": n * (14 if c["kind"] == "blend" else 5)}
    n, w = c["rows"] * c["width"], c["width"]
    if op == "dropout":
        return {"bytes": 2 * n * es, "flops": 2 * n}
    ss = _SIZE[c["stream"]]
    post, pre, gate = c["post"] != "none", c["pre"] != "none", c["gate"] != "none"
    weights = 4 * w * (1 + post + pre)
    if op == "norm":
        return {"bytes": n * (es * (1 + gate + pre) + 2 * ss) + weights,
                "flops": n * (2 + 4 * post + 4 * pre + 6 * gate)}
    return {"bytes": n * (es * (2 + 2 * gate + pre) + (3 if pre else 2) * ss) + 2 * weights,
            "flops": n * (4 + 10 * post + 10 * pre + 12 * gate)}


# ---- the definitions in 64 bits --------------------------------------------------------------------------
def _dropped(c, seed, offset):
    if not c["p"]:
        return None, 1.0
    import numpy as np

    share = round(c["p"] * 65536) / 65536
    lost = np.concatenate([_numbers(c, seed, offset, r) for r in range(0, c["rows"], 1024)]) < share * 65536
    return torch.from_numpy(lost).to("cuda"), 1.0 / (1.0 - share)


def _numbers(c, seed, offset, first):
    """The generator's 16-bit numbers of up to 1024 rows from `first` on, on the host in unsigned 64-bit arithmetic."""
    import numpy as np

    n = min(1024, c["rows"] - first)
    u = np.uint64
    mask, sh = u(0xFFFFFFFF), u(32)
    blocks = -(-c["width"] // 8)
    a = np.broadcast_to(np.arange(blocks, dtype=u), (n, blocks))
    b = np.broadcast_to(np.arange(first, first + n, dtype=u)[:, None], (n, blocks))
    d, e = np.full((n, blocks), offset & 0xFFFFFFFF, u), np.full((n, blocks), offset >> 32, u)
    ka, kb = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        s, t = a * u(0xD2511F53), d * u(0xCD9E8D57)
        a, b, d, e = (t >> sh) ^ b ^ u(ka), t & mask, (s >> sh) ^ e ^ u(kb), s & mask
        ka, kb = (ka + 0x9E3779B9) & 0xFFFFFFFF, (kb + 0xBB67AE85) & 0xFFFFFFFF
    parts = [h for w in (a, b, d, e) for h in (w & u(0xFFFF), w >> u(16))]
    return np.stack(parts, -1).astype(np.uint16).reshape(n, blocks * 8)[:, :c["width"]]


def _exact_scan(c, t):
    axis = _scan_shapes(c)[4]
    x = t["x"].double().movedim(axis, 0)
    gate = t["gate"].double().movedim(axis, 0)
    if c["kind"] == "blend":
        factor, part = torch.sigmoid(gate), torch.sigmoid(-gate)
    else:
        factor, part = gate, None
    through = factor.masked_fill(t["reset"].movedim(axis, 0), 0.0) if c["reset"] else factor
    steps = x.shape[0]
    if c["op"] == "scan":
        h = torch.zeros_like(x[0]) if not c["state"] else t["h0"].double()
        every = x * part if part is not None else x.clone()
        for k in range(steps):
            h = torch.addcmul(every[k], through[k].expand_as(h), h, out=every[k])
        return [every.movedim(0, axis), every[-1].clone()]
    total = t["dh"].double().movedim(axis, 0).contiguous().clone()
    if c["state"]:
        total[-1] += t["dstate"].double()
    for k in range(steps - 2, -1, -1):
        torch.addcmul(total[k], through[k + 1].expand_as(total[k]), total[k + 1], out=total[k])
    past = torch.empty_like(x)
    past[0] = t["h0"].double() if c["state"] else 0.0
    past[1:] = t["h"].double().movedim(axis, 0)[:-1]
    if c["reset"]:
        past.masked_fill_(t["reset"].movedim(axis, 0), 0.0)
    if part is not None:
        dx, dgate = total * part, total * (past - x) * factor * part
    else:
        dx, dgate = total, total * past
    if c["layout"] == "heads":
        dgate = dgate.sum(-1, keepdim=True)
    out = [dx.movedim(0, axis), dgate.movedim(0, axis)]
    return out + [through[0] * total[0]] if c["state"] else out


def _exact_norm(c, t, seed):
    eps = 1e-5
    lost, up = _dropped(c, seed, 3)

    def whiten(v, kind):
        if kind == "none":
            return v, None
        v = v - v.mean(1, keepdim=True) if kind == "layer" else v
        inv = 1.0 / torch.sqrt(v.pow(2).mean(1, keepdim=True) + eps)
        return v * inv, inv

    def unwhiten(grad, n, inv, kind):
        if kind == "none":
            return grad
        along = n * (grad * n).mean(1, keepdim=True)
        flat = grad.mean(1, keepdim=True) if kind == "layer" else 0.0
        return inv * (grad - along - flat)

    wide = {k: v.double() for k, v in t.items()}
    one = torch.ones((), dtype=torch.float64, device="cuda")
    w1, w2, scale = wide.get("post_weight", one), wide.get("pre_weight", one), wide["scale"]
    n1, inv1 = whiten(wide["x"], c["post"])
    if c["gate"] != "none":
        sg = torch.sigmoid(wide["gate"])
        act = wide["gate"] * sg if c["gate"] == "silu" else sg
        slope = sg + wide["gate"] * sg * (1 - sg) if c["gate"] == "silu" else sg * (1 - sg)
    else:
        act, slope = one, None
    through = one * up if lost is None else torch.full(lost.shape, up, dtype=torch.float64, device="cuda").masked_fill_(lost, 0.0)
    d = n1 * w1 * act * through
    if c["op"] == "norm":
        r = wide["residual"] + scale * d
        return [r] + ([whiten(r, c["pre"])[0] * w2] if c["pre"] != "none" else [])
    n2, inv2 = whiten(wide["residual"], c["pre"])
    total = wide["dr"]
    if c["pre"] != "none":
        total = total + unwhiten(wide["dy"] * w2, n2, inv2, c["pre"])
    dv = total * scale * through
    out = [unwhiten(dv * act * w1, n1, inv1, c["post"]), total]
    if slope is not None:
        out.append(dv * n1 * w1 * slope)
    if c["post"] != "none":
        out.append((dv * act * n1).sum(0))
    out.append((total * d).sum(0))
    if c["pre"] != "none":
        out.append((wide["dy"] * n2).sum(0))
    return out


def exact(case, seed):
    c = dict(case)
    if c["op"] in ("scan", "scan_grad"):
        return _exact_scan(c, _tensors(c, seed))
    if c["op"] in ("norm", "norm_grad"):
        return _exact_norm(c, _tensors(c, seed), seed)
    lost, up = _dropped(c, seed, 7)
    return [(_tensors(c, seed)["x"].double() * up).masked_fill_(lost, 0.0)]
