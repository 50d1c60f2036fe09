"""The operators at a language model's two ends, over its vocabulary: what is timed, on which inputs, and their plain forms.

In front of a model's blocks a token becomes a row of a table; behind them a row of logits, as wide as the vocabulary,
becomes a loss in training or the next token in serving.  The operators here are those ends:

* ``embedding``          y[n] = scale table[tokens[n]]; a token outside the table (padding) gives a row of zeros.
* ``embedding_grad``     dtable[v] = scale sum of dy[n] over the n with tokens[n] = v: every row of the table, zeros included.
* ``distill_loss``       p = softmax(teacher / T) over the teacher's top entries of a row (those whose index is a column),
                         q = softmax(z / T), s = softmax(z);
                         loss = weight T^2 sum_k p_k (log p_k - log q[i_k]) - (1 - weight) log s[label].
                         The first term is 0 without entries, the second where the label is no column.  It also gives the
                         highest logit m, log sum exp((z - m) / T) and log sum exp(z - m), 0 where a row has no use for one.
* ``distill_loss_grad``  dz = dloss (weight T (q - p) + (1 - weight) (s - one-hot(label))).
* ``adjust_logits``      for each sequence, with c the number of times a token is in its history:
                         z = (z > 0 ? z / repetition : z repetition) - (frequency c + presence) where c > 0; z += bias;
                         z = -inf where the mask does not allow the token.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32, "i64": torch.int64}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4, "i64": 8}
_PAD = 0.02       # share of tokens that are padding
_UNLABELLED = 0.03


def listed():
    return [
        # One token for each of 16 sequences that are being served.
        {"name": "embed_step", "op": "embed", "tokens": 16, "vocab": 32768, "width": 4096, "dtype": "bf16", "to": "bf16",
         "ids": "i32"},
        # A training batch from a table of 32-bit weights into a 16-bit stream.
        {"name": "embed_batch", "op": "embed", "tokens": 16384, "vocab": 131072, "width": 4096, "dtype": "f32", "to": "bf16",
         "ids": "i64"},
        # That batch's gradient, in the table's type.
        {"name": "embed_grad_batch", "op": "embed_grad", "tokens": 16384, "vocab": 131072, "width": 2048, "dtype": "bf16",
         "to": "f32", "ids": "i64"},
        # Packed rows of odd sizes.
        {"name": "embed_grad_odd", "op": "embed_grad", "tokens": 5003, "vocab": 50001, "width": 1111, "dtype": "f32",
         "to": "f32", "ids": "i32"},
        # A few rows of a small model's distillation: the teacher's top 8, nothing else.
        {"name": "distill_small", "op": "distill", "rows": 64, "vocab": 32768, "entries": 8, "dtype": "bf16",
         "teacher": "f32", "ids": "i64", "temperature": 1.0, "weight": 1.0},
        # A training batch with labels beside the teacher's top 64.
        {"name": "distill_batch", "op": "distill", "rows": 4096, "vocab": 131072, "entries": 64, "dtype": "bf16",
         "teacher": "bf16", "ids": "i32", "temperature": 2.0, "weight": 0.5},
        # Logits in 32 bits and odd sizes.
        {"name": "distill_odd", "op": "distill", "rows": 1023, "vocab": 50001, "entries": 20, "dtype": "f32",
         "teacher": "f32", "ids": "i64", "temperature": 1.5, "weight": 0.7},
        # Both gradients.
        {"name": "distill_grad_batch", "op": "distill_grad", "rows": 4096, "vocab": 131072, "entries": 64, "dtype": "bf16",
         "teacher": "bf16", "ids": "i32", "temperature": 2.0, "weight": 0.5},
        {"name": "distill_grad_odd", "op": "distill_grad", "rows": 1023, "vocab": 50001, "entries": 20, "dtype": "f32",
         "teacher": "f32", "ids": "i64", "temperature": 1.5, "weight": 0.7},
        # Four sequences that are being served, with penalties over short answers.
        {"name": "adjust_step", "op": "adjust", "rows": 4, "vocab": 32768, "dtype": "f32", "to": "f32", "history": 500,
         "ids": "i32", "bias": "none", "entries": 0, "allowed": "none"},
        # A large serving batch under grammars: packed masks, a few biased tokens, 16-bit logits into 32 bits.
        {"name": "adjust_batch", "op": "adjust", "rows": 256, "vocab": 131072, "dtype": "bf16", "to": "f32", "history": 4096,
         "ids": "i32", "bias": "sparse", "entries": 16, "allowed": "bits"},
        # Long histories, one bias for all, a mask of truth values, an odd vocabulary.
        {"name": "adjust_long", "op": "adjust", "rows": 32, "vocab": 50001, "dtype": "f16", "to": "f16", "history": 30000,
         "ids": "i64", "bias": "dense", "entries": 0, "allowed": "bool"},
    ]


_MOST = 1.2e9  # bytes that a drawn case moves, at most


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["embed", "embed_grad", "embed_grad", "distill", "distill", "distill_grad", "adjust", "adjust"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        vocab = rng.choice([_log(rng, 1000, 262144), 64 * _log(rng, 16, 4096)])
        c = {"op": op, "vocab": vocab, "dtype": dtype, "ids": rng.choice(["i32", "i64"])}
        if op in ("embed", "embed_grad"):
            c |= {"tokens": _log(rng, 1, 131072), "width": rng.choice([_log(rng, 64, 16384), 8 * _log(rng, 8, 2048)]),
                  "to": rng.choice([dtype, "f32"])}
        elif op in ("distill", "distill_grad"):
            both = rng.random() < 0.5
            c |= {"rows": _log(rng, 1, 16384), "entries": _log(rng, 1, 256), "teacher": rng.choice([dtype, "f32"]),
                  "temperature": rng.choice([1.0, 1.0, 2.0, 4.0, 0.7]), "weight": rng.choice([0.5, 0.9]) if both else 1.0}
        else:
            c |= {"rows": _log(rng, 1, 512), "to": rng.choice([dtype, "f32"]),
                  "history": rng.choice([0, _log(rng, 1, 32768), _log(rng, 1, 32768)]),
                  "bias": rng.choice(["none", "dense", "sparse"]), "entries": 0,
                  "allowed": rng.choice(["none", "bits", "bits", "bool"])}
            if c["bias"] == "sparse":
                c["entries"] = _log(rng, 1, 256)
        b = work(c)["bytes"]
        if 1e4 <= b <= _MOST:
            return c


# ---- inputs -----------------------------------------------------------------------------------------
def _tensors(c, seed):
    """The case's inputs, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, v, dt, ids = c["op"], c["vocab"], _DT[c["dtype"]], _DT[c["ids"]]

    def normal(shape, dtype, mean=0.0, std=1.0):
        return torch.randn(shape, dtype=torch.float32, device="cuda", generator=g).mul_(std).add_(mean).to(dtype)

    def uniform(shape, lo=0.0, hi=1.0):
        return torch.rand(shape, device="cuda", generator=g) * (hi - lo) + lo

    def tokens(shape, pad):
        """Tokens as text has them: the share of token v falls as 1 / (v + 1).  Some are padding, -1."""
        t = (torch.exp(uniform(shape) * math.log(v + 1)) - 1.0).long().clamp_(0, v - 1)
        return torch.where(uniform(shape) < pad, -1, t).to(ids)

    def distinct(rows, k):
        """k columns of each row, all different."""
        step = int(v * 0.381966) | 1
        while math.gcd(step, v) != 1:
            step += 2
        first = torch.randint(0, v, (rows, 1), device="cuda", generator=g)
        return (first + step * torch.arange(k, device="cuda")) % v

    t = {}
    if op == "embed":
        t["table"] = normal((v, c["width"]), dt, 0.0, 0.02)
        t["tokens"] = tokens((c["tokens"],), _PAD)
    elif op == "embed_grad":
        t["dy"] = normal((c["tokens"], c["width"]), dt)
        t["tokens"] = tokens((c["tokens"],), _PAD)
    elif op in ("distill", "distill_grad"):
        rows, k = c["rows"], c["entries"]
        z = normal((rows, v), torch.float32, 0.0, 2.0)
        index = distinct(rows, k)
        teacher = normal((rows, k), torch.float32, 12.0, 2.5).sort(-1, descending=True).values
        # the student has learnt some of it
        z.scatter_(1, index, 0.6 * teacher + normal((rows, k), torch.float32))
        t["logits"] = z.to(dt)
        # a row's last entries are missing here and there
        keep = torch.randint(1, k + 1, (rows, 1), device="cuda", generator=g)
        keep = torch.where(uniform((rows, 1)) < 0.2, keep, k)
        t["index"] = torch.where(torch.arange(k, device="cuda") < keep, index, -1).to(ids)
        t["teacher"] = teacher.to(_DT[c["teacher"]])
        if c["weight"] < 1.0:
            t["labels"] = torch.where(uniform((rows,)) < _UNLABELLED, -100, index[:, 0]).to(ids)
        if op == "distill_grad":
            t["dloss"] = uniform((rows,), 0.5, 1.5) / rows
            t["sums"] = _log_sums(c, t)
    else:
        rows = c["rows"]
        t["logits"] = normal((rows, v), dt, 0.0, 3.0)
        if c["history"]:
            t["history"] = tokens((rows, c["history"]), 0.0)
            t["lengths"] = torch.randint(c["history"] // 2, c["history"] + 1, (rows,), device="cuda", generator=g).to(ids)
            t["repetition"] = uniform((rows,), 1.0, 1.4)
            t["presence"] = uniform((rows,), 0.0, 1.5)
            t["frequency"] = uniform((rows,), 0.0, 0.5)
        if c["bias"] == "dense":
            t["bias"] = normal((v,), torch.float32)
        elif c["bias"] == "sparse":
            t["bias"] = normal((rows, c["entries"]), torch.float32, 0.0, 4.0)
            t["bias_index"] = distinct(rows, c["entries"]).to(ids)
        if c["allowed"] != "none":
            # a grammar leaves some sequences free and others few tokens
            free = uniform((rows, 1)) < 0.4
            if c["allowed"] == "bits":
                w = [torch.randint(-(1 << 31), 1 << 31, (rows, (v + 31) // 32), device="cuda", generator=g) for _ in range(3)]
                t["allowed"] = torch.where(free, -1, w[0] & w[1] & w[2]).to(torch.int32)
            else:
                t["allowed"] = free | (uniform((rows, v)) < 0.1)
    return t


def _uses(c, t):
    """Truth values (rows, 1): rows with an entry of the teacher's, and rows with a label."""
    index = t["index"].long()
    first = ((index >= 0) & (index < c["vocab"])).any(1, keepdim=True)
    if "labels" not in t:
        return first, None
    label = t["labels"].long()[:, None]
    return first, (label >= 0) & (label < c["vocab"])


def _log_sums(c, t):
    """What the loss keeps for its gradient: (rows, 3), in 64 bits, rounded."""
    out = torch.zeros(c["rows"], 3, device="cuda")
    first, second = _uses(c, t)
    step = max(1, (1 << 28) // c["vocab"])
    for i in range(0, c["rows"], step):
        z = t["logits"][i:i + step].double()
        top = z.max(1, keepdim=True).values
        for j, (used, temp) in enumerate(((first, c["temperature"]), (second, 1.0)), 1):
            if used is not None:
                u = used[i:i + step]
                s = torch.log(torch.exp((z - top) / temp).sum(1, keepdim=True))
                out[i:i + step, j:j + 1] = torch.where(u, s, 0.0).float()
                out[i:i + step, :1] = torch.where(u, top.float(), out[i:i + step, :1])
    return out


def prepare(case, seed):
    c = dict(case)
    t = _tensors(c, seed)
    state = {"case": c, "t": t}
    if own:  # the arrays over these tensors, and those that take the results: a program keeps both
        import musapy_amd as ms

        op, f32 = c["op"], torch.float32
        if op == "embed":
            outs = [((c["tokens"], c["width"]), _DT[c["to"]])]
        elif op == "embed_grad":
            outs = [((c["vocab"], c["width"]), _DT[c["to"]])]
        elif op == "distill":
            outs = [((c["rows"],), f32), ((c["rows"], 3), f32)]
        elif op == "distill_grad":
            outs = [(t["logits"].shape, _DT[c["dtype"]])]
        else:
            outs = [(t["logits"].shape, _DT[c["to"]])]
        state["out_t"] = [torch.empty(s, dtype=d, device="cuda") for s, d in outs]
        state["ms"] = ms
        state["a"] = {k: ms.from_dlpack(x) for k, x in t.items()}
        state["out"] = [ms.from_dlpack(o) for o in state["out_t"]]
    return state


def run(state):
    c = state["case"]
    return (_run_own if own else _run_plain)(c, state)


_SCALE = 8.0  # of the embedding


def _run_own(c, state):
    ms, a, o = state["ms"], state["a"], state["out"]
    op = c["op"]
    if op == "embed":
        ms.embedding(a["table"], a["tokens"], _SCALE, out=o[0])
    elif op == "embed_grad":
        ms.embedding_grad(a["dy"], a["tokens"], c["vocab"], _SCALE, out=o[0])
    elif op == "distill":
        ms.distill_loss(a["logits"], a["index"], a["teacher"], a.get("labels"), temperature=c["temperature"],
                        weight=c["weight"], out=tuple(o))
    elif op == "distill_grad":
        ms.distill_loss_grad(a["dloss"], a["logits"], a["sums"], a["index"], a["teacher"], a.get("labels"),
                             temperature=c["temperature"], weight=c["weight"], out=o[0])
    else:
        penalties = {k: a[k] for k in ("repetition", "presence", "frequency") if k in a}
        ms.adjust_logits(a["logits"], a.get("history"), a.get("lengths"), bias=a.get("bias"), bias_index=a.get("bias_index"),
                         allowed=a.get("allowed"), out=o[0], **penalties)
    return state["out_t"]


# ---- the plain forms ------------------------------------------------------------------------------
def _teacher(c, t):
    """(indices with 0 for what is no column, p with 0 there, log p with 0 where p is 0)"""
    index = t["index"].long()
    valid = (index >= 0) & (index < c["vocab"])
    v = torch.where(valid, t["teacher"].float(), -math.inf) / c["temperature"]
    top = v.max(1, keepdim=True).values
    e = torch.exp(v - torch.where(top > -math.inf, top, 0.0))
    p = e / e.sum(1, keepdim=True).clamp_min(1e-30)
    return torch.where(valid, index, 0), p, torch.where(p > 0.0, torch.log(p), 0.0)


def _run_plain(c, state):
    t = state["t"]
    op, v = c["op"], c["vocab"]
    if op == "embed":
        k = t["tokens"].long()
        inside = (k >= 0) & (k < v)
        rows = t["table"][torch.where(inside, k, 0)].float() * _SCALE
        return [torch.where(inside[:, None], rows, 0.0).to(_DT[c["to"]])]
    if op == "embed_grad":
        k = t["tokens"].long()
        at = torch.where((k >= 0) & (k < v), k, v)
        sums = torch.zeros(v + 1, c["width"], device="cuda").index_add_(0, at, t["dy"].float())
        return [(sums[:v] * _SCALE).to(_DT[c["to"]])]
    if op in ("distill", "distill_grad"):
        temp, weight = c["temperature"], c["weight"]
        z = t["logits"].float()
        index, p, log_p = _teacher(c, t)
        first, second = _uses(c, t)
        if op == "distill":
            top = z.max(1, keepdim=True).values
            soft = torch.log(torch.exp((z - top) / temp).sum(1, keepdim=True))
            log_q = (z.gather(1, index) - top) / temp - soft
            loss = weight * temp * temp * torch.where(p > 0.0, p * (log_p - log_q), 0.0).sum(1)
            hard = torch.zeros_like(soft)
            used = first
            if second is not None:
                hard = torch.where(second, torch.log(torch.exp(z - top).sum(1, keepdim=True)), 0.0)
                at = z.gather(1, torch.where(second, t["labels"].long()[:, None], 0))
                loss = loss + (1.0 - weight) * torch.where(second, top - at + hard, 0.0)[:, 0]
                used = first | second
            return [loss, torch.cat([torch.where(used, top, 0.0), torch.where(first, soft, 0.0), hard], 1)]
        dl, m = t["dloss"][:, None], t["sums"][:, :1]
        scale = dl * (weight * temp)
        grad = torch.where(first, scale * torch.exp((z - m) / temp - t["sums"][:, 1:2]), 0.0)
        grad.scatter_add_(1, index, -scale * p)
        if second is not None:
            scale = dl * (1.0 - weight)
            grad += torch.where(second, scale * torch.exp(z - m - t["sums"][:, 2:]), 0.0)
            grad.scatter_add_(1, torch.where(second, t["labels"].long()[:, None], 0), torch.where(second, -scale, 0.0))
        return [grad.to(_DT[c["dtype"]])]
    z = t["logits"].float()
    if c["history"]:
        k = t["history"].long()
        there = torch.arange(c["history"], device="cuda") < t["lengths"].long()[:, None]
        at = torch.where(there & (k >= 0) & (k < v), k, v)
        n = torch.zeros(c["rows"], v + 1, device="cuda").scatter_add_(1, at, torch.ones_like(at, dtype=torch.float32))[:, :v]
        r = t["repetition"][:, None]
        seen = torch.where(z > 0.0, z / r, z * r) - (t["frequency"][:, None] * n + t["presence"][:, None])
        z = torch.where(n > 0.0, seen, z)
    if c["bias"] == "dense":
        z = z + t["bias"]
    elif c["bias"] == "sparse":
        z = z.scatter_add(1, t["bias_index"].long(), t["bias"])
    if c["allowed"] != "none":
        ok = t["allowed"]
        if c["allowed"] == "bits":
            ok = ((ok[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).flatten(1)[:, :v].bool()
        z = torch.where(ok, z, -math.inf)
    return [z.to(_DT[c["to"]])]


# ---- what the path cannot do without -----------------------------------------------------------------
def _distinct(n, vocab):
    """How many of a vocabulary's tokens n draws find, on average."""
    edge = torch.log(torch.arange(1, vocab + 2, dtype=torch.float64)) / math.log(vocab + 1)
    return float((1.0 - (1.0 - (edge[1:] - edge[:-1])) ** (n * (1.0 - _PAD))).sum())


def work(case):
    """Each input read once, each output written once; a few operations for each element."""
    c, op, v = case, case["op"], case["vocab"]
    es, ids = _SIZE[c["dtype"]], _SIZE[c["ids"]]
    if op == "embed":
        n, w = c["tokens"], c["width"]
        return {"bytes": int(_distinct(n, v) * w * es) + n * ids + n * w * _SIZE[c["to"]], "flops": n * w}
    if op == "embed_grad":
        n, w = c["tokens"], c["width"]
        return {"bytes": int(n * (1.0 - _PAD)) * w * es + n * ids + v * w * _SIZE[c["to"]], "flops": n * w}
    if op in ("distill", "distill_grad"):
        r, k, both = c["rows"], c["entries"], c["weight"] < 1.0
        b = r * v * es + r * k * (ids + _SIZE[c["teacher"]]) + (r * ids if both else 0)
        if op == "distill":
            return {"bytes": b + 16 * r, "flops": r * v * (8 if both else 5)}
        return {"bytes": b + r * v * es + r * (16 if both else 12), "flops": r * v * (10 if both else 5)}
    r = c["rows"]
    b = r * v * (es + _SIZE[c["to"]]) + int(0.75 * r * c["history"]) * ids + (r * (12 + ids) if c["history"] else 0)
    b += {"none": 0, "dense": 4 * v, "sparse": r * c["entries"] * (4 + ids)}[c["bias"]]
    b += {"none": 0, "bits": r * ((v + 31) // 32) * 4, "bool": r * v}[c["allowed"]]
    return {"bytes": b, "flops": r * v * 3}


# ---- the definitions in 64 bits --------------------------------------------------------------------------
def _exact_distill(c, t):
    temp, weight, v = c["temperature"], c["weight"], c["vocab"]
    grad = c["op"] == "distill_grad"
    step = max(1, (1 << 27) // v)
    parts = []
    for i in range(0, c["rows"], step):
        z = t["logits"][i:i + step].double()
        index, value = t["index"][i:i + step].long(), t["teacher"][i:i + step].double()
        n = z.shape[0]
        rows = torch.arange(n, device="cuda")
        outside = (index < 0) | (index >= v)
        p = torch.softmax((value / temp).masked_fill(outside, -math.inf), 1)
        p = torch.nan_to_num(p, nan=0.0)  # a row without entries
        some = ~outside.all(1)
        index = index.masked_fill(outside, 0)
        labelled = torch.zeros(n, dtype=torch.bool, device="cuda")
        if "labels" in t:
            label = t["labels"][i:i + step].long()
            labelled = (label >= 0) & (label < v)
            label = label.masked_fill(~labelled, 0)
        if not grad:
            m = z.amax(1)
            lse, one = torch.logsumexp((z - m[:, None]) / temp, 1), torch.logsumexp(z - m[:, None], 1)
            got = (z[rows[:, None], index] - m[:, None]) / temp - lse[:, None]
            loss = weight * temp ** 2 * (torch.xlogy(p, p) - p * got).sum(1)
            if "labels" in t:
                loss = loss + (1.0 - weight) * (one + m - z[rows, label]).masked_fill(~labelled, 0.0)
            parts.append((loss, torch.stack([m.masked_fill(~(some | labelled), 0.0), lse.masked_fill(~some, 0.0),
                                             one.masked_fill(~labelled, 0.0)], 1)))
            continue
        sums = t["sums"][i:i + step].double()
        d = torch.exp((z - sums[:, :1]) / temp - sums[:, 1:2])
        d[~some] = 0.0
        for k in range(index.shape[1]):
            d[rows, index[:, k]] -= p[:, k]
        d *= weight * temp
        if "labels" in t:
            s = torch.exp(z - sums[:, :1] - sums[:, 2:])
            s[rows, label] -= 1.0
            s[~labelled] = 0.0
            d += (1.0 - weight) * s
        parts.append((d * t["dloss"][i:i + step].double()[:, None],))
    return [torch.cat(x) for x in zip(*parts)]


def _exact_adjust(c, t):
    v = c["vocab"]
    z = t["logits"].double()
    for r in range(c["rows"]):
        row = z[r]
        if c["history"]:
            past = t["history"][r, :int(t["lengths"][r])].long()
            past = past[(past >= 0) & (past < v)]
            tok, n = torch.unique(past, return_counts=True)
            old = row[tok]
            rep = t["repetition"][r].double()
            row[tok] = old * torch.where(old > 0, 1.0 / rep, rep) - n * t["frequency"][r].double() - t["presence"][r].double()
        if c["bias"] == "sparse":
            for k, b in zip(t["bias_index"][r].tolist(), t["bias"][r].tolist()):
                row[k] += b
        elif c["bias"] == "dense":
            row += t["bias"].double()
        if c["allowed"] == "bits":
            column = torch.arange(v, device="cuda")
            row[((t["allowed"][r].long()[column // 32] >> (column % 32)) & 1) == 0] = -math.inf
        elif c["allowed"] == "bool":
            row[~t["allowed"][r]] = -math.inf
    return [z]


def exact(case, seed):
    c = dict(case)
    t = _tensors(c, seed)
    v = c["vocab"]
    if c["op"] == "embed":
        table = torch.cat([t["table"], torch.zeros(1, c["width"], dtype=t["table"].dtype, device="cuda")])
        k = t["tokens"].long()
        k[(k < 0) | (k >= v)] = v
        return [table.index_select(0, k).double() * _SCALE]
    if c["op"] == "embed_grad":
        k, order = torch.sort(t["tokens"].long())
        dy = t["dy"].double()[order]
        out = torch.zeros(v, c["width"], dtype=torch.float64, device="cuda")
        inside = (k >= 0) & (k < v)
        out.index_put_((k[inside],), dy[inside], accumulate=True)
        return [out * _SCALE]
    return _exact_distill(c, t) if c["op"] in ("distill", "distill_grad") else _exact_adjust(c, t)
