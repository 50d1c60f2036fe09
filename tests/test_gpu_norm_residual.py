"""norm_residual and norm_residual_grad on the GPU against their 64-bit forms.

Bounds: a row's sums of squares err by (width + 8) 2^-24 at most and by about sqrt(width) 2^-24 in a tree, relative, which a
norm's result takes over by half; a gate's activation by (10 + 2 |g|) 2^-24.  Each result is held to
(64 + 2 sqrt(width)) 2^-24 of the size of its own terms (a row's largest, where they are subtracted), and half an ulp of its type;
column sums to the same of the sum of their terms' sizes."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import blocks_reference as R

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]


def make(rng, shape, dt, st, o, gate=True, weights=True, wdt="f32"):
    w = shape[-1:]
    v = {"x": R.rounded(rng.standard_normal(shape) + 0.2, dt), "residual": R.rounded(rng.standard_normal(shape) * 2, st),
         "dr": R.rounded(rng.standard_normal(shape), st), "dy": R.rounded(rng.standard_normal(shape), dt) if o["pre"] else None,
         "gate": R.rounded(rng.standard_normal(shape), dt) if gate else None}
    for k, on in (("w1", o["post"]), ("w2", o["pre"]), ("scale", True)):
        v[k] = R.rounded(1 + 0.3 * rng.standard_normal(w), wdt) if on and weights else None
    return v


def device(v, dt, st, wdt="f32"):
    kinds = {"x": dt, "residual": st, "dr": st, "dy": dt, "gate": dt, "w1": wdt, "w2": wdt, "scale": wdt}
    return {k: None if a is None else R.to_device(a, kinds[k]) for k, a in v.items()}


def keep_of(shape, p, seed, offset):
    if p == 0:
        return np.ones(shape)
    return R.kept(int(np.prod(shape[:-1])), shape[-1], p, seed, offset).reshape(shape) * R.keep_scale(p)


def near(got, want, size, dt, what, width):
    tol = (64 + 2 * np.sqrt(width)) * R.EPS
    ulp, tiny = R.ROUND[dt]
    bound = tol * size + 1.01 * ulp * np.abs(want) + tiny
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3], want[bad][:3], np.broadcast_to(bound, bad.shape)[bad][:3])


def amax(v):
    return np.abs(v).max(-1, keepdims=True) if v.shape[-1] else np.abs(v)


def run(rng, shape, dt, st, o, p=0.0, gate=True, weights=True, wdt="f32", seed=77, offset=5, views=None):
    v = make(rng, shape, dt, st, o, gate, weights, wdt)
    d = device(v, dt, st, wdt)
    if views:
        v, d = views(v, d)
        shape = v["x"].shape
    one = lambda k: 1.0 if v[k] is None else v[k]  # noqa: E731
    keep = keep_of(shape, p, seed, offset)
    kw = dict(o, p=p, seed=seed, offset=offset, gate=d["gate"], post_weight=d["w1"], scale=d["scale"], pre_weight=d["w2"])
    r, y = ms.norm_residual(d["x"], d["residual"], **kw)
    wr, wy = R.block(v["x"], v["residual"], v["gate"], one("w1"), one("scale"), one("w2"), keep, o)
    width = shape[-1]
    assert r.dtype == st
    branch = np.abs(wr - v["residual"])
    lift = 1.0
    if o["post"] == "layer":  # x less its mean: the error is that of x, not of the difference
        inv = R.norm(v["x"], "layer", o["eps"])[1]
        lift = amax(v["x"]) * inv * np.abs(one("scale") * one("w1")) * (np.abs(R.act(v["gate"], o["gate_kind"])[0]) if gate else 1) * keep
    rsize = np.abs(v["residual"]) + branch + lift
    near(R.values(r), wr, rsize, st, "r", width)
    if o["pre"]:
        assert y.dtype == dt
        inv2 = R.norm(wr, o["pre"], o["eps"])[1]
        size = np.abs(wy) + np.abs(one("w2")) * inv2 * (rsize + (amax(wr) if o["pre"] == "layer" else 0))
        near(R.values(y), wy, size, dt, "y", width)
    else:
        assert y is None

    stored = R.rounded(wr, st)
    got = ms.norm_residual_grad(d["dr"], d["dy"], d["x"], R.to_device(stored, st), **kw)
    names = ("dx", "dresidual", "dgate", "dpost_weight", "dscale", "dpre_weight")
    dy = np.zeros(shape) if v["dy"] is None else v["dy"]
    want = R.block_grad(v["dr"], dy, v["x"], stored, v["gate"], one("w1"), one("scale"), one("w2"), keep, o)
    have = {"dgate": gate, "dpost_weight": v["w1"] is not None, "dscale": v["scale"] is not None,
            "dpre_weight": v["w2"] is not None}
    # sizes: the same forms with every term's absolute value
    n1, inv1 = R.norm(v["x"], o["post"], o["eps"])
    a, slope = (np.abs(t) for t in R.act(v["gate"], o["gate_kind"])) if gate else (1.0, 0.0)
    an1 = np.abs(n1) + (amax(v["x"]) * inv1 if o["post"] == "layer" else 0)
    D = np.abs(v["dr"])
    if o["pre"]:
        n2, inv2 = R.norm(stored, o["pre"], o["eps"])
        an2 = np.abs(n2) + (amax(stored) * inv2 if o["pre"] == "layer" else 0)
        q = np.abs(dy * one("w2"))
        D = D + inv2 * (q + an2 * (q * an2).mean(-1, keepdims=True) + q.mean(-1, keepdims=True))
    aw1, asc = np.abs(one("w1")), np.abs(one("scale"))
    dv = D * asc * keep
    du = dv * a
    q = du * aw1
    dx = q if not o["post"] else inv1 * (q + an1 * (q * an1).mean(-1, keepdims=True) + q.mean(-1, keepdims=True))
    gsize = dv * an1 * aw1 * ((slope + np.abs(v["gate"])) if gate else 0)
    size = {"dx": dx, "dresidual": D, "dgate": gsize, "dpost_weight": du * an1, "dscale": D * an1 * aw1 * a * keep,
            "dpre_weight": np.abs(dy) * an2 if o["pre"] else None}
    kinds = {"dx": dt, "dresidual": st, "dgate": dt}
    rows = int(np.prod(shape[:-1]))
    for name, g in zip(names, got):
        if not have.get(name, True):
            assert g is None, name
            continue
        s = size[name]
        if name not in kinds:
            s = s.sum(tuple(range(len(shape) - 1)))
        near(R.values(g), want[name], s, kinds.get(name, wdt), name, max(width, rows))
    return v, d, got


OPTIONS = [dict(post=a, pre=b, gate_kind=g, eps=1e-5) for a, b, g in
           [("rms", "rms", "silu"), ("layer", "layer", "sigmoid"), ("rms", "layer", "sigmoid"), ("layer", "rms", "silu"),
            (None, "rms", "silu"), ("rms", None, "silu"), (None, None, "silu"), (None, "layer", "silu")]]
WIDTHS = [1, 2, 7, 8, 9, 63, 64, 65, 256, 511, 512, 513, 1000, 1024, 1111, 2048, 2056, 4096, 5000, 8192, 9001]


@pytest.mark.parametrize("width", WIDTHS)
def test_widths(width):
    rng = np.random.default_rng(width)
    run(rng, (5, width), "f32", "f32", OPTIONS[0], p=0.2 if width < 600 else 0.0)
    run(rng, (3, width), "bf16", "f32", OPTIONS[1])


@pytest.mark.parametrize("width", [12000, 16384, 20000, 33000, 70001])
def test_wide_rows(width):
    rng = np.random.default_rng(width)
    run(rng, (2, width), "f32", "f32", OPTIONS[0])
    run(rng, (2, width), "bf16", "bf16", OPTIONS[3])


@pytest.mark.parametrize("o", OPTIONS, ids=lambda o: f"{o['post']}-{o['pre']}")
@pytest.mark.parametrize("dt,st", TYPES)
def test_options_and_types(o, dt, st):
    rng = np.random.default_rng(1)
    run(rng, (4, 3, 96), dt, st, o, p=0.1)
    run(rng, (4, 3, 96), dt, st, o, gate=False)
    run(rng, (4, 3, 96), dt, st, o, weights=False, p=0.1)
    run(rng, (4, 3, 99), dt, st, o, wdt=dt)


@pytest.mark.parametrize("rows", [1, 2, 3, 255, 256, 257, 512, 513, 2000, 5000])
def test_rows(rows):
    rng = np.random.default_rng(rows)
    run(rng, (rows, 72), "f32", "f32", OPTIONS[0])
    run(rng, (rows, 33), "bf16", "bf16", OPTIONS[1])


def test_slices_of_wider_rows():
    """x and the gate as halves of one product's rows, the others with offsets and odd pitches; leading axes that are no
    single row stride, and strided columns, are copied."""
    rng = np.random.default_rng(3)

    def halves(v, d):
        w = v["x"].shape[-1] // 2
        cut = lambda a, lo: a[..., lo:lo + w]  # noqa: E731
        at = {"x": 0, "gate": w, "residual": 1, "dr": 3, "dy": 2}
        hv = {k: (cut(a, at[k]) if k in at else a[:w]) if a is not None else None for k, a in v.items()}
        hd = {k: (a[:, :, at[k]:at[k] + w] if k in at else a[:w]) if a is not None else None for k, a in d.items()}
        return hv, hd

    def turned(v, d):
        hv = {k: None if a is None else a.transpose(1, 0, 2) if a.ndim == 3 else a for k, a in v.items()}
        hd = {k: None if a is None else ms.permute(a, (1, 0, 2)) if a.ndim == 3 else a for k, a in d.items()}
        return hv, hd

    def stepped(v, d):
        hv = {k: None if a is None else a[..., ::2] for k, a in v.items()}
        hd = {k: None if a is None else a[:, :, ::2] if a.ndim == 3 else a[::2] for k, a in d.items()}
        return hv, hd

    for views in (halves, turned, stepped):
        for dt in ("f32", "bf16"):
            run(rng, (3, 5, 200), dt, "f32", OPTIONS[0], p=0.1, views=views)


def test_numbers_and_absent_parts():
    """A scale that is a number, no residual, and gradients of one output alone."""
    rng = np.random.default_rng(4)
    o = OPTIONS[0]
    x, gate = (R.rounded(rng.standard_normal((6, 80)), "f32") for _ in range(2))
    w = np.ones(80)
    r, y = ms.norm_residual(ms.array(x, dtype="f32"), gate=ms.array(gate, dtype="f32"), scale=0.5, **o)
    wr, wy = R.block(x, 0.0, gate, w, 0.5, w, 1.0, o)
    assert np.allclose(R.values(r), wr, rtol=1e-5, atol=1e-6) and np.allclose(R.values(y), wy, rtol=1e-5, atol=1e-6)
    # the block's first norm alone: r is x
    r, y = ms.norm_residual(ms.array(x, dtype="f32"), post=None)
    assert np.array_equal(R.values(r), x) and np.allclose(R.values(y), R.norm(x, "rms", 1e-6)[0], rtol=1e-5, atol=1e-6)
    dr, dy = (rng.standard_normal((6, 80)) for _ in range(2))
    A = lambda v: ms.array(v, dtype="f32")  # noqa: E731
    for use_r, use_y in ((True, False), (False, True)):
        got = ms.norm_residual_grad(A(dr) if use_r else None, A(dy) if use_y else None, A(x), A(wr), gate=A(gate), scale=0.5, **o)
        want = R.block_grad(dr * use_r, dy * use_y, x, wr, gate, w, 0.5, w, 1.0, o)
        for k, g in zip(("dx", "dresidual", "dgate"), got):
            assert np.allclose(R.values(g), want[k], rtol=1e-4, atol=1e-5), (use_r, k)
        assert got[3:] == (None, None, None)


def test_masked_rows_and_values():
    """A row of zeros has a finite norm and gradient; a dropped infinity or NaN reaches no one through the dropout; rows do
    not reach each other."""
    rng = np.random.default_rng(5)
    o = dict(OPTIONS[0])
    x = rng.standard_normal((4, 64))
    x[1] = 0
    A = lambda v: ms.array(v, dtype="f32")  # noqa: E731
    res = rng.standard_normal((4, 64))
    res[1] = 0
    r, y = ms.norm_residual(A(x), A(res), **o)
    assert np.isfinite(R.values(r)).all() and (R.values(y)[1] == 0).all()
    got = ms.norm_residual_grad(A(x), A(x), A(x), r, **o)
    assert all(np.isfinite(R.values(g)).all() for g in got if g is not None)
    # no post norm: each value of x stands for itself, and drops with its own number
    keep = R.kept(4, 64, 0.5, 3, 0)
    bad = np.where(keep, x, np.nan)
    o["post"] = None
    r, y = ms.norm_residual(A(bad), A(res), p=0.5, seed=3, **o)
    assert np.isfinite(R.values(r)).all() and np.isfinite(R.values(y)).all()
    got = ms.norm_residual_grad(A(x), A(x), A(bad), r, p=0.5, seed=3, scale=A(np.ones(64)), **o)
    assert all(np.isfinite(R.values(g)).all() for g in got if g is not None)
    x[2, 5] = np.nan
    r, y = ms.norm_residual(A(x), A(res), **OPTIONS[0])
    assert np.isfinite(R.values(y)[[0, 1, 3]]).all() and np.isnan(R.values(y)[2]).all()


def test_dropout_is_the_dropout_operators():
    """The mask inside is the one that ms.dropout draws for the same seed, offset and place."""
    for width in (64, 100, 1111):
        x = np.ones((7, width))
        r, _ = ms.norm_residual(ms.array(x, dtype="f32"), post=None, pre=None, p=0.3, seed=2 ** 35 + 1, offset=2 ** 34)
        assert np.array_equal(r.numpy(), ms.dropout(ms.ones((7, width)), 0.3, seed=2 ** 35 + 1, offset=2 ** 34).numpy())


def test_gradient_against_differences():
    rng = np.random.default_rng(6)
    for o in OPTIONS[:4]:
        shape = (6, 40)
        v = make(rng, shape, "f32", "f32", o)
        keep = keep_of(shape, 0.25, 4, 1)
        wr, wy = R.block(v["x"], v["residual"], v["gate"], v["w1"], v["scale"], v["w2"], keep, o)
        A = lambda a: ms.array(a, dtype="f32")  # noqa: E731
        got = ms.norm_residual_grad(A(v["dr"]), A(v["dy"]), A(v["x"]), A(wr), gate=A(v["gate"]), post_weight=A(v["w1"]),
                                    scale=A(v["scale"]), pre_weight=A(v["w2"]), p=0.25, seed=4, offset=1, **o)

        def loss(x, residual, gate, w1, scale, w2):
            r, y = R.block(x, residual, gate, w1, scale, w2, keep, o)
            return (v["dr"] * r).sum() + (v["dy"] * y).sum()

        args = [v[k] for k in ("x", "residual", "gate", "w1", "scale", "w2")]
        step = 1e-5
        for i, g in enumerate(got):
            u = rng.standard_normal(args[i].shape)
            ends = [loss(*(a + s * u if j == i else a for j, a in enumerate(args))) for s in (step, -step)]
            slope = (ends[0] - ends[1]) / (2 * step)
            grad = R.values(g)
            # f32 entries: 2e-5 of their size; the difference itself: step^2 and 64-bit noise; r was rounded to f32
            assert abs((grad * u).sum() - slope) <= 2e-5 * np.abs(grad * u).sum() + 2e-4


def test_empty_calls():
    for shape in ((0, 16), (4, 0), (0, 0)):
        x = ms.array(np.zeros(shape), dtype="f32")
        w = ms.array(np.ones(shape[1]), dtype="f32")
        r, y = ms.norm_residual(x, x, post_weight=w, scale=w, pre_weight=w)
        assert r.shape == shape and y.shape == shape
        got = ms.norm_residual_grad(x, x, x, r, post_weight=w, scale=w, pre_weight=w)
        assert got[0].shape == shape and all((g.numpy() == 0).all() for g in got[3:])


def test_the_same_bits_again():
    rng = np.random.default_rng(8)
    o = OPTIONS[0]
    v, d, first = run(rng, (3000, 256), "bf16", "bf16", o, p=0.0)
    wr = R.rounded(R.block(v["x"], v["residual"], v["gate"], v["w1"], v["scale"], v["w2"], 1.0, o)[0], "bf16")
    r = R.to_device(wr, "bf16")
    kw = dict(o, gate=d["gate"], post_weight=d["w1"], scale=d["scale"], pre_weight=d["w2"])
    for _ in range(3):
        again = ms.norm_residual_grad(d["dr"], d["dy"], d["x"], r, **kw)
        for a, b in zip(first, again):
            assert np.array_equal(a.numpy(), b.numpy())


def test_given_outputs_and_streams():
    rng = np.random.default_rng(9)
    x = ms.array(rng.standard_normal((300, 512)), dtype="f32")
    zero = ms.array(np.zeros(1), dtype="f32")
    w = ms.ones((512,))
    r0, y0 = ms.norm_residual(x, x, pre_weight=w)
    outs = (ms.array(np.zeros((300, 512)), dtype="f32"), ms.array(np.zeros((300, 512)), dtype="f32"))
    r, y = ms.norm_residual(x, x, pre_weight=w, out=outs)
    assert r.data_ptr == outs[0].data_ptr and y.data_ptr == outs[1].data_ptr
    assert np.array_equal(r.numpy(), r0.numpy()) and np.array_equal(y.numpy(), y0.numpy())
    want = [g.numpy() for g in ms.norm_residual_grad(x, x, x, r0, pre_weight=w) if g is not None]
    a, b = ms.Stream(), ms.Stream()
    for _ in range(3):
        with ms.stream(a):
            x2 = ms.add(x, zero)
        with ms.stream(b):
            got = ms.norm_residual_grad(x2, x2, x2, r0, pre_weight=w)
            del x2
        for g, h in zip([g for g in got if g is not None], want):
            assert np.array_equal(g.numpy(), h)


def test_refusals():
    f = lambda *s: ms.array(np.zeros(s), dtype="f32")  # noqa: E731
    x, w = f(3, 8), f(8)
    half = ms.astype(x, "bf16")
    hw = ms.astype(w, "bf16")
    for call, error in [
        (lambda: ms.norm_residual(ms.array(np.zeros((3, 8)), dtype="f64")), ms.DtypeError),
        (lambda: ms.norm_residual(ms.array(np.zeros(()), dtype="f32")), ms.ShapeError),
        (lambda: ms.norm_residual(x, half), ms.DtypeError),
        (lambda: ms.norm_residual(x, f(3, 9)), ms.ShapeError),
        (lambda: ms.norm_residual(x, gate=f(3, 1)), ms.ShapeError),
        (lambda: ms.norm_residual(half, gate=x), ms.DtypeError),
        (lambda: ms.norm_residual(x, post_weight=f(7)), ms.ShapeError),
        (lambda: ms.norm_residual(x, post_weight=hw), ms.DtypeError),
        (lambda: ms.norm_residual(half, post_weight=hw, scale=w), ms.DtypeError),
        (lambda: ms.norm_residual(x, post=None, post_weight=w), ms.ShapeError),
        (lambda: ms.norm_residual(x, pre=None, pre_weight=w), ms.ShapeError),
        (lambda: ms.norm_residual(x, post="other"), ValueError),
        (lambda: ms.norm_residual(x, gate_kind="other"), ValueError),
        (lambda: ms.norm_residual(x, eps=-1.0), ValueError),
        (lambda: ms.norm_residual(x, p=2.0), ValueError),
        (lambda: ms.norm_residual(x, x, out=(x, None)), ms.MemoryError),
        (lambda: ms.norm_residual(x, pre=None, out=(None, f(3, 8))), ms.ShapeError),
        (lambda: ms.norm_residual(x, out=f(2, 3, 8)[0]), (TypeError, RuntimeError)),
        (lambda: ms.norm_residual_grad(None, None, x, x), ms.ShapeError),
        (lambda: ms.norm_residual_grad(x, x, x, None), ms.ShapeError),
        (lambda: ms.norm_residual_grad(x, x, x, x, pre=None), ms.ShapeError),
        (lambda: ms.norm_residual_grad(half, x, x, x), ms.DtypeError),
        (lambda: ms.norm_residual_grad(x, x, x, f(3, 9)), ms.ShapeError),
        (lambda: ms.norm_residual_grad(x, x, x, x, out=(None, None, f(3, 8), None, None, None)), ms.ShapeError),
        (lambda: ms.norm_residual_grad(x, x, x, x, out=(None, None)), TypeError),
    ]:
        with pytest.raises(error):
            call()
