"""gated_scan and gated_scan_grad on the GPU against step-by-step 64-bit forms.

Bounds: an f32 product or sum errs by 2^-24, relative; a decay enters a product of factors once, with a rounding for
the product and one for the sum it goes into, wherever the factors are grouped (3 x 2^-24 a factor and a few for the
groups); a sigmoid adds the errors of its exponential (2^-23 of its own, and 2 |g| 2^-24 from the rounded exponent), of 1 + e
and of the reciprocal (2^-23).  tests/blocks_reference.py carries these along the recurrence; the stored result adds half an ulp
of its type."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import blocks_reference as R

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]


def case(rng, shape, axis, kind, dt, gdt, gshape=None, h0=False, reset=None):
    x = R.rounded(rng.standard_normal(shape), dt)
    g = rng.standard_normal(shape if gshape is None else gshape) * 1.5 + 2.0
    g = R.rounded(R.sigmoid(g) if kind == "decay" else g, gdt)
    lanes = tuple(n for i, n in enumerate(shape) if i != axis % len(shape))
    first = R.rounded(rng.standard_normal(lanes), "f32") if h0 else None
    cut = None if reset is None else rng.random(reset) < 0.1
    return x, g, first, cut


def factor_error(g, kind):
    extra = 8 + 2 * np.abs(g).max(initial=0) if kind == "blend" else 0
    return (6 + extra) * R.EPS


def forward_bounds(x, g, h0, cut, axis, kind, want, dt):
    a, b = R.factors(x, g, kind)
    a, b = (np.moveaxis(np.broadcast_to(v, x.shape), axis, 0) for v in (a, b))
    if cut is not None:
        a = np.where(np.moveaxis(np.broadcast_to(cut, x.shape), axis, 0), 0.0, a)
    first = np.zeros(b.shape[1:]) if h0 is None else h0
    f = factor_error(g, kind)
    E, mag = R.scan_error(a, b, first, f, f)
    E = E + 16 * R.EPS * mag
    E = np.moveaxis(E, 0, axis)
    ulp, tiny = R.ROUND[dt]
    return E + ulp * np.abs(want) * 1.01 + ulp * E + tiny, E


def check(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3], want[bad][:3], np.broadcast_to(bound, bad.shape)[bad][:3])


def last_of(v, axis):
    return np.take(v, v.shape[axis] - 1, axis)


def run_forward(rng, shape, axis, kind, dt, gdt, gshape=None, h0=False, reset=None):
    x, g, first, cut = case(rng, shape, axis, kind, dt, gdt, gshape, h0, reset)
    want, state = R.scan(x, g, first, cut, axis, kind)
    h, s = ms.gated_scan(R.to_device(x, dt), R.to_device(g, gdt), None if first is None else ms.array(first, dtype="f32"),
                         reset=None if cut is None else R.to_device(cut, "bool"), axis=axis, kind=kind)
    assert h.dtype == dt and s.dtype == "f32"
    bound, E = forward_bounds(x, g, first, cut, axis, kind, want, dt)
    check(R.values(h), want, bound, "h")
    e = last_of(E, axis)
    check(R.values(s), state, e + 4 * R.EPS * np.abs(state), "state")


def run_grad(rng, shape, axis, kind, dt, gdt, gshape=None, h0=False, reset=None, dstate=False):
    x, g, first, cut = case(rng, shape, axis, kind, dt, gdt, gshape, h0, reset)
    h = R.rounded(R.scan(x, g, first, cut, axis, kind)[0], dt)
    dh = R.rounded(rng.standard_normal(shape), dt)
    lanes = tuple(n for i, n in enumerate(shape) if i != axis % len(shape))
    ds = R.rounded(rng.standard_normal(lanes), "f32") if dstate else None
    want = R.scan_grad(dh, x, g, h, first, cut, ds, axis, kind)
    f32 = lambda v: None if v is None else ms.array(v, dtype="f32")  # noqa: E731
    dev = lambda v, d: R.to_device(v, d)  # noqa: E731
    got = ms.gated_scan_grad(dev(dh, dt), dev(x, dt), dev(g, gdt), dev(h, dt), f32(first),
                             reset=None if cut is None else dev(cut, "bool"), dstate=f32(ds), axis=axis, kind=kind)
    # the flow back is the recurrence over reversed time, with factors shifted by one step
    a, _ = R.factors(x, g, kind)
    a = np.moveaxis(np.broadcast_to(a, shape), axis, 0)[::-1]
    c = np.zeros(shape, bool) if cut is None else np.broadcast_to(cut, shape)
    a = np.where(np.moveaxis(c, axis, 0)[::-1], 0.0, a)
    late = np.moveaxis(dh, axis, 0)[::-1].copy()
    if ds is not None:
        late[0] = np.abs(late[0]) + np.abs(ds)
    shifted = np.concatenate([np.zeros((1,) + a.shape[1:]), a[:-1]])
    f = factor_error(g, kind)
    E, mag = R.scan_error(shifted, late, np.zeros(a.shape[1:]), f, f)
    E = E + 16 * R.EPS * mag
    first0 = a[-1] * (E[-1] + f * mag[-1]) + 4 * R.EPS * mag[-1]
    E, mag = (np.moveaxis(v[::-1], 0, axis) for v in (E, mag))
    before = np.moveaxis(np.concatenate([(np.zeros(a.shape[1:]) if first is None else first)[None],
                                         np.moveaxis(h, axis, 0)[:-1]]), 0, axis)
    if kind == "decay":
        ex, eg, mg = E, E * np.abs(before), mag * np.abs(before)
    else:
        rest, slope = R.sigmoid(-g), R.sigmoid(g) * R.sigmoid(-g)
        ex = rest * (E + f * mag)
        span = np.abs(before) + np.abs(x)
        eg, mg = slope * span * (E + 3 * f * mag), slope * span * mag
    ulp, tiny = R.ROUND[dt]
    check(R.values(got[0]), want[0], ex * 1.01 + ulp * 1.01 * np.abs(want[0]) + tiny, "dx")
    gulp, gtiny = R.ROUND[gdt]
    n = mg.size // max(1, want[1].size)  # elements of one sum: their order is the kernel's
    eg = R.unspread(eg + (4 + n) * R.EPS * mg, want[1].shape)
    check(R.values(got[1]), want[1], eg * 1.01 + gulp * 1.01 * np.abs(want[1]) + gtiny, "dgate")
    if first is None:
        assert got[2] is None
    else:
        check(R.values(got[2]), want[2], first0 * 1.01 + 4 * R.EPS * np.abs(want[2]), "dh0")
    return got


STEPS = [1, 2, 7, 8, 9, 33, 64, 65, 127, 128, 129, 255, 256, 257, 1000]


@pytest.mark.parametrize("kind", ["decay", "blend"])
@pytest.mark.parametrize("steps", STEPS)
def test_lengths_channels_innermost(kind, steps):
    rng = np.random.default_rng(steps)
    run_forward(rng, (2, steps, 72), 1, kind, "f32", "f32", h0=True)
    run_grad(rng, (2, steps, 72), 1, kind, "bf16", "bf16", h0=True, dstate=True)


@pytest.mark.parametrize("kind", ["decay", "blend"])
@pytest.mark.parametrize("steps", STEPS + [511, 513, 4100])
def test_lengths_time_innermost(kind, steps):
    rng = np.random.default_rng(steps)
    run_forward(rng, (2, 5, steps), 2, kind, "f32", "f32", h0=True)
    run_grad(rng, (2, 5, steps), -1, kind, "bf16", "bf16", h0=True, dstate=True)


@pytest.mark.parametrize("dt,gdt", TYPES)
@pytest.mark.parametrize("width", [1, 3, 8, 37, 64, 65, 130])
def test_widths_and_types(dt, gdt, width):
    rng = np.random.default_rng(width)
    for kind in ("decay", "blend"):
        run_forward(rng, (3, 70, width), 1, kind, dt, gdt, reset=(3, 70, 1))
        run_grad(rng, (3, 70, width), 1, kind, dt, gdt, reset=(3, 70, 1))
        run_forward(rng, (3, width, 70), 2, kind, dt, gdt, reset=(3, 1, 70))
        run_grad(rng, (3, width, 70), 2, kind, dt, gdt, reset=(3, 1, 70))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("width", [1, 5, 16, 32, 64, 96, 128, 200])
def test_gates_shared_by_a_heads_channels(dt, width):
    rng = np.random.default_rng(width)
    for kind in ("decay", "blend"):
        run_forward(rng, (2, 300, 3, width), 1, kind, dt, "f32", gshape=(2, 300, 3, 1), h0=True)
        run_grad(rng, (2, 300, 3, width), 1, kind, dt, "f32", gshape=(2, 300, 3, 1), h0=True, reset=(2, 300, 1, 1),
                 dstate=True)
    run_grad(rng, (2, 40, 3, width), 1, "decay", dt, dt, gshape=(2, 40, 3, 1))


@pytest.mark.parametrize("gshape", [(1, 1, 24), (24,), (1, 90, 1), (90, 1), (1, 1, 1), (2, 1, 1), (2, 1, 24), (2, 90, 1)])
def test_gates_broadcast_along_any_axes(gshape):
    rng = np.random.default_rng(5)
    for kind in ("decay", "blend"):
        for dt, gdt in (("f32", "f32"), ("bf16", "bf16")):
            run_forward(rng, (2, 90, 24), 1, kind, dt, gdt, gshape=gshape)
            run_grad(rng, (2, 90, 24), 1, kind, dt, gdt, gshape=gshape)


@pytest.mark.parametrize("reset", [(2, 90, 1), (1, 90, 1), (90, 1), (1, 1, 24), (2, 90, 24), (2, 1, 1)])
def test_resets_broadcast_along_any_axes(reset):
    rng = np.random.default_rng(6)
    for kind in ("decay", "blend"):
        run_forward(rng, (2, 90, 24), 1, kind, "f32", "f32", h0=True, reset=reset)
        run_grad(rng, (2, 90, 24), 1, kind, "f32", "f32", h0=True, reset=reset)
        run_grad(rng, (2, 90, 24), 1, kind, "f32", "f32", gshape=(2, 90, 1), h0=True, reset=reset)


@pytest.mark.parametrize("shape,axis", [((700,), 0), ((90, 24), 0), ((90, 24), 1), ((3, 4, 33, 2, 5), 2), ((33, 2, 5), 0),
                                        ((3, 33, 1), 1), ((1, 33, 1), 1), ((2, 3000, 48), 1), ((1, 5000, 3), 1),
                                        ((3, 9000), 1)])
def test_axes(shape, axis):
    rng = np.random.default_rng(7)
    for kind in ("decay", "blend"):
        run_forward(rng, shape, axis, kind, "f32", "f32", h0=True)
        run_grad(rng, shape, axis, kind, "f32", "f32", h0=True, dstate=True)


@pytest.mark.parametrize("shape,axis", [((2, 9001, 72), 1), ((3, 20000), 1), ((1, 30011, 8), 1), ((4, 2, 17000), 2)])
def test_long_sequences(shape, axis):
    rng = np.random.default_rng(8)
    reset = tuple(n if i in (0, axis) else 1 for i, n in enumerate(shape))
    run_forward(rng, shape, axis, "decay", "bf16", "f32", h0=True, reset=reset)
    run_grad(rng, shape, axis, "blend", "f32", "f32", h0=True, reset=reset, dstate=True)


def test_a_long_scan_gives_the_same_bits_again():
    rng = np.random.default_rng(9)
    x, g, _, _ = case(rng, (1, 30000, 128), 1, "decay", "f32", "f32")
    X, G = R.to_device(x, "f32"), R.to_device(g, "f32")
    first = [a.numpy().copy() for a in ms.gated_scan(X, G)]
    for _ in range(4):
        for a, b in zip(first, ms.gated_scan(X, G)):
            assert np.array_equal(a, b.numpy())


VIEWS = {
    "transposed": lambda a: ms.permute(a, (0, 2, 1)),
    "flipped": lambda a: ms.flip(a, 1),
    "columns": lambda a: a[:, :, 1:],
    "stepped": lambda a: a[:, ::2, ::3],
    "steps": lambda a: a[:, 3:, :],
    "one": lambda a: a[:, :, 4:5],
}
HOST = {
    "transposed": lambda a: a.transpose(0, 2, 1), "flipped": lambda a: a[:, ::-1], "columns": lambda a: a[:, :, 1:],
    "stepped": lambda a: a[:, ::2, ::3], "steps": lambda a: a[:, 3:, :], "one": lambda a: a[:, :, 4:5],
}


@pytest.mark.parametrize("axis", [1, 2])
@pytest.mark.parametrize("view", sorted(VIEWS))
def test_views(view, axis):
    """Every operand as a view, and each one as a view beside plain ones."""
    rng = np.random.default_rng(11)
    base = (2, 60, 39)
    dev = {k: ms.array(R.rounded(rng.random(base) * 0.9, "f32"), dtype="f32") for k in ("x", "g", "h", "dh")}
    host = {k: HOST[view](R.values(v)) for k, v in dev.items()}
    plain = {k: ms.array(v, dtype="f32") for k, v in host.items()}
    views = {k: VIEWS[view](v) for k, v in dev.items()}
    for turned in (["x", "g", "h", "dh"], ["x"], ["g"], ["h"], ["dh"]):
        a = {k: views[k] if k in turned else plain[k] for k in plain}
        for kind in ("decay", "blend"):
            want = R.scan(host["x"], host["g"], None, None, axis, kind)
            bound, E = forward_bounds(host["x"], host["g"], None, None, axis, kind, want[0], "f32")
            h, s = ms.gated_scan(a["x"], a["g"], axis=axis, kind=kind)
            check(R.values(h), want[0], bound, (view, turned, "h"))
            ref = ms.gated_scan_grad(plain["dh"], plain["x"], plain["g"], plain["h"], axis=axis, kind=kind)
            got = ms.gated_scan_grad(a["dh"], a["x"], a["g"], a["h"], axis=axis, kind=kind)
            gw = R.scan_grad(host["dh"], host["x"], host["g"], host["h"], None, None, None, axis, kind)
            for i in range(2):
                # all values are positive: no cancellation, so the bound of the plain call's own terms holds
                check(R.values(got[i]), gw[i], 2e-5 * np.abs(gw[i]).max(), (view, turned, i))
                check(R.values(ref[i]), gw[i], 2e-5 * np.abs(gw[i]).max(), (view, "plain", i))


def test_nothing_crosses_a_reset():
    """NaN and infinities before a reset, and in the first state, stay there, forward and backward, in short and long rows
    and in both layouts."""
    rng = np.random.default_rng(12)
    for steps in (6, 40, 700, 5000):
        for axis in (1, 2):
            shape = (1, steps, 16) if axis == 1 else (1, 16, steps)
            x = rng.standard_normal(shape)
            g = rng.random(shape)
            at = steps // 2
            cut = np.zeros((1, steps, 1) if axis == 1 else (1, 1, steps), bool)
            cut.reshape(-1)[at] = True
            early = (slice(None), slice(0, at)) if axis == 1 else (slice(None), slice(None), slice(0, at))
            late = (slice(None), slice(at, None)) if axis == 1 else (slice(None), slice(None), slice(at, None))
            for bad in (np.nan, np.inf):
                xb, first = x.copy(), np.full((1, 16), bad)
                if axis == 1:
                    xb[:, at // 2, :] = bad
                else:
                    xb[:, :, at // 2] = bad
                h, s = ms.gated_scan(ms.array(xb, dtype="f32"), ms.array(g, dtype="f32"), ms.array(first, dtype="f32"),
                                     reset=ms.array(cut, dtype="bool"), axis=axis)
                h, s = R.values(h), R.values(s)
                want, ws = R.scan(x[late], g[late], None, None, axis, "decay")
                assert np.isfinite(h[late]).all() and np.isfinite(s).all(), (steps, axis, bad)
                assert np.allclose(h[late], want, rtol=1e-4, atol=1e-5) and np.allclose(s, ws, rtol=1e-4, atol=1e-5)
                assert not np.isfinite(np.take(h, at - 1, axis)).any()
                # backward: what lies behind the reset does not reach what lies before it
                db = rng.standard_normal(shape)
                dbad = db.copy()
                dbad[late] = bad
                got = ms.gated_scan_grad(ms.array(dbad, dtype="f32"), ms.array(x, dtype="f32"), ms.array(g, dtype="f32"),
                                         ms.array(x, dtype="f32"), ms.array(np.ones((1, 16)), dtype="f32"),
                                         reset=ms.array(cut, dtype="bool"), dstate=ms.array(first, dtype="f32"), axis=axis)
                dx, dg, d0 = (R.values(v) for v in got)
                wx, wg, w0 = R.scan_grad(db[early], x[early], g[early], x[early], np.ones((1, 16)), None, None, axis, "decay")
                assert np.allclose(dx[early], wx, rtol=1e-4, atol=1e-5) and np.allclose(dg[early], wg, rtol=1e-4, atol=1e-5)
                assert np.allclose(d0, w0, rtol=1e-4, atol=1e-5)
                # the state before the reset may be anything: its gate's gradient is 0
                hb = x.copy()
                if axis == 1:
                    hb[:, at - 1] = bad
                else:
                    hb[:, :, at - 1] = bad
                dg = R.values(ms.gated_scan_grad(ms.array(db, dtype="f32"), ms.array(x, dtype="f32"), ms.array(g, dtype="f32"),
                                                 ms.array(hb, dtype="f32"), reset=ms.array(cut, dtype="bool"), axis=axis)[1])
                assert (np.take(dg, at, axis) == 0).all()


def test_nan_gates_stay_visible():
    """A NaN gate gives NaN from its step on, also beside resets elsewhere."""
    for axis, shape in ((1, (1, 600, 8)), (2, (1, 8, 600))):
        x, g = np.ones(shape), np.full(shape, 0.5)
        at = (slice(None), 300) if axis == 1 else (slice(None), slice(None), 300)
        g[at] = np.nan
        cut = np.zeros((1, 600, 1) if axis == 1 else (1, 1, 600), bool)
        cut.reshape(-1)[100] = True
        for kind in ("decay", "blend"):
            for reset in (None, ms.array(cut, dtype="bool")):
                h = R.values(ms.gated_scan(ms.array(x, dtype="f32"), ms.array(g, dtype="f32"), axis=axis, kind=kind,
                                           reset=reset)[0])
                h = np.moveaxis(h, axis, 0)
                assert np.isfinite(h[:300]).all() and np.isnan(h[300:]).all()


def test_extreme_preactivations():
    """Gates whose sigmoid is 0 or 1 in every digit: no NaN from the exponential's ends."""
    g = np.array([-np.inf, -1e4, -100.0, -30.0, 0.0, 30.0, 100.0, 1e4, np.inf])
    x = np.full((1, 1, 9), 2.0)
    h, _ = ms.gated_scan(ms.array(x, dtype="f32"), ms.array(g.reshape(1, 1, 9), dtype="f32"),
                         ms.array(np.full((1, 9), 3.0), dtype="f32"), kind="blend")
    s = R.sigmoid(g)
    assert np.allclose(R.values(h).reshape(-1), s * 3 + R.sigmoid(-g) * 2, rtol=1e-6)
    got = ms.gated_scan_grad(ms.array(np.ones((1, 1, 9)), dtype="f32"), ms.array(x, dtype="f32"),
                             ms.array(g.reshape(1, 1, 9), dtype="f32"), h, ms.array(np.full((1, 9), 3.0), dtype="f32"),
                             kind="blend")
    assert np.allclose(R.values(got[0]).reshape(-1), R.sigmoid(-g), rtol=1e-6)
    assert np.allclose(R.values(got[1]).reshape(-1), s * R.sigmoid(-g), rtol=2e-6)


def test_steps_continue_a_sequence():
    """Prompt and single steps, the state handed on, against the whole sequence in one call."""
    rng = np.random.default_rng(13)
    x, g, _, _ = case(rng, (3, 40, 50), 1, "blend", "bf16", "bf16")
    X, G = R.to_device(x, "bf16"), R.to_device(g, "bf16")
    want, state = R.scan(x, g, None, None, 1, "blend")
    parts = []
    h, s = ms.gated_scan(X[:, :25, :], G[:, :25, :], kind="blend")
    parts.append(R.values(h))
    for t in range(25, 40):
        h, s = ms.gated_scan(X[:, t:t + 1, :], G[:, t:t + 1, :], s, kind="blend")
        parts.append(R.values(h))
    bound, E = forward_bounds(x, g, None, None, 1, "blend", want, "bf16")
    check(np.concatenate(parts, 1), want, bound, "h")
    check(R.values(s), state, last_of(E, 1) + 40 * R.EPS * np.abs(state), "state")


def test_empty_calls():
    for shape in ((2, 0, 5), (0, 4, 5), (2, 4, 0)):
        x = ms.array(np.zeros(shape), dtype="f32")
        lanes = (shape[0], shape[2])
        h0 = ms.array(np.full(lanes, 3.0), dtype="f32")
        h, s = ms.gated_scan(x, x, h0)
        assert h.shape == shape and (s.numpy() == h0.numpy()).all()
        assert (ms.gated_scan(x, x)[1].numpy() == 0).all()
        dx, dg, d0 = ms.gated_scan_grad(x, x, x, x, h0, dstate=h0)
        assert dx.shape == shape and dg.shape == shape and (d0.numpy() == h0.numpy()).all()
    # a gate shared along an axis of no elements has a gradient of zero
    x = ms.array(np.zeros((2, 0, 5)), dtype="f32")
    g = ms.array(np.ones((1, 1, 5)), dtype="f32")
    assert (ms.gated_scan_grad(x, x, g, x)[1].numpy() == 0).all()


def test_results_go_to_given_arrays():
    rng = np.random.default_rng(14)
    x, g, first, _ = case(rng, (2, 30, 20), 1, "decay", "f32", "f32", h0=True)
    X, G, H0 = (ms.array(v, dtype="f32") for v in (x, g, first))
    out, st = ms.array(np.zeros((2, 30, 20)), dtype="f32"), ms.array(np.zeros((2, 20)), dtype="f32")
    h, s = ms.gated_scan(X, G, H0, out=out, state_out=st)
    assert h.data_ptr == out.data_ptr and s.data_ptr == st.data_ptr
    fresh = ms.gated_scan(X, G, H0)
    assert (out.numpy() == fresh[0].numpy()).all() and (st.numpy() == fresh[1].numpy()).all()
    outs = tuple(ms.array(np.zeros(v), dtype="f32") for v in ((2, 30, 20), (2, 30, 20), (2, 20)))
    got = ms.gated_scan_grad(X, X, G, h, H0, out=outs)
    fresh = ms.gated_scan_grad(X, X, G, h, H0)
    for a, b, c in zip(outs, got, fresh):
        assert a.data_ptr == b.data_ptr and (a.numpy() == c.numpy()).all()


def test_other_streams():
    """Inputs written on one stream and used on another, results used on a third."""
    rng = np.random.default_rng(15)
    x, g, _, _ = case(rng, (4, 3000, 256), 1, "decay", "f32", "f32")
    a, b = ms.Stream(), ms.Stream()
    X, G = ms.array(x, dtype="f32"), ms.array(g, dtype="f32")
    zero = ms.array(np.zeros(1), dtype="f32")
    want = ms.gated_scan(X, G)[0].numpy()
    for _ in range(3):
        with ms.stream(a):
            X2 = ms.add(X, zero)
        with ms.stream(b):
            h, s = ms.gated_scan(X2, G)
            del X2
        with ms.stream(a):
            y = ms.add(h, zero)
        assert (y.numpy() == want).all()


def test_gradient_against_differences():
    """The gradient along random directions against central differences of the 64-bit forward form."""
    rng = np.random.default_rng(16)
    for kind in ("decay", "blend"):
        for gshape in ((2, 50, 4, 8), (2, 50, 4, 1)):
            shape, axis = (2, 50, 4, 8), 1
            x, g, first, cut = case(rng, shape, axis, kind, "f32", "f32", gshape, True, (2, 50, 1, 1))
            w, ws = rng.standard_normal(shape), rng.standard_normal((2, 4, 8))
            h = R.scan(x, g, first, cut, axis, kind)[0]
            got = ms.gated_scan_grad(*(ms.array(v, dtype="f32") for v in (w, x, g, h, first)),
                                     reset=ms.array(cut, dtype="bool"), dstate=ms.array(ws, dtype="f32"), axis=axis, kind=kind)

            def loss(x, g, f):
                h, s = R.scan(x, g, f, cut, axis, kind)
                return (w * h).sum() + (ws * s).sum()

            step = 1e-5
            for i, v in enumerate((x, g, first)):
                u = rng.standard_normal(v.shape)
                args = [x, g, first]
                at = [(loss(*(a + d * u if j == i else a for j, a in enumerate(args)))) for d in (step, -step)]
                slope = (at[0] - at[1]) / (2 * step)
                grad = R.values(got[i])
                # the gradient's f32 entries: 1e-5 of their size at these 50 steps; the difference: step^2 and 64-bit noise
                assert abs((grad * u).sum() - slope) <= 1e-5 * np.abs(grad * u).sum() + 1e-4


def test_refusals():
    f = lambda *s: ms.array(np.zeros(s), dtype="f32")  # noqa: E731
    x, h0 = f(2, 6, 4), f(2, 4)
    half = ms.astype(x, "bf16")
    wide = ms.array(np.zeros((2, 6, 4)), dtype="f64")
    flags = ms.array(np.zeros((2, 6, 1)), dtype="bool")
    for call, error in [
        (lambda: ms.gated_scan(wide, wide), ms.DtypeError),
        (lambda: ms.gated_scan(x, half), ms.DtypeError),
        (lambda: ms.gated_scan(half, ms.astype(x, "f16")), ms.DtypeError),
        (lambda: ms.gated_scan(x, x, half), ms.DtypeError),
        (lambda: ms.gated_scan(x, x, f(4, 2)), ms.ShapeError),
        (lambda: ms.gated_scan(x, x, f(2, 6, 4)), ms.ShapeError),
        (lambda: ms.gated_scan(x, f(2, 6, 3)), ms.ShapeError),
        (lambda: ms.gated_scan(x, f(1, 2, 6, 4)), ms.ShapeError),
        (lambda: ms.gated_scan(x, x, axis=3), ms.ShapeError),
        (lambda: ms.gated_scan(f(4), f(4)), ms.ShapeError),
        (lambda: ms.gated_scan(x, x, reset=f(2, 6, 1)), ms.DtypeError),
        (lambda: ms.gated_scan(x, x, reset=ms.array(np.zeros((2, 5, 1)), dtype="bool")), ms.ShapeError),
        (lambda: ms.gated_scan(x, x, kind="other"), ValueError),
        (lambda: ms.gated_scan(x, f(2, 6, 4), out=x), ms.MemoryError),
        (lambda: ms.gated_scan(x, x, h0, state_out=h0), ms.MemoryError),
        (lambda: ms.gated_scan(x, x, out=f(2, 6, 5)), ms.ShapeError),
        (lambda: ms.gated_scan(x, x, out=half), ms.DtypeError),
        (lambda: ms.gated_scan(x, x, out=ms.permute(f(4, 6, 2), (2, 1, 0))), ms.ShapeError),
        (lambda: ms.gated_scan_grad(f(2, 6, 5), x, x, x), ms.ShapeError),
        (lambda: ms.gated_scan_grad(half, x, x, x), ms.DtypeError),
        (lambda: ms.gated_scan_grad(x, x, x, half), ms.DtypeError),
        (lambda: ms.gated_scan_grad(x, x, x, x, dstate=f(2, 5)), ms.ShapeError),
        (lambda: ms.gated_scan_grad(x, x, x, x, out=(f(2, 6, 4), f(2, 6, 4), f(2, 4))), ms.ShapeError),
        (lambda: ms.gated_scan_grad(x, x, x, x, out=(f(2, 6, 4), f(2, 6, 4))), TypeError),
        (lambda: ms.gated_scan_grad(x, x, x, x, out=(x, None, None)), ms.MemoryError),
    ]:
        with pytest.raises(error):
            call()
    o = f(2, 6, 4)
    with pytest.raises(ms.MemoryError):
        ms.gated_scan_grad(x, x, x, x, out=(o, o, None))
    ms.gated_scan(x, x, reset=flags)  # and the calls that they differ from are taken
