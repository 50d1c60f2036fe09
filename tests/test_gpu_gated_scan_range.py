"""Decays above 1 and below: wherever the states stay in range the answer does, however far the product of a run of decays
goes on the way; what leaves the range is seen.  Step-by-step 64-bit forms, with the bounds of tests/test_gpu_gated_scan.py: a
relative error of 6 x 2^-24 for each factor, whatever their order."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import blocks_reference as R
from tests.test_gpu_gated_scan import check, factor_error, forward_bounds

pytestmark = pytest.mark.gpu


def lanes_of(steps, axis, width, v):
    """A sequence of values as gates of `width` lanes."""
    v = np.broadcast_to(np.asarray(v, np.float64)[:, None], (steps, width))
    return v[None] if axis == 1 else v.T[None]


def up_and_down(up, n, times):
    """n steps of `up`, n of its (rounded) inverse, again and again."""
    down = float(np.float32(1.0 / up))
    return np.tile(np.concatenate([np.full(n, up), np.full(n, down)]), times)


# (decays, the first state): what its product reaches in between is beyond f32 on either side
SEQUENCES = {
    "1.5 up 256": (up_and_down(1.5, 256, 1), 1e-30),
    "2 up 128": (np.full(128, 2.0), 1e-30),
    "2 up 200": (np.full(200, 2.0), 1e-30),
    "2 down 200": (up_and_down(0.5, 200, 1), 1e30),
    "2 up 200 again": (up_and_down(2.0, 200, 12), 1e-30),
    "2 down 230 long": (up_and_down(0.5, 230, 20), 3e37),
    "3 up 140": (up_and_down(3.0, 140, 8), 1e-30),
    "-2 up 200": (up_and_down(-2.0, 200, 3), 1e-30),
    "steep": (np.tile([1e18, 1e18, 1e-18, 1e-18, 1e-30, 1e30, 1e30, 1e-30], 400), 1e-3),
}


@pytest.mark.parametrize("axis", [1, 2])
@pytest.mark.parametrize("width", [3, 72])
@pytest.mark.parametrize("name", sorted(SEQUENCES))
def test_states_in_range(name, width, axis):
    seq, first = SEQUENCES[name]
    steps = len(seq)
    rng = np.random.default_rng(steps + width)
    sign = R.rounded(rng.choice([-1.0, 1.0], width) * (1 + rng.random(width)) * first, "f32")[None]
    gates = R.rounded(lanes_of(steps, axis, width, seq), "f32")
    x = np.zeros(gates.shape)
    for dt in ("f32", "bf16"):
        want, state = R.scan(x, gates, sign, None, axis, "decay")
        assert np.abs(want).max() < 3e38 and np.abs(want).min() > 1.2e-38
        h, s = ms.gated_scan(R.to_device(x, dt), ms.array(gates, dtype="f32"), ms.array(sign, dtype="f32"), axis=axis)
        bound, E = forward_bounds(x, gates, sign, None, axis, "decay", want, dt)
        check(R.values(h), want, bound, (name, dt, "h"))
        check(R.values(s), state, np.take(E, steps - 1, axis) + 4 * R.EPS * np.abs(state), (name, dt, "state"))


@pytest.mark.parametrize("axis", [1, 2])
@pytest.mark.parametrize("name", sorted(SEQUENCES))
def test_gradients_in_range(name, axis):
    """What flows back from the last state alone: products of the decays behind a step, each with its relative error."""
    seq, first = SEQUENCES[name]
    seq = seq[::-1]
    steps, width = len(seq), 24
    gates = R.rounded(lanes_of(steps, axis, width, seq), "f32")
    zero = np.zeros(gates.shape)
    dstate = np.full((1, width), float(np.float32(first)))
    one = np.ones((1, width))
    h = np.ones(gates.shape)
    want = R.scan_grad(zero, zero, gates, h, one, None, dstate, axis, "decay")
    assert np.abs(want[0]).max() < 3e38 and np.abs(want[0]).min() > 1.2e-38
    dev = lambda v: ms.array(v, dtype="f32")  # noqa: E731
    got = ms.gated_scan_grad(dev(zero), dev(zero), dev(gates), dev(h), dev(one), dstate=dev(dstate), axis=axis)
    for g, w, what in zip(got, want, ("dx", "dgate", "dh0")):
        check(R.values(g), w, (steps * factor_error(gates, "decay") + 16 * R.EPS) * np.abs(w), (name, what))


@pytest.mark.parametrize("axis", [1, 2])
def test_growth_between_resets_and_from_nothing(axis):
    """Decays of 2 throughout: each document starts from nothing; and a state that a decay of 0 has ended stays 0 through any
    growth, until there is something to grow again."""
    rng = np.random.default_rng(3)
    steps, width = 6000, 40
    shape = (1, steps, width) if axis == 1 else (1, width, steps)
    cut = (np.arange(steps) % 90 == 17)
    gates = np.full(shape, 2.0)
    x = R.rounded(rng.standard_normal(shape), "f32")
    reset = cut.reshape((1, steps, 1) if axis == 1 else (1, 1, steps))
    first = R.rounded(rng.standard_normal((1, width)), "f32")
    want, state = R.scan(x, gates, first, reset, axis, "decay")
    h, s = ms.gated_scan(ms.array(x, dtype="f32"), ms.array(gates, dtype="f32"), ms.array(first, dtype="f32"),
                         reset=ms.array(reset, dtype="bool"), axis=axis)
    bound, E = forward_bounds(x, gates, first, reset, axis, "decay", want, "f32")
    check(R.values(h), want, bound, "h")

    seq = np.full(steps, 2.0)
    seq[3] = 0.0
    gates = lanes_of(steps, axis, width, seq)
    x = np.zeros(shape)
    at = (slice(None), 5950) if axis == 1 else (slice(None), slice(None), 5950)
    x[at] = 1.0
    want, state = R.scan(x, gates, first, None, axis, "decay")
    h, s = ms.gated_scan(ms.array(x, dtype="f32"), ms.array(gates, dtype="f32"), ms.array(first, dtype="f32"), axis=axis)
    assert np.array_equal(R.values(h), want) and np.array_equal(R.values(s), state)


@pytest.mark.parametrize("axis", [1, 2])
def test_what_leaves_the_range_is_seen(axis):
    """A state beyond f32's range is infinite or no number there.  Where it comes back in 64 bits it is the 64-bit one, or still
    infinite or no number, but never another: nothing is lost as if it were a reset."""
    for up, n, times in ((2.0, 300, 1), (1.5, 1500, 2), (2.0, 1500, 2)):
        seq = up_and_down(up, n, times)
        gates = R.rounded(lanes_of(len(seq), axis, 24, seq), "f32")
        zero, one = np.zeros(gates.shape), np.ones((1, 24))
        with np.errstate(over="ignore", invalid="ignore"):
            want, _ = R.scan(zero, gates, one, None, axis, "decay")
        h, s = ms.gated_scan(ms.array(zero, dtype="f32"), ms.array(gates, dtype="f32"), ms.array(one, dtype="f32"), axis=axis)
        h = R.values(h)
        out = ~(np.abs(want) < 3.4028235e38)
        assert out.any() and not np.isfinite(h[out]).any()
        back = ~out & np.isfinite(h)
        assert np.isfinite(np.moveaxis(h, axis, 0)[:int(127 / np.log2(up))]).all()
        assert (np.abs(h[back] - want[back]) <= (len(seq) * factor_error(gates, "decay") + 16 * R.EPS) * np.abs(want[back]) + 2.0 ** -126).all()
