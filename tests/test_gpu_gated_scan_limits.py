"""The gated scan's look-back when its waits run out, and calls at the edges of what it takes."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import blocks_reference as R
from tests.test_gpu_gated_scan import run_forward, run_grad
from tests.test_gpu_wait_faults import _fresh_stream_case

pytestmark = pytest.mark.gpu


def arrays(shape, axis):
    rng = np.random.default_rng(5)
    x = R.rounded(rng.standard_normal(shape), "f32")
    g = R.rounded(R.sigmoid(rng.standard_normal(shape) + 2.0), "f32")
    want, _ = R.scan(x, g, None, None, axis, "decay")
    return x, g, want


# tiles of channels, and rows of unit-stride steps, both split over workgroups
@pytest.mark.parametrize("shape,axis", [((2, 1000, 24), 1), ((2, 3, 5000), 2)])
def test_the_look_back_gives_up_and_recovers(shape, axis):
    x, g, want = arrays(shape, axis)

    def check(got, what):
        # decays below 1 and about e^-0.13 on average: sums of some ten terms of size 1, each with a rounding of 2^-24
        assert np.abs(got - want).max() <= 1e-4, what

    _fresh_stream_case(lambda: (ms.array(x, dtype="f32"), ms.array(g, dtype="f32")),
                       lambda X, G: ms.gated_scan(X, G, axis=axis)[0], check)
    back, _ = R.scan(np.flip(x, axis), np.flip(np.roll(g, -1, axis), axis), None, None, axis, "decay")
    back = np.flip(back, axis)  # G[t] = dh[t] + g[t+1] G[t+1], and nothing comes in at the end

    def check_grad(got, what):
        assert np.abs(got - back).max() <= 1e-4, what

    _fresh_stream_case(lambda: (ms.array(x, dtype="f32"), ms.array(g, dtype="f32"), ms.array(want, dtype="f32")),
                       lambda D, G, H: ms.gated_scan_grad(D, D, G, H, axis=axis)[0], check_grad)


@pytest.mark.parametrize("kind", ["decay", "blend"])
def test_eight_dimensions_and_no_more(kind):
    rng = np.random.default_rng(8)
    run_forward(rng, (2, 1, 3, 2, 1, 2, 9, 5), 6, kind, "f32", "f32", gshape=(2, 1, 1, 2, 1, 1, 9, 5), h0=True)
    x = ms.array(np.zeros((1, 2, 1, 2, 1, 2, 1, 4, 4)), dtype="f32")
    with pytest.raises(ms.ShapeError):
        ms.gated_scan(x, x, kind=kind)


def test_vectors_that_end_inside_rows_of_any_size():
    rng = np.random.default_rng(9)
    for width in range(1, 40, 3):
        for steps in (3, 20, 300):
            run_forward(rng, (2, steps, width), 1, "blend", "bf16", "bf16", h0=True)
            run_forward(rng, (2, steps, width), 1, "decay", "f16", "f32", reset=(2, steps, 1))


# few steps of many lanes go step by step, one step more in tiles
@pytest.mark.parametrize("steps", [20, 21])
@pytest.mark.parametrize("dt,gdt", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")])
def test_few_steps_of_many_lanes(dt, gdt, steps):
    rng = np.random.default_rng(steps)
    run_forward(rng, (5, steps, 9999), 1, "blend", dt, gdt, h0=True, reset=(5, steps, 1))
    run_grad(rng, (5, steps, 9999), 1, "blend", dt, gdt, h0=True, reset=(5, steps, 1), dstate=True)


@pytest.mark.parametrize("steps", [1, 6, 8, 9, 20])
@pytest.mark.parametrize("width", [64, 125, 128, 200])
def test_few_steps_of_gates_shared_by_a_heads_channels(width, steps):
    rng = np.random.default_rng(width + steps)
    for dt, gdt in (("f16", "f32"), ("bf16", "bf16"), ("f32", "f32")):
        for heads in (3, 80):
            run_grad(rng, (5, steps, heads, width), 1, "decay", dt, gdt, gshape=(5, steps, heads, 1), h0=True, dstate=True)
