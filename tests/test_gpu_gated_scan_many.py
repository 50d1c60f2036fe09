"""Gated scans of as many rows and elements as large calls have: rows of unit-stride steps over several tiles without a
look-back, streaming loads and stores (more than 32 MB), and long scans of very many lanes, which go step by step."""
import numpy as np
import pytest

from tests.test_gpu_gated_scan import run_forward, run_grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["decay", "blend"])
@pytest.mark.parametrize("shape", [(1100, 1500), (1030, 4500), (2, 520, 2049), (3, 400, 4096)])
def test_rows_of_several_tiles(kind, shape):
    rng = np.random.default_rng(shape[-1])
    reset = (1,) * (len(shape) - 1) + shape[-1:]
    run_forward(rng, shape, -1, kind, "f32", "f32", h0=True, reset=reset)
    run_grad(rng, shape, -1, kind, "bf16", "bf16", h0=True, reset=reset, dstate=True)
    run_forward(rng, shape, -1, kind, "f16", "f32")
    run_grad(rng, shape, -1, kind, "f32", "f32")


@pytest.mark.parametrize("kind", ["decay", "blend"])
@pytest.mark.parametrize("shape,axis,dt", [((2, 2100, 2048), 1, "f32"), ((4, 1100, 4096), 1, "bf16"), ((60, 100, 2048), 1, "f32"),
                                           ((2, 2100, 2040), 1, "f32"), ((1100, 8000), 1, "f32"), ((300, 56000), 1, "bf16"),
                                           ((21000, 400), 1, "f32"), ((150000, 60), 1, "f32")])
def test_streaming(kind, shape, axis, dt):
    rng = np.random.default_rng(shape[0])
    reset = tuple(n if i == axis else 1 for i, n in enumerate(shape))
    run_forward(rng, shape, axis, kind, dt, "f32", h0=True, reset=reset)
    run_grad(rng, shape, axis, kind, dt, "f32", h0=True, reset=reset, dstate=True)


def test_many_lanes_step_by_step():
    rng = np.random.default_rng(2)
    run_forward(rng, (1, 137, 524289), 1, "blend", "bf16", "bf16", h0=True)
    run_grad(rng, (1, 137, 524289), 1, "decay", "bf16", "bf16", reset=(1, 137, 1), dstate=True)
