"""Norms around a block at widths where a thread holds several vectors, whole and odd, with dropout."""
import numpy as np
import pytest

from tests.test_gpu_norm_residual import OPTIONS, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("o", OPTIONS[:4], ids=lambda o: f"{o['post']}-{o['pre']}")
@pytest.mark.parametrize("width", [4099, 4432, 8190, 8193, 12287, 12288, 13056])
def test_several_vectors_a_thread(width, o):
    rng = np.random.default_rng(width)
    run(rng, (5, width), "bf16", "bf16", o, p=0.2)
    run(rng, (3, width), "f32", "f32", o, p=0.1)


@pytest.mark.parametrize("width", [8, 60, 64, 100, 124, 128, 132, 252, 256, 260])
def test_several_rows_a_wave(width):
    rng = np.random.default_rng(width)
    for rows in (1, 15, 16, 17, 700):
        run(rng, (rows, width), "f16", "f32", OPTIONS[1], p=0.2)
        run(rng, (rows, width - 1), "bf16", "bf16", OPTIONS[0])
