"""Norms around a block with more rows than there are workgroups or groups of lanes for them: every one takes several, with the
next row's loads, dropout bits and column sums carried along."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import blocks_reference as R
from tests.test_gpu_norm_residual import OPTIONS

pytestmark = pytest.mark.gpu


def test_rows_past_the_registers_in_turn():
    """2053 rows of 16390 columns: the last ones as they are alone, where the formulas hold them."""
    rng = np.random.default_rng(1)
    rows, width, tail = 2053, 16390, 8
    x = R.rounded(rng.standard_normal((rows, width), dtype=np.float32), "bf16").astype(np.float32)
    X = R.to_device(x, "bf16")
    w = ms.array(1 + 0.1 * rng.standard_normal(width), dtype="f32")
    o = OPTIONS[1]
    r, y = ms.norm_residual(X, X, gate=X, post_weight=w, pre_weight=w, **o)
    part = X[rows - tail:, :]
    r1, y1 = ms.norm_residual(part, part, gate=part, post_weight=w, pre_weight=w, **o)
    assert np.array_equal(r[rows - tail:, :].numpy(), r1.numpy()) and np.array_equal(y[rows - tail:, :].numpy(), y1.numpy())
    xs = x[-tail:].astype(np.float64)
    wr, wy = R.block(xs, xs, xs, w.numpy(), 1.0, w.numpy(), 1.0, o)
    # bf16 results: half an ulp, and f32 sums over 16390 columns well below it
    assert np.allclose(R.values(r1), wr, rtol=2.0 ** -8, atol=2e-3) and np.allclose(R.values(y1), wy, rtol=2.0 ** -8, atol=2e-3)
