"""Norms around a block with more rows than there are workgroups or groups of lanes for them: every one takes several, with the
next row's loads, dropout bits and column sums carried along."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import blocks_reference as R
from tests.test_gpu_norm_residual import OPTIONS, run

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


def kept(rows, width, p, seed, offset):
    """blocks_reference.kept for all rows at once."""
    u = np.uint64
    m, blocks = u(0xFFFFFFFF), -(-width // 8)
    c0 = np.broadcast_to(np.arange(blocks, dtype=u), (rows, blocks))
    c1 = np.broadcast_to(np.arange(rows, dtype=u)[:, None], (rows, blocks))
    c2, c3 = np.full((rows, blocks), offset & 0xFFFFFFFF, u), np.full((rows, blocks), offset >> 32, u)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = u(0xD2511F53) * c0, u(0xCD9E8D57) * c2
        c0, c1, c2, c3 = (b >> u(32)) ^ c1 ^ u(k0), b & m, (a >> u(32)) ^ c3 ^ u(k1), a & m
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    halves = np.stack([h for w in (c0, c1, c2, c3) for h in (w & u(0xFFFF), w >> u(16))], -1)
    return halves.reshape(rows, blocks * 8)[:, :width] >= round(p * 65536)


@pytest.fixture
def fast(monkeypatch):
    assert np.array_equal(kept(7, 45, 0.3, 2 ** 40 + 9, 2 ** 33 + 1), R.kept(7, 45, 0.3, 2 ** 40 + 9, 2 ** 33 + 1))
    monkeypatch.setattr(R, "kept", kept)


# Rows in turn for lanes of 16, 32 and 64, for workgroups with one, two and three vectors a thread, and past the registers;
# whole vectors and parts of them; of these, 4.2 million elements and more in whole vectors take streaming loads.
@pytest.mark.parametrize("rows,width", [(9000, 60), (5000, 125), (3000, 256), (9000, 472), (33100, 100), (2100, 600), (5003, 1111),
                                        (1100, 4096), (2500, 2048), (600, 5120), (600, 8192), (580, 8190), (530, 12280), (1100, 12300)])
def test_several_rows_in_turn(fast, rows, width):
    rng = np.random.default_rng(rows)
    run(rng, (rows, width), "bf16", "bf16", OPTIONS[0], p=0.2)
    run(rng, (rows, width), "f16", "f32", OPTIONS[1], p=0.2)


def test_many_elements_of_dropout(fast):
    """More than 32 MB: streaming loads and stores."""
    for dt, shape in (("f32", (2100, 4096)), ("bf16", (4200, 4099)), ("f32", (3, 700, 4096))):
        X = R.to_device(np.ones(shape, np.float32), dt)
        y = R.values(ms.dropout(X, 0.3, seed=11, offset=12)).reshape(-1, shape[-1])
        scale = float(R.rounded(np.array([np.float32(R.keep_scale(0.3))]), dt)[0])
        assert np.array_equal(y, np.where(kept(*y.shape, 0.3, 11, 12), scale, 0.0))
