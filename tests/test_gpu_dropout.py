"""dropout on the GPU: which elements are kept is whole-number arithmetic and has to be the generator's exactly; a kept
value is one f32 product, rounded once more to the array's type."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import blocks_reference as R

pytestmark = pytest.mark.gpu


def want(x, p, seed, offset, dt):
    rows = int(np.prod(x.shape[:-1])) if x.ndim else 1
    width = x.shape[-1] if x.ndim else 1
    keep = R.kept(rows, width, p, seed, offset).reshape(x.shape)
    scale = np.float64(np.float32(R.keep_scale(p)))
    product = (x * scale).astype(np.float32).astype(np.float64)
    return np.where(keep, R.rounded(product, dt), 0.0), keep


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(), (1,), (7,), (8,), (9,), (1000,), (5, 3), (3, 64), (4, 257), (2, 3, 41), (1, 1, 8), (70, 1)])
def test_exact(dt, shape):
    rng = np.random.default_rng(1)
    x = np.asarray(R.rounded(rng.standard_normal(shape), dt))
    for p, seed, offset in ((0.1, 5, 0), (0.5, 2 ** 40 + 3, 2 ** 33 + 1), (0.0, 1, 0), (1.0, 1, 0), (1e-5, 3, 4)):
        y = ms.dropout(R.to_device(x, dt), p, seed=seed, offset=offset)
        assert y.dtype == dt and y.shape == shape
        assert np.array_equal(R.values(y), want(x, p, seed, offset, dt)[0]), (p, seed, offset)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_views_keep_what_their_copies_keep(dt):
    rng = np.random.default_rng(2)
    x = R.rounded(rng.standard_normal((4, 30, 50)), dt)
    X = R.to_device(x, dt)
    for v, h in [(X[:, :, 3:], x[:, :, 3:]), (ms.permute(X, (2, 0, 1)), x.transpose(2, 0, 1)), (ms.flip(X, 2), x[:, :, ::-1]),
                 (X[:, ::2, ::3], x[:, ::2, ::3]), (X[1], x[1]), (X[:, 5, :], x[:, 5])]:
        assert np.array_equal(R.values(ms.dropout(v, 0.3, seed=9, offset=2)), want(np.ascontiguousarray(h), 0.3, 9, 2, dt)[0])


def test_dropped_values_are_zero_whatever_they_were():
    x = np.full((40, 64), np.nan, np.float32)
    x[::2] = np.inf
    y = ms.dropout(ms.array(x), 0.5, seed=3).numpy()
    keep = R.kept(40, 64, 0.5, 3, 0)
    assert (y[~keep] == 0).all() and not np.isfinite(y[keep]).any()


def test_rate_and_independence():
    """The share kept over a million elements is within five deviations of the rate; other seeds, offsets and rows are other
    masks."""
    x = ms.ones((1024, 1024))
    masks = [ms.dropout(x, 0.3, seed=s, offset=o).numpy() != 0 for s, o in ((1, 0), (2, 0), (1, 1))]
    n = 1 << 20
    for m in masks:
        assert abs(m.mean() - 0.7) < 5 * np.sqrt(0.21 / n) + 2.0 ** -17
    for a, b in ((0, 1), (0, 2), (1, 2)):
        same = (masks[a] == masks[b]).mean()
        assert abs(same - (0.49 + 0.09)) < 5 * np.sqrt(0.58 * 0.42 / n)
    assert abs((masks[0][1:] == masks[0][:-1]).mean() - 0.58) < 5 * np.sqrt(0.58 * 0.42 / n)


def test_the_gradient_is_the_same_call():
    rng = np.random.default_rng(4)
    dy = rng.standard_normal((9, 100)).astype(np.float32)
    y = ms.dropout(ms.ones((9, 100)), 0.25, seed=8, offset=1).numpy()
    dx = ms.dropout(ms.array(dy), 0.25, seed=8, offset=1).numpy()
    assert np.array_equal(dx, dy * y)


def test_empty_and_out():
    assert ms.dropout(ms.array(np.zeros((0, 4)), dtype="f32"), 0.5, seed=1).shape == (0, 4)
    assert ms.dropout(ms.array(np.zeros((4, 0)), dtype="f32"), 0.5, seed=1).shape == (4, 0)
    x, o = ms.ones((3, 5)), ms.array(np.zeros((3, 5)), dtype="f32")
    assert ms.dropout(x, 0.5, seed=1, out=o).data_ptr == o.data_ptr
    assert np.array_equal(o.numpy(), ms.dropout(x, 0.5, seed=1).numpy())


def test_refusals():
    x = ms.ones((3, 4))
    for call, error in [
        (lambda: ms.dropout(x, -0.1, seed=1), ValueError),
        (lambda: ms.dropout(x, 1.5, seed=1), ValueError),
        (lambda: ms.dropout(x, float("nan"), seed=1), ValueError),
        (lambda: ms.dropout(x, 0.5, seed=-1), TypeError),
        (lambda: ms.dropout(ms.array(np.zeros(3), dtype="f64"), 0.5, seed=1), ms.DtypeError),
        (lambda: ms.dropout(ms.array(np.zeros(3), dtype="i32"), 0.5, seed=1), ms.DtypeError),
        (lambda: ms.dropout(x, 0.5, seed=1, out=x), ms.MemoryError),
        (lambda: ms.dropout(x, 0.5, seed=1, out=ms.ones((4, 3))), ms.ShapeError),
    ]:
        with pytest.raises(error):
            call()
