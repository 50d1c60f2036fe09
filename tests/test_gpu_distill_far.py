"""The distillation loss and its gradient where logits lie so far from 0, or temperatures so low, that m log2(e) / T is no
small number of 32 bits: masks of -1e9 and beyond that leave a row nothing else, large offsets of all logits, far ones in
some segments or rows only."""
import numpy as np
import pytest

from tests import vocab_reference as R
from tests.test_gpu_distill import check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temp,weight", [(1.0, 0.5), (2.0, 0.5), (1.5, 0.5), (0.01, 1.0), (2.0 ** -20, 0.3), (2.0 ** 20, 0.5)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("width", [40, 9000])
def test_rows_of_one_far_value(width, dt, temp, weight):
    """Every column alike, as a mask of that value leaves it: uniform, whatever the value."""
    rng = np.random.default_rng(width)
    far = [1e3, -1e4, 1e7, -2e7, -1e9, 1e9, -1e10, 3e10, -1e15, 1e20, -1e30, -2e30, 1e30, 3e38]
    _, index, teacher, label = inputs(rng, len(far), width, 3, dt, "f32")
    z = R.rounded(np.repeat(np.array(far)[:, None], width, 1), dt)
    _, sums, _ = check(z, index, teacher, label, dt, "f32", temp, weight)
    assert np.isfinite(sums.numpy()).all()


@pytest.mark.parametrize("temp,weight", [(1.0, 0.5), (2.0, 0.5), (3.0, 0.5)])
@pytest.mark.parametrize("rows,width", [(4, 3000), (4, 70001), (2100, 300)])
def test_far_rows_with_a_spread(rows, width, temp, weight):
    """Logits some steps of f32 apart, at offsets where m log2(e) is below 2^24, about it and above it; rows whole and in segments."""
    rng = np.random.default_rng(width)
    for offset in (4e6, -8e6, 1.1e7, -1.17e7, 2.4e7, -5e7, 2e9, -3e9, 1e10):
        z, index, teacher, label = inputs(rng, min(rows, 7), width, 5, "f32", "f32", spread=4.0)
        rep = np.arange(rows) % len(z)
        z = R.rounded(z + offset, "f32")
        check(z[rep], index[rep], teacher[rep], label[rep], "f32", "f32", temp, weight)


@pytest.mark.parametrize("temp", [1.0, 2.0, 2.5])
@pytest.mark.parametrize("width", [900, 9000, 70001])
def test_across_the_border(width, temp):
    """Maxima that rise over where far logits begin, from both signs: a first part far below 0 and a second less far, parts of
    one row near and far, and rows that are far but for one column."""
    rng = np.random.default_rng(width)
    border = 2.0 ** 24 * np.log(2.0)  # of m log2(e)
    z, index, teacher, label = inputs(rng, 7, width, 4, "f32", "f32")
    steps = np.arange(width) / width
    z[0] = -border - 6 + 12 * steps            # rises over -border by steps of 1
    z[1] = border - 6 + 12 * steps             # and over border
    z[2] = -border + 6 - 12 * steps            # falls
    z[3, : width // 2] = -1e10
    z[4] = -1e10
    z[4, width - 1] = 2.0
    z[5, width // 3] = 1e10
    z[6] = np.where(steps < 0.5, -border - 1, -border + 1)
    check(R.rounded(z, "f32"), index, teacher, label, "f32", "f32", temp, 0.5)
