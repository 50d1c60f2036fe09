"""Biases of named columns, and of all, in the logits' own 16-bit types; masks of unsigned words, of one row."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import vocab_reference as R
from tests.test_gpu_adjust_logits import check, some

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,to", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("bias_dt", ["own", "f32"])
@pytest.mark.parametrize("width,m", [(7, 3), (2049, 64), (5003, 65), (20000, 300), (50001, 1024)])
def test_biases_of_named_columns(width, m, bias_dt, dt, to):
    bias_dt = dt if bias_dt == "own" else bias_dt
    rng = np.random.default_rng(width + m)
    z = R.draw(rng, (4, width), dt, 3.0)
    index = rng.integers(-1, width + 1, (4, m))
    index[1] = rng.permutation(max(width, m))[:m]  # (some past the last column where there are too few)
    index[2, : m // 2] = width - 1                 # many of one
    bias = R.draw(rng, (4, m), bias_dt, 4.0)
    for id_dt in ("i32", "i64"):
        check(z, dt, to, bias=bias, bias_index=index, bias_dt=bias_dt, id_dt=id_dt)
    check(z, dt, to, bias=bias, bias_index=index, bias_dt=bias_dt, allowed=rng.random((4, width)) < 0.7, packed=True,
          **some(rng, 4, width, 50))


def test_views_of_biases():
    """Rows of biases and of their columns apart by a stride, and columns in steps."""
    rng = np.random.default_rng(3)
    z = R.draw(rng, (6, 900), "bf16", 3.0)
    index, bias = rng.integers(0, 900, (6, 40)), R.draw(rng, (6, 40), "bf16")
    Z, I, B = R.to_device(z, "bf16"), R.ids(index), R.to_device(bias, "bf16")
    for s in ((slice(None), slice(3, 30)), (slice(None), slice(0, 40, 3)), (slice(None), slice(0, 1))):
        got = ms.adjust_logits(Z, bias=B[s], bias_index=I[s], dtype="f32")
        want, bound = map(np.stack, zip(*[R.adjust(z[r], bias=bias[s][r], bias_index=index[s][r]) for r in range(6)]))
        R.within(got, want, bound, "f32", str(s))


def test_unsigned_words_of_one_row():
    rng = np.random.default_rng(4)
    z, ok = R.draw(rng, (5, 1001), "f32"), rng.random(1001) < 0.5
    words = R.pack(ok)
    a = ms.adjust_logits(R.to_device(z, "f32"), allowed=ms.from_numpy(words)).numpy()
    b = ms.adjust_logits(R.to_device(z, "f32"), allowed=ms.from_numpy(words.view(np.int32))).numpy()
    assert np.array_equal(a, b) and np.array_equal(a, np.where(ok, z.astype(np.float32), -np.inf))
