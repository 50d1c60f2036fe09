"""Results of 64 MB and more, which are stored past the caches by kernels of their own, against the same rows in small calls, bit for
bit: a row's numbers do not depend on how many rows there are."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import vocab_reference as R
from tests.test_gpu_adjust_logits import check as check_adjusted
from tests.test_gpu_adjust_logits import some
from tests.test_gpu_distill import check as check_distilled
from tests.test_gpu_distill import inputs
from tests.test_gpu_embedding_many import check as check_embedding_grad
from tests.test_gpu_embedding_many import whole

pytestmark = pytest.mark.gpu

KINDS = 5
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def copies(rows, width, dt):
    """The kind of each of `rows` rows of `width`, which have 64 MB together."""
    assert rows * width * BYTES[dt] >= 64 << 20
    return np.arange(rows) % KINDS


def rows_for(width, dt):
    return -((-64 << 20) // (width * BYTES[dt]))


def same_rows(large, small, kind):
    """Every row of `large` against the row of its kind; the first, the last and some between one by one."""
    front = R.values(small)
    for r in np.unique(np.r_[0, 1, len(kind) - 1, len(kind) - 2, np.linspace(0, len(kind) - 1, 40).astype(int)]):
        assert np.array_equal(R.values(large[int(r)]), front[kind[r]], equal_nan=True), r
    # and all of them on the device, widened
    wide = ms.embedding(large, R.ids(np.arange(len(kind))), dtype="f32"), ms.embedding(small, R.ids(kind), dtype="f32")
    assert not ms.ne(*wide).numpy().any()


@pytest.mark.parametrize("dt,to", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("width,length", [(4099, 0), (4099, 40), (32768, 300), (50001, 66000), (20000, 20000)])
def test_adjusted_logits(width, length, dt, to):
    rng = np.random.default_rng(width + length)
    z = R.draw(rng, (KINDS, width), dt, 3.0)
    kw = some(rng, KINDS, width, length) if length else {}
    ok, bias, index = rng.random((KINDS, width)) < 0.7, R.draw(rng, (KINDS, 6), "f32"), rng.integers(-1, width, (KINDS, 6))
    small = check_adjusted(z, dt, to, allowed=ok, packed=True, bias=bias, bias_index=index, **kw)
    kind = copies(rows_for(width, to), width, to)
    large = ms.adjust_logits(ms.embedding(R.to_device(z, dt), R.ids(kind)), dtype=to, allowed=ms.from_numpy(R.pack(ok)[kind]),
                             bias=ms.from_numpy(bias.astype(np.float32)[kind]), bias_index=R.ids(index[kind]),
                             **{k: ms.from_numpy(np.ascontiguousarray(v[kind])) for k, v in kw.items()})
    same_rows(large, small, kind)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("temp", [1.0, 2.0, 1.5])
@pytest.mark.parametrize("width,k", [(4099, 8), (32768, 100), (50001, 200)])
def test_distillation_gradient(width, k, temp, dt):
    rng = np.random.default_rng(width + k)
    z, index, teacher, label = inputs(rng, KINDS, width, k, dt, "f32")
    index[1], label[2], index[3], label[3] = index[1, 0], -100, -1, -100
    dl = R.rounded(rng.uniform(0.5, 1.5, KINDS), "f32")
    _, sums, small = check_distilled(z, index, teacher, label, dt, "f32", temp, 0.5, dl=dl)
    kind = copies(rows_for(width, dt), width, dt)
    large = ms.distill_loss_grad(ms.from_numpy(dl.astype(np.float32)[kind]), ms.embedding(R.to_device(z, dt), R.ids(kind)),
                                 ms.from_numpy(sums.numpy()[kind]), R.ids(index[kind]), R.to_device(teacher[kind], "f32"),
                                 R.ids(label[kind]), temperature=temp, weight=0.5)
    same_rows(large, small, kind)


@pytest.mark.parametrize("dt,to", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("n", [400, 6000])
def test_embedding_gradient(n, dt, to):
    rng = np.random.default_rng(n)
    rows, width = 70001, 513 if BYTES[to] == 2 else 257
    assert rows * width * BYTES[to] >= 64 << 20
    check_embedding_grad(whole(rng, (n, width)), rng.integers(-1, rows, n), rows, dt, to)
