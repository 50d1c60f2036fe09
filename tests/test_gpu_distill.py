"""The distillation loss and its gradient against 64-bit forms, row by row."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import vocab_reference as R

pytestmark = pytest.mark.gpu


def inputs(rng, rows, width, k, dt, tdt, labelled=True, spread=2.0):
    z = R.draw(rng, (rows, width), dt, spread)
    index = np.stack([rng.permutation(width)[:k] if k <= width else rng.integers(0, width, k) for _ in range(rows)]) if k else \
        np.zeros((rows, 0), np.int64)
    teacher = R.draw(rng, (rows, k), tdt, 2.0)
    label = rng.integers(0, width, rows) if labelled else None
    return z, index, teacher, label


def check(z, index, teacher, label, dt, tdt, temp=1.0, weight=1.0, id_dt="i64", dl=None, arrays=None):
    """Loss and gradient of 2-D logits."""
    Z, I, T = arrays or (R.to_device(z, dt), R.ids(index, id_dt), R.to_device(teacher, tdt))
    L = None if label is None else R.ids(label, id_dt)
    rows = len(z)
    loss, sums = ms.distill_loss(Z, I, T, L, temperature=temp, weight=weight)
    assert loss.shape == (rows,) and sums.shape == (rows, 3) and loss.dtype == sums.dtype == "f32"
    label = [None] * rows if label is None else label
    with np.errstate(all="ignore"):
        want = np.array([R.distill(z[r], index[r], teacher[r], label[r], temp, weight) for r in range(rows)]).reshape(rows, 4)
        bound = np.array([R.distill_bound(z[r], index[r], teacher[r], label[r], temp, weight) for r in range(rows)]).reshape(rows, 4)
    got = sums.numpy()
    R.within(loss, want[:, 0], bound[:, 0], "f32", "loss")
    # What a row has no use for is 0 exactly.  A logarithm that is 0 (one column that counts) is formed of a sum off by a
    # rounding, as any other, and of the rounding of m c: its bound is log_sum_bound too.
    used = np.array([R.uses(z[r], R.entries(index[r], teacher[r], z.shape[1], temp)[0], label[r], weight) for r in range(rows)])
    used = np.concatenate([used.reshape(rows, 2).any(1)[:, None], used.reshape(rows, 2)], 1)
    for j in (0, 1, 2):
        R.within(got[:, j].astype(np.float64), want[:, 1 + j], np.where(used[:, j], bound[:, 1 + j], 0), "f32", f"sums {j}")
    dl = np.linspace(0.5, 1.5, rows) if dl is None else dl
    dl = R.rounded(dl, "f32")
    g = ms.distill_loss_grad(R.to_device(dl, "f32"), Z, sums, I, T, L, temperature=temp, weight=weight)
    assert g.shape == z.shape and g.dtype == dt
    with np.errstate(all="ignore"):
        gw = np.stack([R.distill_grad(dl[r], z[r], got[r].astype(np.float64), index[r], teacher[r], label[r], temp, weight)
                       for r in range(rows)])
        gb = np.stack([R.distill_grad_bound(dl[r], z[r], got[r].astype(np.float64), index[r], teacher[r], label[r], temp, weight)
                       for r in range(rows)])
    R.within(g, gw, gb, dt, "gradient")
    return loss, sums, g


@pytest.mark.parametrize("dt,tdt", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("temp,weight", [(1.0, 1.0), (2.0, 0.5), (1.0, 0.3), (0.5, 0.0), (3.0, 1.0)])
def test_types_and_factors(dt, tdt, temp, weight):
    rng = np.random.default_rng(1)
    check(*inputs(rng, 5, 1003, 12, dt, tdt), dt, tdt, temp, weight, "i32")
    check(*inputs(rng, 3, 640, 7, dt, tdt, labelled=False), dt, tdt, temp, weight)


@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 7, 8, 9, 255, 2048, 2049, 4095, 4096, 16384, 16385, 50001])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_widths(width, dt):
    rng = np.random.default_rng(width)
    check(*inputs(rng, 3, width, min(width, 6), dt, "f32"), dt, "f32", 2.0, 0.5)


@pytest.mark.parametrize("k", [0, 1, 2, 63, 64, 65, 200, 1024])
def test_numbers_of_entries(k):
    rng = np.random.default_rng(k)
    check(*inputs(rng, 3, 5000, k, "f32", "f32"), "f32", "f32", 2.0, 0.5)
    check(*inputs(rng, 2, 5000, k, "bf16", "bf16", labelled=False), "bf16", "bf16")


@pytest.mark.parametrize("k", [2, 40, 130, 300])
@pytest.mark.parametrize("dt,width", [("bf16", 4001), ("f32", 4001), ("f16", 2100), ("bf16", 9), ("f32", 5)])
def test_columns_that_several_entries_name(k, dt, width):
    """A few columns in all entries, the first and last of the row among them, and the label one of them."""
    rng = np.random.default_rng(k + width)
    rows = 9
    z, _, teacher, label = inputs(rng, rows, width, k, dt, "f32")
    few = np.stack([rng.choice(np.r_[0, 1, 2, width - 3, width - 2, width - 1, rng.integers(0, width, 20)], 6) for _ in range(rows)])
    index = np.take_along_axis(few, rng.integers(0, 6, (rows, k)), 1)
    index[4] = rng.permutation(max(width, k))[:k]  # a row without any, or with some past the width
    label[::2] = index[::2, 0] % width
    check(z, index, teacher, label, dt, "f32", 1.5, 0.6)


@pytest.mark.parametrize("rows", [1, 2, 600, 2100])
def test_numbers_of_rows(rows):
    rng = np.random.default_rng(rows)
    check(*inputs(rng, rows, 777, 5, "bf16", "f32"), "bf16", "f32", 1.5, 0.5)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width", [(2047, 300), (2048, 1), (2048, 9), (2049, 300), (2049, 4003), (2048, 8197), (2048, 33000), (8192, 12001)])
def test_many_rows(rows, width, dt):
    """Rows of five kinds, by a wave, four and eight each."""
    rng = np.random.default_rng(rows + width)
    k = min(width, 70)
    z, index, teacher, label = inputs(rng, 5, width, k, dt, "f32")
    label[1], index[2] = -100, -1
    kind = rng.integers(0, 5, rows)
    loss, sums = ms.distill_loss(ms.embedding(R.to_device(z, dt), R.ids(kind)), R.ids(index[kind]), R.to_device(teacher[kind], "f32"),
                                 R.ids(label[kind]), temperature=1.5, weight=0.5)
    want = np.array([R.distill(z[r], index[r], teacher[r], label[r], 1.5, 0.5) for r in range(5)])
    bound = np.array([R.distill_bound(z[r], index[r], teacher[r], label[r], 1.5, 0.5) for r in range(5)])
    R.within(loss, want[kind, 0], bound[kind, 0], "f32", "loss")
    for j in (0, 1, 2):
        R.within(sums.numpy()[:, j].astype(np.float64), want[kind, 1 + j], bound[kind, 1 + j], "f32", f"sums {j}")


def test_no_rows():
    z = ms.from_numpy(np.zeros((0, 10), np.float32))
    i, t = ms.from_numpy(np.zeros((0, 2), np.int64)), ms.from_numpy(np.zeros((0, 2), np.float32))
    loss, sums = ms.distill_loss(z, i, t)
    assert loss.shape == (0,) and sums.shape == (0, 3)
    assert ms.distill_loss_grad(loss, z, sums, i, t).shape == (0, 10)


def test_entries_that_do_not_count():
    """Padding, columns outside, values of -inf, the same index several times, rows of none; labels outside."""
    rng = np.random.default_rng(2)
    z, index, teacher, label = inputs(rng, 8, 300, 6, "f32", "f32")
    index[0, 2:] = -1
    index[1] = -1
    index[2] = [5, 5, 5, 9, 9, label[2]]
    index[3] = [300, 1 << 40, -(1 << 40), (1 << 32) + 1, 4, 4]
    teacher[4, :3] = -np.inf
    teacher[5] = -np.inf
    index[6], label[6] = -1, -100
    label[7] = 300
    for weight, temp in ((0.5, 2.0), (1.0, 1.0), (0.0, 1.0)):
        _, sums, g = check(z, index, teacher, label, "f32", "f32", temp, weight)
        assert not sums.numpy()[6].any() and not g.numpy()[6].any()
    _, sums, g = check(z, index, teacher, None, "f32", "f32", 2.0, 1.0)
    assert not g.numpy()[[1, 5, 6]].any()


def test_rows_without_a_use_are_not_read():
    z = np.full((2, 500), np.nan)
    for dt in ("f32", "bf16"):
        loss, sums, g = check(z, np.full((2, 3), -1), np.ones((2, 3)), np.array([-1, 500]), dt, "f32", 1.0, 0.5)
        assert not loss.numpy().any() and not sums.numpy().any() and not R.values(g).any()


def test_masked_columns():
    """Columns of -inf and of the types' lowest values; whole threads' and whole rows' worth of them."""
    rng = np.random.default_rng(3)
    for dt, low in (("f32", -np.finfo(np.float32).max), ("bf16", -float.fromhex("0x1.fep127")), ("f16", -65504.0)):
        for width in (40, 9000):
            z, index, teacher, label = inputs(rng, 6, width, 3, dt, "f32")
            z[0, rng.random(width) < 0.9] = -np.inf
            z[1, rng.random(width) < 0.9] = low
            z[2, 1:] = -np.inf
            z[3, 1:] = low
            z[4] = low                       # all alike: uniform
            z[5, : width // 2] = -np.inf
            index[:, 0], label[:] = 0, 0
            index[2:4] = [[0, -1, -1]] * 2   # what is not masked there
            z[0, index[0]], z[1, index[1]], z[5, index[5]] = 1.0, 2.0, 0.5
            check(z, index, teacher, label, dt, "f32", 1.0, 0.5)
            if dt != "f16":
                check(z, index, teacher, label, dt, "f32", 2.0, 1.0)


def test_a_teacher_on_a_masked_column():
    """p > 0 where q = 0: an infinite loss, a gradient that is not."""
    z = np.array([[-np.inf, 1.0, 2.0, 3.0]])
    loss, _, g = check(z, np.array([[0, 1]]), np.array([[1.0, 1.0]]), None, "f32", "f32")
    assert loss.numpy()[0] == np.inf and np.isfinite(g.numpy()).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_infinities_and_nan(bad):
    rng = np.random.default_rng(4)
    z, index, teacher, label = inputs(rng, 4, 3000, 4, "f32", "f32")
    z[1, 2999] = bad
    teacher[2, 1] = bad
    Z, I, T, L = R.to_device(z, "f32"), R.ids(index), R.to_device(teacher, "f32"), R.ids(label)
    loss, sums = ms.distill_loss(Z, I, T, L, temperature=2.0, weight=0.5)
    g = ms.distill_loss_grad(R.to_device(np.ones(4), "f32"), Z, sums, I, T, L, temperature=2.0, weight=0.5).numpy()
    assert np.isnan(loss.numpy()).tolist() == [False, True, True, False]
    assert np.isfinite(g[[0, 3]]).all() and np.isnan(g[1]).all()
    assert np.isnan(g[2, index[2]]).all()
    # the other rows do not feel it
    z[1], teacher[2] = 0.0, 0.0
    clean, _ = ms.distill_loss(R.to_device(z, "f32"), I, R.to_device(teacher, "f32"), L, temperature=2.0, weight=0.5)
    assert np.array_equal(clean.numpy()[[0, 3]], loss.numpy()[[0, 3]])


@pytest.mark.parametrize("temp", [2.0 ** -20, 2.0 ** 20, 0.01, 100.0])
def test_far_temperatures(temp):
    rng = np.random.default_rng(5)
    z, index, teacher, label = inputs(rng, 3, 2000, 5, "f32", "f32")
    check(z, index, teacher, label, "f32", "f32", temp, 0.5)


def test_large_logits():
    rng = np.random.default_rng(6)
    z, index, teacher, label = inputs(rng, 3, 5000, 5, "f32", "f32", spread=1000.0)
    check(R.rounded(z + 1e4, "f32"), index, teacher, label, "f32", "f32", 1.0, 0.5)


def test_views_and_shapes():
    rng = np.random.default_rng(7)
    z, index, teacher, label = inputs(rng, 12, 200, 5, "bf16", "f32")
    Z, I, T = R.to_device(z, "bf16"), R.ids(index), R.to_device(teacher, "f32")
    check(z[:, 3:180], index, teacher, None, "bf16", "f32", arrays=(Z[:, 3:180], I, T))
    check(z[::2], index[::2], teacher[::2], None, "bf16", "f32", arrays=(Z[::2], I[::2], T[::2]))
    check(z[:, ::3], index[:, ::2], teacher[:, ::2], None, "bf16", "f32", arrays=(Z[:, ::3], I[:, ::2], T[:, ::2]))
    check(z[::-1], index[::-1], teacher, None, "bf16", "f32", arrays=(ms.flip(Z, 0), ms.flip(I, 0), T))
    # (3, 4, columns), one number for all rows' dloss, and one row without an axis
    cube = lambda a: ms.from_numpy(a.reshape((3, 4) + a.shape[1:]))
    z32 = z.astype(np.float32)
    loss, sums = ms.distill_loss(cube(z32), cube(index), cube(teacher.astype(np.float32)), cube(label), weight=0.5)
    flat, fsums = ms.distill_loss(ms.from_numpy(z32), I, T, R.ids(label), weight=0.5)
    assert loss.shape == (3, 4) and sums.shape == (3, 4, 3)
    assert np.array_equal(loss.numpy().ravel(), flat.numpy())
    whole = ms.distill_loss_grad(ms.from_numpy(np.float32(0.25)), ms.from_numpy(z32), fsums, I, T, R.ids(label), weight=0.5)
    each = ms.distill_loss_grad(ms.from_numpy(np.full((3, 4), 0.25, np.float32)), cube(z32), sums, cube(index),
                                cube(teacher.astype(np.float32)), cube(label), weight=0.5)
    assert each.shape == (3, 4, 200) and np.array_equal(each.numpy().reshape(12, 200), whole.numpy())
    one, osums = ms.distill_loss(ms.from_numpy(z32)[3], I[3], T[3], R.ids(label)[3], weight=0.5)
    assert one.shape == () and osums.shape == (3,) and one.numpy() == flat.numpy()[3]
    two = ms.from_numpy(np.repeat(np.linspace(1, 2, 12, dtype=np.float32), 2))[::2]
    got = ms.distill_loss_grad(two, ms.from_numpy(z32), fsums, I, T, R.ids(label), weight=0.5).numpy()
    plain = ms.distill_loss_grad(ms.contiguous(two), ms.from_numpy(z32), fsums, I, T, R.ids(label), weight=0.5).numpy()
    assert np.array_equal(got, plain)


def test_the_same_from_call_to_call():
    rng = np.random.default_rng(8)
    z, index, teacher, label = inputs(rng, 9, 30000, 100, "bf16", "f32")
    index[:, :50] = 7  # many entries of one column
    a = [R.to_device(z, "bf16"), R.ids(index), R.to_device(teacher, "f32"), R.ids(label)]
    one = ms.from_numpy(np.float32(1.0))
    first = None
    for _ in range(3):
        loss, sums = ms.distill_loss(*a, temperature=2.0, weight=0.5)
        g = ms.distill_loss_grad(one, a[0], sums, *a[1:], temperature=2.0, weight=0.5)
        now = (loss.numpy().tobytes(), sums.numpy().tobytes(), g.numpy().tobytes())
        assert first in (None, now)
        first = now


def test_the_gradient_against_differences():
    """The loss's slope along a direction, by a central difference in f32: the difference's own error is the third derivative's
    and the losses' rounding, 2^-22 of some 5, over the step."""
    rng = np.random.default_rng(9)
    z, index, teacher, label = inputs(rng, 4, 500, 6, "f32", "f32")
    I, T, L = R.ids(index), R.to_device(teacher, "f32"), R.ids(label)
    kw = dict(temperature=2.0, weight=0.5)
    _, sums = ms.distill_loss(R.to_device(z, "f32"), I, T, L, **kw)
    g = ms.distill_loss_grad(ms.from_numpy(np.float32(1.0)), R.to_device(z, "f32"), sums, I, T, L, **kw).numpy().astype(np.float64)
    d = g / np.linalg.norm(g) + rng.standard_normal(g.shape) / np.sqrt(g.size)
    step = 0.02
    up, down = (ms.distill_loss(ms.from_numpy((z + s * step * d).astype(np.float32)), I, T, L, **kw)[0].numpy().astype(np.float64).sum()
                for s in (1, -1))
    assert abs((up - down) / (2 * step) - (g * d).sum()) < 1e-3


def test_refusals():
    z = ms.from_numpy(np.zeros((4, 9), np.float32))
    i, t, l = R.ids(np.zeros((4, 2), np.int64)), ms.from_numpy(np.zeros((4, 2), np.float32)), R.ids(np.zeros(4, np.int64))
    sums, dl = ms.from_numpy(np.zeros((4, 3), np.float32)), ms.from_numpy(np.ones(4, np.float32))
    many = ms.from_numpy(np.zeros((4, 1025), np.int64))
    for err, call in [
        (ms.DtypeError, lambda: ms.distill_loss(ms.from_numpy(np.zeros((4, 9))), i, t)),
        (ms.DtypeError, lambda: ms.distill_loss(z, t, t)),
        (ms.DtypeError, lambda: ms.distill_loss(z, i, i)),
        (ms.DtypeError, lambda: ms.distill_loss(z, i, t, dl)),
        (ms.ShapeError, lambda: ms.distill_loss(z, i[:3], t[:3])),
        (ms.ShapeError, lambda: ms.distill_loss(z, i, t[:, :1])),
        (ms.ShapeError, lambda: ms.distill_loss(z, i, t, l[:3])),
        (ms.ShapeError, lambda: ms.distill_loss(z, many, ms.from_numpy(np.zeros((4, 1025), np.float32)))),
        (ValueError, lambda: ms.distill_loss(z, i, t, temperature=0.0)),
        (ValueError, lambda: ms.distill_loss(z, i, t, temperature=float("nan"))),
        (ValueError, lambda: ms.distill_loss(z, i, t, temperature=2.0 ** 21)),
        (ValueError, lambda: ms.distill_loss(z, i, t, weight=1.5)),
        (ValueError, lambda: ms.distill_loss(z, i, t, weight=float("nan"))),
        (TypeError, lambda: ms.distill_loss(z, i, t, out=dl)),
        (ms.ShapeError, lambda: ms.distill_loss(z, i, t, out=(sums, None))),
        (ms.ShapeError, lambda: ms.distill_loss_grad(dl[:3], z, sums, i, t)),
        (ms.ShapeError, lambda: ms.distill_loss_grad(dl, z, dl, i, t)),
        (ms.DtypeError, lambda: ms.distill_loss_grad(ms.from_numpy(np.ones(4)), z, sums, i, t)),
        (ms.MemoryError, lambda: ms.distill_loss_grad(dl, z, sums, i, t, out=z)),
        (ms.DtypeError, lambda: ms.distill_loss_grad(dl, z, sums, i, t, out=ms.array(np.zeros((4, 9)), dtype="f16"))),
    ]:
        with pytest.raises(err):
            call()


@pytest.mark.parametrize("rows,width", [(1, 65536), (1, 131072), (2, 65600), (9, 70001), (9, 131072), (128, 65600), (129, 65600)])
def test_few_long_rows(rows, width):
    """Rows that are split into segments, among them ones without a use and segments of nothing but masked columns."""
    rng = np.random.default_rng(rows)
    few = min(rows, 9)
    for dt in ("bf16", "f32"):
        z, index, teacher, label = inputs(rng, few, width, 70, dt, "f32")
        z[few - 1, 1000:60000] = -np.inf
        if few > 1:
            index[0], label[0] = -1, -100
            z[1, :] = R.rounded(np.full(1, -3e38), dt)
            z[1, width - 1], index[1, :2], label[1] = 1.0, [width - 1, -1], width - 1
            index[1, 2:] = -1
        rep = np.arange(rows) % few
        check(z[rep], index[rep], teacher[rep], label[rep], dt, "f32", 2.0, 0.5)
        check(z[rep], index[rep], teacher[rep], None, dt, "f32", 1.0, 1.0)


def test_offsets_past_32_bits():
    """Logits, and a gradient, that lie past 2^32 elements: two of 8 GiB.  Every row has the bits of the row of its kind near
    the front: each is summed alike, as all begin on a multiple of 16 bytes."""
    rows, width, kinds = 65601, 65544, 3
    rng = np.random.default_rng(11)
    z, index, teacher, label = inputs(rng, kinds, width, 7, "bf16", "f32")
    kind = np.arange(rows) % kinds
    Z = ms.embedding(R.to_device(z, "bf16"), R.ids(kind))
    I, T, L = R.ids(index[kind]), R.to_device(teacher[kind], "f32"), R.ids(label[kind])
    dl = np.linspace(0.5, 1.5, kinds, dtype=np.float32)
    loss, sums = ms.distill_loss(Z, I, T, L, weight=0.5, temperature=2.0)
    grad = ms.distill_loss_grad(ms.from_numpy(dl[kind]), Z, sums, I, T, L, weight=0.5, temperature=2.0)
    assert np.array_equal(loss.numpy(), loss.numpy()[kind]) and np.array_equal(sums.numpy(), sums.numpy()[kind])
    top = np.array([R.distill(z[r], index[r], teacher[r], label[r], 2.0, 0.5) for r in range(kinds)])
    bound = np.array([R.distill_bound(z[r], index[r], teacher[r], label[r], 2.0, 0.5) for r in range(kinds)])
    R.within(loss[:kinds], top[:, 0], bound[:, 0], "f32", "loss")
    got = sums.numpy().astype(np.float64)
    want = [R.distill_grad(dl[r], z[r], got[r], index[r], teacher[r], label[r], 2.0, 0.5) for r in range(kinds)]
    room = [R.distill_grad_bound(dl[r], z[r], got[r], index[r], teacher[r], label[r], 2.0, 0.5) for r in range(kinds)]
    R.within(grad[:kinds], np.stack(want), np.stack(room), "bf16", "gradient")
    front = R.values(grad[:kinds])
    for r in (32767, 32768, 65527, 65528, 65529, rows - 2, rows - 1):
        assert np.array_equal(R.values(grad[r]), front[r % kinds]), r
    # the same rows apart by a stride: two that lie 2^32 elements from each other
    far = Z[::65529]
    assert np.array_equal(ms.distill_loss(far, I[::65529], T[::65529], L[::65529], weight=0.5, temperature=2.0)[0].numpy(),
                          loss.numpy()[[0, 65529]])
