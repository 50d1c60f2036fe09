"""The embedding's gradient for batches of very many tokens and tables of very many rows: orders in two to four passes, of several
tiles and several steps of one, chunks longer than the 64 tokens that a wave holds at once, tables that many launches clear.

dy holds whole numbers from -8 to 8, the scale is a power of two and a token's sum stays below 2^24 in size: every sum in 32 bits is exact
in any order, and results are compared for equality."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import vocab_reference as R

pytestmark = pytest.mark.gpu


def whole(rng, shape):
    return rng.integers(-8, 9, shape).astype(np.float64)


def mixed(rng, n, rows, main):
    """A third of one token, the others all over, some of them outside the table."""
    t = rng.integers(-1, rows + 2, n)
    t[rng.random(n) < 1 / 3] = main
    return t


def expected(dy, tokens, scale):
    """(rows that occur, ascending; their sums)"""
    found, at = np.unique(tokens, return_inverse=True)
    sums = np.zeros((len(found), dy.shape[1]))
    np.add.at(sums, at, dy)
    return found, sums * scale


def check(dy, tokens, rows, dt, to, id_dt="i64", old=None):
    """Into an array of 7, with a row of it in front and one behind, or added to `old`."""
    scale, width = 0.5, dy.shape[1]
    found, sums = expected(dy, tokens, scale)
    inside = (found >= 0) & (found < rows)
    found, sums = found[inside], sums[inside]
    array = np.full((rows + 2, width), 7.0)
    if old is not None:
        array[1:-1] = old
    around = R.to_device(array, to)
    part = around[1:rows + 1]
    got = ms.embedding_grad(R.to_device(dy, dt), R.ids(tokens, id_dt), rows, scale, accumulate=old is not None, out=part)
    assert got.data_ptr == part.data_ptr
    v = R.values(around)
    assert (v[[0, -1]] == 7).all()
    v = v[1:-1]
    want = sums if old is None else old[found] + sums
    assert np.array_equal(v[found], want if to == "f32" else R.rounded(want, to))
    still = np.ones(rows, bool)
    still[found] = False
    assert np.array_equal(v[still], np.zeros((still.sum(), width)) if old is None else old[still])


@pytest.mark.parametrize("n", [32769, 40001, 131072, 131136, 131137, 200000, 262145])
@pytest.mark.parametrize("rows,width,dt,to", [(300, 9, "f32", "f32"), (70000, 3, "bf16", "f32"), (300001, 4, "f32", "f32"),
                                              (262143, 8, "bf16", "bf16"), (262144, 8, "f16", "f32")])
def test_passes_and_chunks(n, rows, width, dt, to):
    """Numbers of up to 9, 18 and 27 bits, in one to three passes (a number outside takes the table's size itself, a bit more at
    a power of two); chunks of 16 to 256 tokens."""
    rng = np.random.default_rng(n + rows)
    check(whole(rng, (n, width)), mixed(rng, n, rows, rows - 1), rows, dt, to, "i32" if n % 2 else "i64")


@pytest.mark.parametrize("n", [33000, 200000])
def test_four_passes(n):
    """28 bits; a table of one column, half a gigabyte, compared where tokens are and counted elsewhere."""
    rng = np.random.default_rng(n)
    rows = (1 << 27) + 3
    tokens = mixed(rng, n, rows, 12345678)
    tokens[:40] = np.repeat([0, 1, rows - 1, rows, (1 << 27) - 1], 8)
    dy = rng.integers(1, 9, (n, 1)).astype(np.float64)
    got = ms.embedding_grad(R.to_device(dy, "f32"), R.ids(tokens, "i32"), rows, 0.5).numpy()[:, 0]
    found, sums = expected(dy, tokens, 0.5)
    inside = (found >= 0) & (found < rows)
    assert np.array_equal(got[found[inside]], sums[inside, 0])
    assert np.count_nonzero(got) == inside.sum()  # (all sums are above 0)


@pytest.mark.parametrize("rows,width", [(300001, 64), (300001, 257), (511, 9000)])
def test_tables_that_several_launches_clear(rows, width):
    """Shares of some MB and of the most that a launch clears; rows of the table that begin between multiples of 16 bytes."""
    rng = np.random.default_rng(width)
    n = 40001 if width < 1000 else 32800
    some = rng.permutation(rows)[:3000]
    tokens = some[rng.integers(0, len(some), n)]
    dy = whole(rng, (n, width))
    found, sums = expected(dy, tokens, 0.5)
    around = ms.embedding(R.to_device(np.full((1, width), 7.0), "f32"), R.ids(np.zeros(rows + 2, np.int64)))
    part = around[1:rows + 1]
    ms.embedding_grad(R.to_device(dy, "f32"), R.ids(tokens), rows, 0.5, out=part)
    assert np.array_equal(ms.embedding(part, R.ids(found)).numpy(), sums.astype(np.float32))
    assert (ms.contiguous(around[0]).numpy() == 7).all() and (ms.contiguous(around[rows + 1]).numpy() == 7).all()
    others = np.ones(rows, bool)
    others[found] = False
    at = np.flatnonzero(others)
    for i in range(0, len(at), 40000):
        rest = ms.embedding(part, R.ids(at[i:i + 40000]))
        assert ms.max(ms.abs(rest)).numpy() == 0


@pytest.mark.parametrize("n", [524288, 524289, 700001, 1200000])
@pytest.mark.parametrize("rows,width", [(90, 3), (262200, 2)])
def test_several_steps_of_a_tile(n, rows, width):
    rng = np.random.default_rng(n + rows)
    check(whole(rng, (n, width)), mixed(rng, n, rows, 17), rows, "f32", "f32", "i32")


@pytest.mark.parametrize("dt,to", [("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("n,width", [(40001, 13), (131137, 13), (262145, 4), (600000, 3)])
@pytest.mark.parametrize("rows", [100, 262145])
def test_added(rows, n, width, dt, to):
    rng = np.random.default_rng(n)
    check(whole(rng, (n, width)), mixed(rng, n, rows, 40), rows, dt, to, old=whole(rng, (rows, width)))


@pytest.mark.parametrize("token", [0, 77, 99, -1, 100])
@pytest.mark.parametrize("n", [131137, 600000])
def test_one_token(n, token):
    rng = np.random.default_rng(n)
    check(whole(rng, (n, 5)), np.full(n, token), 100, "f32", "f32")


def test_the_same_from_call_to_call():
    """Sums that do round: the same bits, and places in order among equals."""
    rng = np.random.default_rng(7)
    dy, tokens = R.to_device(rng.standard_normal((600000, 5)), "f32"), R.ids((300000 ** rng.random(600000)).astype(np.int64))
    first = ms.embedding_grad(dy, tokens, 300001).numpy()
    for _ in range(3):
        assert np.array_equal(ms.embedding_grad(dy, tokens, 300001).numpy(), first)
