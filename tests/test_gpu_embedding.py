"""Embedding and its gradient against 64-bit forms."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import vocab_reference as R

pytestmark = pytest.mark.gpu


def look_up(table, tokens, scale, dt, to, id_dt, **kw):
    got = ms.embedding(R.to_device(table, dt), R.ids(tokens, id_dt), scale, dtype=to, **kw)
    assert got.shape == tokens.shape + table.shape[1:] and got.dtype == to
    # A product of a 24-bit and a 24-bit number is exact in 64 bits.  It is rounded to f32 (U of itself) and then to the result's
    # type, or at once: the hardware's multiply-add of f16 and f32 does the latter, and a tie of the first way is none then.
    want = R.embedding(table, tokens, float(np.float32(scale)))
    R.within(got, want, R.U * np.abs(want), to)


@pytest.mark.parametrize("dt,to", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "f32"),
                                   ("f16", "f16"), ("f16", "bf16"), ("bf16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("width", [1, 3, 4, 7, 8, 9, 64, 1111])
def test_embedding(dt, to, width):
    rng = np.random.default_rng(width)
    table = R.draw(rng, (50, width), dt)
    for n, id_dt in ((1, "i32"), (37, "i64")):
        look_up(table, rng.integers(-3, 53, n), 1.7, dt, to, id_dt)


@pytest.mark.parametrize("shape", [(), (0,), (2, 3, 5), (1000, 2)])
def test_embedding_shapes(shape):
    rng = np.random.default_rng(1)
    look_up(R.draw(rng, (9, 40), "bf16"), rng.integers(-1, 9, shape), 1.0, "bf16", "bf16", "i32")


def test_embedding_far_numbers():
    """Numbers whose low 32 bits name a row, and the lowest and highest ones."""
    table = R.draw(np.random.default_rng(2), (5, 16), "f32")
    far = np.array([0, 1 << 32, (1 << 32) + 3, -(1 << 32) + 1, -1, 4, 5, (1 << 63) - 1, -(1 << 63)], dtype=np.int64)
    look_up(table, far, 2.0, "f32", "f32", "i64")
    look_up(table, np.array([-(1 << 31), (1 << 31) - 1, 4], dtype=np.int32), 2.0, "f32", "f32", "i32")


def test_embedding_infinities_and_padding():
    table = np.array([[np.inf, -np.inf, np.nan, 1.0]] * 2)
    got = ms.embedding(R.to_device(table, "f32"), R.ids([0, 7, -1]), 0.0).numpy()
    assert np.isnan(got[0, :3]).all() and got[0, 3] == 0
    assert not got[1:].any() and np.isfinite(got[1:]).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_embedding_of_views(dt):
    rng = np.random.default_rng(3)
    table, tokens = R.draw(rng, (60, 70), dt), rng.integers(0, 30, (4, 6))
    t, k = R.to_device(table, dt), R.ids(tokens)
    want = lambda tab, tok: R.embedding(tab, tok, 1.0)
    assert np.array_equal(R.values(ms.embedding(ms.transpose(t), k)), want(table.T, tokens))
    assert np.array_equal(R.values(ms.embedding(t[10:50:1, 3:36], k)), want(table[10:50, 3:36], tokens))
    assert np.array_equal(R.values(ms.embedding(t[::2, ::3], k)), want(table[::2, ::3], tokens))
    assert np.array_equal(R.values(ms.embedding(ms.flip(t, 0), k)), want(table[::-1], tokens))
    assert np.array_equal(R.values(ms.embedding(ms.flip(t, 1)[:, 68:], k)), want(table[:, ::-1][:, 68:], tokens))
    assert np.array_equal(R.values(ms.embedding(t, ms.transpose(k))), want(table, tokens.T))
    assert np.array_equal(R.values(ms.embedding(t, k[1:3, ::2])), want(table, tokens[1:3, ::2]))


# ---- gradient ------------------------------------------------------------------------------------------
def grad(dy, tokens, rows, scale, dt, to, id_dt="i64", device=None):
    got = ms.embedding_grad(device or R.to_device(dy, dt), R.ids(tokens, id_dt), rows, scale, dtype=to)
    assert got.shape == (rows, dy.shape[-1]) and got.dtype == to
    want, bound = R.embedding_grad(dy, tokens, rows, scale)
    R.within(got, want, bound, to, f"{dy.shape} {rows} {dt} {to}")
    return got


@pytest.mark.parametrize("dt,to", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"),
                                   ("f32", "bf16"), ("f32", "f16"), ("bf16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("width", [1, 3, 4, 7, 8, 9, 64, 257, 1111])
def test_gradient(dt, to, width):
    rng = np.random.default_rng(width)
    for n, rows in ((1, 3), (33, 100), (200, 7)):
        grad(R.draw(rng, (n, width), dt), rng.integers(-2, rows + 2, n), rows, 1.7, dt, to, "i32" if n > 1 else "i64")


@pytest.mark.parametrize("n", [0, 1, 2, 31, 32, 33, 63, 64, 65, 1024, 1025, 2049, 5000, 8193, 16384, 16385, 24001, 32768, 32769, 40001])
@pytest.mark.parametrize("rows", [1, 2, 511, 512, 70000])
def test_gradient_numbers_of_tokens(n, rows):
    """Orders by rank and in one and two passes; runs within a chunk, over its end, over many chunks."""
    rng = np.random.default_rng(n + rows)
    tokens = (rows ** rng.random(n)).astype(np.int64) - rng.integers(0, 2, n)
    grad(R.draw(rng, (n, 9), "f32"), tokens, rows, 0.5, "f32", "f32")


@pytest.mark.parametrize("n,rows,width", [(255, 300, 40), (256, 300, 40), (257, 300, 40), (64, 20, 2100), (65, 20, 2100), (64, 8200, 1030),
                                          (200, 8200, 1030), (200, 5, 4), (4095, 50, 24), (4096, 5000, 24), (4097, 50, 24), (5120, 5000, 24), (5121, 50, 24)])
@pytest.mark.parametrize("dt,to", [("bf16", "f32"), ("f32", "bf16"), ("f32", "f32"), ("f16", "f16")])
def test_gradient_from_way_to_way(n, rows, width, dt, to):
    """At the numbers of tokens, and the sizes of a table, where one way ends and the next begins."""
    rng = np.random.default_rng(n + width)
    tokens = (rows ** rng.random(n)).astype(np.int64) - rng.integers(0, 2, n)
    grad(R.draw(rng, (n, width), dt), tokens, rows, 0.5, dt, to, "i32" if n < 4096 or n > 5000 else "i64")


@pytest.mark.parametrize("to", ["f32", "bf16"])
@pytest.mark.parametrize("width", [4, 8, 9, 13, 64, 255, 1001])
@pytest.mark.parametrize("n", [0, 1, 30, 150, 600])
def test_gradient_into_part_of_an_array(n, width, to):
    """Rows that begin and end between two multiples of 16 bytes, with other rows around them."""
    rng = np.random.default_rng(n + width)
    dy = R.draw(rng, (n, width), "f32")
    for before in (1, 2, 3):
        rows = 41
        tokens = np.sort((rows ** rng.random(n)).astype(np.int64) - 1)[::-1].copy()
        whole = R.to_device(np.full((before + rows + 2, width), 7.0), to)
        part = whole[before:before + rows]
        got = ms.embedding_grad(R.to_device(dy, "f32"), R.ids(tokens), rows, 1.0, out=part)
        want, bound = R.embedding_grad(dy, tokens, rows, 1.0)
        R.within(got, want, bound, to)
        v = R.values(whole)
        assert (v[:before] == 7).all() and (v[before + rows:] == 7).all()


def test_gradient_three_passes():
    rng = np.random.default_rng(5)
    grad(R.draw(rng, (20000, 4), "bf16"), rng.integers(0, 300001, 20000), 300001, 1.0, "bf16", "bf16")


@pytest.mark.parametrize("n", [1000, 30000])
@pytest.mark.parametrize("token", [0, 77, 99, -1, 100])
def test_gradient_of_one_token(n, token):
    rng = np.random.default_rng(6)
    grad(R.draw(rng, (n, 20), "f32"), np.full(n, token), 100, 1.0, "f32", "f32")


def test_gradient_is_the_same_from_call_to_call():
    rng = np.random.default_rng(7)
    dy = R.to_device(rng.standard_normal((30000, 65)), "f32")
    tokens = R.ids((500 ** rng.random(30000)).astype(np.int64))
    first = ms.embedding_grad(dy, tokens, 600).numpy()
    for _ in range(3):
        assert np.array_equal(ms.embedding_grad(dy, tokens, 600).numpy(), first)


@pytest.mark.parametrize("dt,to", [("bf16", "f32"), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("width", [3, 64, 101])
@pytest.mark.parametrize("n", [0, 40, 300, 6000, 20000])
def test_gradient_added(dt, to, width, n):
    rng = np.random.default_rng(8)
    rows = 90
    dy, tokens, old = R.draw(rng, (n, width), dt), rng.integers(-1, rows // 2, n), R.draw(rng, (rows, width), to)
    out = R.to_device(old, to)
    got = ms.embedding_grad(R.to_device(dy, dt), R.ids(tokens), rows, 0.5, accumulate=True, out=out)
    assert got.data_ptr == out.data_ptr
    sums, bound = R.embedding_grad(dy, tokens, rows, 0.5)
    R.within(got, old + sums, bound + 2 * R.U * (np.abs(old) + np.abs(sums)), to)
    still = ~np.isin(np.arange(rows), tokens)
    assert np.array_equal(R.values(got)[still], old[still])


def test_gradient_of_views_and_shapes():
    rng = np.random.default_rng(9)
    dy, tokens = R.draw(rng, (6, 10, 48), "bf16"), rng.integers(-1, 20, (6, 10))
    d, k = R.to_device(dy, "bf16"), R.ids(tokens)

    def check(got, dy, tokens):
        want, bound = R.embedding_grad(dy, tokens, 20, 1.0)
        R.within(got, want, bound, "bf16")

    check(ms.embedding_grad(d, k, 20), dy, tokens)
    check(ms.embedding_grad(d[:, :, 5:30], k, 20), dy[:, :, 5:30], tokens)
    check(ms.embedding_grad(d[1:4, ::3, ::2], k[1:4, ::3], 20), dy[1:4, ::3, ::2], tokens[1:4, ::3])
    check(ms.embedding_grad(ms.transpose(d, [1, 0, 2]), ms.transpose(k), 20), dy.transpose(1, 0, 2), tokens.T)
    check(ms.embedding_grad(ms.flip(d, 0), k, 20), dy[::-1], tokens)
    check(ms.embedding_grad(d[0, 0], k[0, 0], 20), dy[0, 0], tokens[0, 0])  # one token, no axis


def test_gradient_of_infinities():
    """A NaN or an infinity reaches the rows of its own token and no others."""
    dy = np.ones((100, 12))
    dy[40, 3], dy[41, 5] = np.inf, np.nan
    tokens = np.arange(100) % 50
    tokens[60] = -1
    dy[60] = np.nan
    got = ms.embedding_grad(R.to_device(dy, "f32"), R.ids(tokens), 60).numpy()
    want = np.zeros((60, 12))
    np.add.at(want, tokens[tokens >= 0], dy[tokens >= 0])
    assert np.array_equal(got, want, equal_nan=True)


def test_offsets_past_32_bits():
    """Rows of a table, of a batch and of a gradient that lie past 2^32 elements: 2 x 8 GiB of bf16."""
    rows, width = 131073, 32776
    out = ms.embedding_grad(R.to_device(np.ones((3, width)), "bf16"), R.ids([rows - 1, 5, rows - 1]), rows)
    assert R.values(out[rows - 1]).tolist() == [2.0] * width and R.values(out[5]).tolist() == [1.0] * width
    assert not R.values(out[rows - 2]).any() and not R.values(out[6]).any()
    got = ms.embedding(out, R.ids([rows - 1, 0, 5, rows]), 3.0)
    assert np.array_equal(R.values(got), np.repeat([[6.0], [0.0], [3.0], [0.0]], width, 1))


def test_offsets_near_31_bits():
    """Few tokens and a gradient of just below 2^31 values: 8 GiB of f32, begun 8 bytes off."""
    rows, width = 65524, 32774
    assert rows * width < 1 << 31 < (rows + 1) * width
    whole = ms.embedding(R.to_device(np.ones((1, width)), "f32"), R.ids(np.zeros(rows + 1)))
    out = whole[1:]
    ms.embedding_grad(R.to_device(np.ones((3, width)), "f32"), R.ids([rows - 1, 5, rows - 1]), rows, out=out)
    assert R.values(out[rows - 1]).tolist() == [2.0] * width and R.values(out[5]).tolist() == [1.0] * width
    assert not R.values(out[rows - 2]).any() and not R.values(out[6]).any() and not R.values(out[0]).any()
    assert R.values(whole[0]).tolist() == [1.0] * width
    assert R.values(ms.max(out[6:rows - 1])) == 0.0


def test_refusals():
    t, k = ms.from_numpy(np.ones((4, 8), np.float32)), R.ids([0, 1])
    d = ms.from_numpy(np.ones((2, 8), np.float32))
    with pytest.raises(ms.DtypeError):
        ms.embedding(ms.from_numpy(np.ones((4, 8))), k)
    with pytest.raises(ms.DtypeError):
        ms.embedding(t, ms.from_numpy(np.zeros(2, np.int16)))
    with pytest.raises(ms.DtypeError):
        ms.embedding(t, k, dtype="f64")
    with pytest.raises(ms.ShapeError):
        ms.embedding(t[0], k)
    with pytest.raises(ms.ShapeError):
        ms.embedding(t[4:], k)
    with pytest.raises(ms.ShapeError):
        ms.embedding(t, k, out=ms.from_numpy(np.ones((2, 7), np.float32)))
    with pytest.raises(ms.DtypeError):
        ms.embedding(t, k, dtype="bf16", out=ms.from_numpy(np.ones((2, 8), np.float32)))
    with pytest.raises(ms.MemoryError):
        ms.embedding(t, k, out=t[:2])
    with pytest.raises(ValueError):
        ms.embedding(t, k, float("nan"))
    with pytest.raises(ms.ShapeError):
        ms.embedding_grad(d, R.ids([0, 1, 2]), 4)
    with pytest.raises(ms.ShapeError):
        ms.embedding_grad(d, k, 4, out=ms.from_numpy(np.ones((5, 8), np.float32)))
    with pytest.raises(ValueError):
        ms.embedding_grad(d, k, 4, accumulate=True)
    with pytest.raises(ms.DtypeError):
        ms.embedding_grad(d, ms.from_numpy(np.zeros(2, np.float32)), 4)
    with pytest.raises(TypeError):
        ms.embedding_grad(d, k, -1)
