"""The vocabulary's operators between streams: inputs that another stream has just written, outputs that another reads."""
import numpy as np
import pytest

import musapy_amd as ms
from tests import vocab_reference as R

pytestmark = pytest.mark.gpu


def test_a_chain_over_two_streams():
    rng = np.random.default_rng(1)
    rows, width = 300, 20000
    z = [rng.standard_normal((rows, width)).astype(np.float32) for _ in range(2)]
    index = rng.integers(0, width, (rows, 8))
    teacher = rng.standard_normal((rows, 8)).astype(np.float32)
    tokens = rng.integers(0, 50, 4000)
    one = ms.from_numpy(np.float32(1.0))

    def chain(x, a, b):
        """every step on another stream than the one in front of it"""
        with ms.stream(a):
            y = ms.add(x, x)
        with ms.stream(b):
            i, t = R.ids(index), ms.from_numpy(teacher)
            loss, sums = ms.distill_loss(y, i, t, temperature=2.0)
        with ms.stream(a):
            g = ms.distill_loss_grad(one, y, sums, i, t, temperature=2.0)
        with ms.stream(b):
            adjusted = ms.adjust_logits(g, i, presence=0.5, bias=t, bias_index=i)
            flat = ms.embedding(adjusted, R.ids(np.arange(4000) % rows))
        with ms.stream(a):
            table = ms.embedding_grad(flat, R.ids(tokens), 60)
        return loss, g, table

    s = ms.Stream()
    plain = [[v.numpy() for v in chain(ms.from_numpy(x), s, s)] for x in z]
    a, b = ms.Stream(), ms.Stream()
    for k in range(6):
        with ms.stream(a if k % 2 else b):
            x = ms.from_numpy(z[k % 2])
        got = chain(x, a, b)
        for v, w in zip(got, plain[k % 2]):
            assert np.array_equal(v.numpy(), w), k


def test_sums_are_read_and_written_again_on_their_own_stream():
    rng = np.random.default_rng(2)
    a, b = ms.Stream(), ms.Stream()
    with ms.stream(a):
        z = [ms.from_numpy(rng.standard_normal((2000, 5000)).astype(np.float32)) for _ in range(2)]
        i, t = R.ids(rng.integers(0, 5000, (2000, 4))), ms.from_numpy(rng.standard_normal((2000, 4)).astype(np.float32))
        loss = ms.from_numpy(np.zeros(2000, np.float32))
        want = [ms.distill_loss(v, i, t)[1].numpy() for v in z]
    with ms.stream(b):
        sums = ms.from_numpy(np.zeros((2000, 3), np.float32))
    for k in range(6):
        ms.distill_loss(z[k % 2], i, t, out=(loss, sums))
        with ms.stream(b):
            read = ms.neg(sums)
        ms.distill_loss(z[1 - k % 2], i, t, out=(loss, sums))  # waits for that read
        assert np.array_equal(-read.numpy(), want[k % 2]) and np.array_equal(sums.numpy(), want[1 - k % 2])
