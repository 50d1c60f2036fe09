"""Outputs that live on another stream than the call's: read back from there, and written again after reads there."""
import numpy as np
import pytest

import musapy_amd as ms

pytestmark = pytest.mark.gpu


def test_outputs_are_read_and_written_again_on_their_own_streams():
    rng = np.random.default_rng(1)
    a, b = ms.Stream(), ms.Stream()
    shape = (3000, 2048)
    with ms.stream(a):
        x = [ms.array(rng.standard_normal(shape), dtype="f32") for _ in range(2)]
        r = ms.array(np.zeros(shape), dtype="f32")
        h = ms.array(np.zeros(shape), dtype="f32")
        g = ms.array(np.full(shape, 0.5), dtype="f32")
        want = [[v.numpy() for v in (ms.norm_residual(v, v)[1], ms.gated_scan(v, g, axis=0)[1])] for v in x]
    with ms.stream(b):
        y = ms.array(np.zeros(shape), dtype="f32")
        s = ms.array(np.zeros(shape[1]), dtype="f32")
    for k in range(6):
        i = k % 2
        ms.norm_residual(x[i], x[i], out=(r, y))
        ms.gated_scan(x[i], g, axis=0, out=h, state_out=s)
        if k % 3 == 0:
            assert np.array_equal(y.numpy(), want[i][0]) and np.array_equal(s.numpy(), want[i][1])
        with ms.stream(b):
            y2, s2 = ms.neg(y), ms.neg(s)
        ms.norm_residual(x[1 - i], x[1 - i], out=(r, y))  # waits for those reads
        ms.gated_scan(x[1 - i], g, axis=0, out=h, state_out=s)
        assert np.array_equal(-y2.numpy(), want[i][0]) and np.array_equal(-s2.numpy(), want[i][1])
        with ms.stream(b):
            ms.neg(y2, out=y)  # written at home behind the call
        assert np.array_equal(y.numpy(), want[i][0])
