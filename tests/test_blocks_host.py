"""The gated recurrent block's operators without a GPU: the 64-bit forms that the GPU tests compare with against central
differences and published values, and the C entry points' refusals (which launch nothing)."""
import ctypes
import os

import numpy as np
import pytest

from tests import blocks_reference as R

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "musapy_amd", "libmusapy_hip.so")


def test_philox_known_answers():
    """The known-answer vectors that the generator's authors publish for Philox4x32-10."""
    ones = 0xFFFFFFFF
    assert R.philox4x32((0, 0, 0, 0), (0, 0)) == (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)
    assert R.philox4x32((ones,) * 4, (ones,) * 2) == (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)
    assert R.philox4x32((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == (
        0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)


@pytest.mark.parametrize("kind", ["decay", "blend"])
@pytest.mark.parametrize("gshape", [(2, 9, 3), (2, 9, 1), (1, 1, 3)])
def test_scan_gradient_formula(kind, gshape):
    rng = np.random.default_rng(1)
    x, g, h0 = rng.standard_normal((2, 9, 3)), rng.random(gshape), rng.standard_normal((2, 3))
    cut = rng.random((2, 9, 1)) < 0.2
    w, ws = rng.standard_normal((2, 9, 3)), rng.standard_normal((2, 3))

    def loss(x, g, h0):
        h, s = R.scan(x, g, h0, cut, 1, kind)
        return (w * h).sum() + (ws * s).sum()

    grads = R.scan_grad(w, x, g, R.scan(x, g, h0, cut, 1, kind)[0], h0, cut, ws, 1, kind)
    check_differences(loss, [x, g, h0], grads)


@pytest.mark.parametrize("post", ["rms", "layer", None])
@pytest.mark.parametrize("pre", ["rms", "layer", None])
@pytest.mark.parametrize("gate_kind", ["silu", "sigmoid"])
def test_block_gradient_formula(post, pre, gate_kind):
    rng = np.random.default_rng(2)
    o = {"post": post, "pre": pre, "gate_kind": gate_kind, "eps": 1e-5}
    x, res, gate, dr, dy = (rng.standard_normal((4, 11)) for _ in range(5))
    w1, scale, w2 = (rng.standard_normal(11) for _ in range(3))
    keep = (rng.random((4, 11)) < 0.7) / 0.7

    def loss(x, res, gate, w1, scale, w2):
        r, y = R.block(x, res, gate, w1, scale, w2, keep, o)
        return (dr * r).sum() + ((dy * y).sum() if pre else 0.0)

    r, _ = R.block(x, res, gate, w1, scale, w2, keep, o)
    g = R.block_grad(dr, dy, x, r, gate, w1, scale, w2, keep, o)
    grads = [g["dx"], g["dresidual"], g["dgate"], g["dpost_weight"], g["dscale"],
             np.zeros(11) if g["dpre_weight"] is None else g["dpre_weight"]]
    check_differences(loss, [x, res, gate, w1, scale, w2], grads)


def check_differences(loss, args, grads):
    """Every entry of every gradient against a central difference: 64-bit noise of 1e-10 and the square of the step."""
    step = 1e-6
    for i, a in enumerate(args):
        d = np.empty(a.shape)
        for at in np.ndindex(a.shape):
            ends = []
            for s in (step, -step):
                b = a.copy()
                b[at] += s
                ends.append(loss(*(b if j == i else v for j, v in enumerate(args))))
            d[at] = (ends[0] - ends[1]) / (2 * step)
        assert np.allclose(d, grads[i], rtol=1e-6, atol=1e-7), i


def test_rounding_to_bf16():
    x = np.array([1.0, 1.00390625, 1.01171875, -3.14159, 1e-40, 65504.0])
    assert R.rounded(x, "bf16").tolist() == [1.0, 1.0, 1.015625, -3.140625, 2.0 ** -133, 65536.0]


# ---- the C entry points -----------------------------------------------------------------------------
I, P, S, F = ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_float
SZ, SS = ctypes.POINTER(ctypes.c_size_t), ctypes.POINTER(ctypes.c_ssize_t)


class ScanArgs(ctypes.Structure):
    _fields_ = [("kind", I), ("dtype", I), ("gate_dtype", I), ("dgate_dtype", I), ("ndim", I), ("axis", I), ("shape", SZ),
                ("x", P), ("x_strides", SS), ("gate", P), ("gate_strides", SS), ("reset", P), ("reset_strides", SS),
                ("h", P), ("h_strides", SS), ("dh", P), ("dh_strides", SS), ("first", P), ("dlast", P), ("out", P),
                ("dgate", P), ("last", P), ("parts", S)]


class NormArgs(ctypes.Structure):
    _fields_ = [("dtype", I), ("stream_dtype", I), ("weight_dtype", I), ("post", I), ("pre", I), ("gate_kind", I),
                ("eps", F), ("scale_value", F), ("threshold", ctypes.c_uint32), ("seed", ctypes.c_uint64),
                ("offset", ctypes.c_uint64), ("rows", S), ("width", S), ("x", P), ("x_pitch", S), ("residual", P),
                ("residual_pitch", S), ("gate", P), ("gate_pitch", S), ("dr", P), ("dr_pitch", S), ("dy", P), ("dy_pitch", S),
                ("post_weight", P), ("scale", P), ("pre_weight", P), ("r", P), ("y", P), ("dx", P), ("dresidual", P),
                ("dgate", P), ("dpost_weight", P), ("dscale", P), ("dpre_weight", P)]


F32, F64, BF16 = 10, 11, 12


def lib():
    L = ctypes.CDLL(LIB)
    for n, args in {"musapy_gated_scan_v1": [P, P, S, P, S, P], "musapy_gated_scan_grad_v1": [P, P, S, P, S, P],
                    "musapy_norm_residual_v1": [P, P], "musapy_norm_residual_grad_v1": [P, P, S, P],
                    "musapy_dropout_v1": [P, P, I, I, SZ, SS, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_uint64, P]}.items():
        getattr(L, n).argtypes = args
        getattr(L, n).restype = I
    for n, args in {"musapy_gated_scan_scratch_v1": [P, I], "musapy_gated_scan_parts_v1": [P],
                    "musapy_norm_residual_scratch_v1": [P]}.items():
        getattr(L, n).argtypes = args
        getattr(L, n).restype = S
    return L


def scan_args(**kw):
    shape, st = (S * 3)(2, 50, 64), (ctypes.c_ssize_t * 3)(3200, 64, 1)
    a = ScanArgs(kind=0, dtype=F32, gate_dtype=F32, dgate_dtype=F32, ndim=3, axis=1, shape=shape, x=64, x_strides=st, gate=64,
                 gate_strides=st, h=64, h_strides=st, dh=64, dh_strides=st, out=64, dgate=64)
    a.keep = (shape, st)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("name", ["musapy_gated_scan_v1", "musapy_gated_scan_grad_v1"])
def test_scan_refusals(name):
    L = lib()
    fn = getattr(L, name)
    grad = "grad" in name
    bad = [dict(kind=2), dict(kind=-1), dict(dtype=F64), dict(gate_dtype=BF16), dict(shape=None), dict(gate_strides=None),
           dict(gate=None), dict(out=None), dict(reset=64)]
    bad += [dict(h=None), dict(dh=None), dict(dgate=None), dict(h_strides=None), dict(dgate_dtype=BF16), dict(parts=1),
            dict(kind=1, x=None)] if grad else [dict(x=None), dict(x_strides=None)]
    L.musapy_kernels_take_error()
    for kw in bad:
        assert fn(ctypes.byref(scan_args(**kw)), None, 0, None, 0, None) == -1, kw
        assert L.musapy_kernels_take_error() == 6, kw
    for kw in (dict(ndim=0), dict(ndim=33), dict(axis=3), dict(axis=-1)):
        assert fn(ctypes.byref(scan_args(**kw)), None, 0, None, 0, None) == -1, kw
        assert L.musapy_kernels_take_error() == 3, kw
    assert fn(None, None, 0, None, 0, None) == -1 and L.musapy_kernels_take_error() == 6
    empty = scan_args(shape=(S * 3)(2, 50, 0), x=None, gate=None, out=None, h=None, dh=None, dgate=None)
    assert fn(ctypes.byref(empty), None, 0, None, 0, None) == 0
    # lanes are numbered in 32 bits
    assert fn(ctypes.byref(scan_args(shape=(S * 3)(1 << 20, 1, 1 << 20))), None, 0, None, 0, None) == -1
    assert L.musapy_kernels_take_error() == 6


def test_shared_gate_parts():
    L = lib()
    st = (ctypes.c_ssize_t * 3)(50, 1, 0)
    for width, dtype, want in ((64, F32, 2), (64, BF16, 1), (128, BF16, 2), (96, BF16, 3), (37, BF16, 5), (1, F32, 1),
                               (16, F32, 1), (12, F32, 3)):
        a = scan_args(gate_strides=st, dtype=dtype, shape=(S * 3)(2, 50, width))
        assert L.musapy_gated_scan_parts_v1(ctypes.byref(a)) == want, width
    assert L.musapy_gated_scan_parts_v1(ctypes.byref(scan_args())) == 0  # a gate of its own for every lane
    assert L.musapy_gated_scan_parts_v1(None) == 0


def test_norm_refusals():
    L = lib()

    def args(**kw):
        a = NormArgs(dtype=F32, stream_dtype=F32, weight_dtype=F32, post=1, pre=1, gate_kind=1, eps=1e-6, scale_value=1.0,
                     rows=4, width=64, x=64, x_pitch=64, residual=64, residual_pitch=64, r=64, y=64, dx=64)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    L.musapy_kernels_take_error()
    for kw in (dict(dtype=F64), dict(stream_dtype=BF16), dict(weight_dtype=BF16), dict(post=3), dict(pre=-1),
               dict(gate=64, gate_kind=0), dict(threshold=65537), dict(rows=1 << 31), dict(width=1 << 31), dict(x=None)):
        assert L.musapy_norm_residual_v1(ctypes.byref(args(**kw)), None) == -1, kw
        assert L.musapy_kernels_take_error() == 6, kw
        assert L.musapy_norm_residual_grad_v1(ctypes.byref(args(**kw)), None, 0, None) == -1, kw
        assert L.musapy_kernels_take_error() == 6, kw
    assert L.musapy_norm_residual_v1(ctypes.byref(args(r=None)), None) == -1 and L.musapy_kernels_take_error() == 6
    assert L.musapy_norm_residual_grad_v1(ctypes.byref(args(residual=None)), None, 0, None) == -1
    assert L.musapy_kernels_take_error() == 6
    # column sums without scratch
    a = args(dscale=64)
    assert L.musapy_norm_residual_scratch_v1(ctypes.byref(a)) > 0
    assert L.musapy_norm_residual_grad_v1(ctypes.byref(a), None, 0, None) == -1 and L.musapy_kernels_take_error() == 1
    assert L.musapy_norm_residual_scratch_v1(ctypes.byref(args())) == 0
    assert L.musapy_norm_residual_v1(None, None) == -1 and L.musapy_kernels_take_error() == 6
    assert L.musapy_norm_residual_v1(ctypes.byref(args(rows=0, x=None, r=None)), None) == 0


def test_dropout_refusals():
    L = lib()
    shape, st = (S * 2)(4, 8), (ctypes.c_ssize_t * 2)(8, 1)
    L.musapy_kernels_take_error()
    for dtype, ndim, sh, t, a, err in ((F64, 2, shape, 1, 64, 6), (F32, 2, shape, 65537, 64, 6), (F32, 2, shape, 1, None, 6),
                                       (F32, 33, shape, 1, 64, 3), (F32, -1, shape, 1, 64, 3), (F32, 2, None, 1, 64, 6),
                                       (F32, 2, (S * 2)(1 << 32, 8), 1, 64, 6), (F32, 2, (S * 2)(1, 1 << 35), 1, 64, 6)):
        assert L.musapy_dropout_v1(a, 64, dtype, ndim, sh, st, t, 1, 0, None) == -1
        assert L.musapy_kernels_take_error() == err
    assert L.musapy_dropout_v1(None, None, F32, 2, (S * 2)(4, 0), st, 1, 1, 0, None) == 0
