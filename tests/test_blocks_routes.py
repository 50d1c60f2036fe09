"""How the gated scans are launched, without a GPU: every route covers every lane with a kernel that there is."""
import ctypes

import pytest

from tests.test_blocks_host import BF16, F32, S, ScanArgs, lib

WALK, TILES, ROWS = 0, 1, 2


class Route(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int), ("vector", ctypes.c_int), ("split", ctypes.c_int), ("rows", S), ("lanes", S),
                ("vectors", S), ("chains", S), ("tiles", S)]


def route(shape, axis, dtype, grad, shared=False):
    """The route of contiguous operands; shared: one gate for the last axis, its gradient summed over it."""
    L = lib()
    L.musapy_gated_scan_route_v1.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    n = len(shape)
    st = [1] * n
    for i in range(n - 2, -1, -1):
        st[i] = st[i + 1] * shape[i + 1]
    sh, sts = (S * n)(*shape), (ctypes.c_ssize_t * n)(*st)
    gst = (ctypes.c_ssize_t * n)(*[0 if shared and i == n - 1 else s for i, s in enumerate(st)])
    a = ScanArgs(kind=0, dtype=dtype, gate_dtype=F32, dgate_dtype=F32, ndim=n, axis=axis, shape=sh, x=64, x_strides=sts, gate=64,
                 gate_strides=gst, h=64, h_strides=sts, dh=64, dh_strides=sts, out=64, dgate=64)
    if shared and grad:
        a.parts = L.musapy_gated_scan_parts_v1(ctypes.byref(a))
        assert a.parts > 0
    r = Route()
    assert L.musapy_gated_scan_route_v1(ctypes.byref(a), grad, ctypes.byref(r)) == 0
    return r


# below and above the longest axis whose tiles' workgroups a grid can number, which goes step by step
LONG = [(1, 65_000_000, 4), (1, 65_100_000, 4), (1, 65_100_000, 64), (1, 65_100_000, 61), (3, 40_000_000, 200),
        (1, 1 << 31, 9), (2, 65_100_000, 1)]
SHORT = [(1, 1, 5), (8, 1, 2048), (2, 6, 37), (64, 16, 8192), (2, 300, 61), (8, 2048, 4096), (4, 21, 999), (1, 1, 600000)]


@pytest.mark.parametrize("shape", LONG + SHORT, ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("grad", [0, 1])
@pytest.mark.parametrize("shared", [False, True])
def test_every_lane_has_a_thread(shape, dtype, grad, shared):
    if shared and shape[2] == 1:
        return
    r = route(shape, 1, dtype, grad, shared)
    whole = 4 if dtype == F32 else 8
    assert r.rows * r.lanes == shape[0] * shape[2]
    assert r.vectors == -(-r.lanes // r.vector)
    if r.kind == WALK:
        assert r.vector in ((1, 2, whole) if grad else (1, 2))
    elif r.kind == TILES:
        assert r.vector == whole and r.chains * 8 >= r.rows * r.vectors and r.tiles * 128 >= shape[1]
        assert (r.chains + 31) * r.tiles * 256 < 1 << 32
    else:
        assert r.vector == 1 and r.chains == r.rows * r.lanes
    if r.split:
        assert r.tiles > 1


def test_which_calls_go_step_by_step():
    assert route((1, 65_000_000, 4), 1, BF16, 0).kind == TILES
    assert route((1, 65_100_000, 4), 1, BF16, 0).kind == WALK
    assert route((1, 65_100_000, 4), 1, BF16, 0).vector == 2
    assert route((8, 1, 2048), 1, BF16, 0).kind == WALK
    assert route((4, 1500, 5001), 2, F32, 0).kind == ROWS
    assert route((2, 0, 5), 1, F32, 0).rows == 2 and route((2, 4, 0), 1, F32, 0).rows == 0
    L = lib()
    assert L.musapy_gated_scan_route_v1(None, 0, ctypes.byref(Route())) == -1 and L.musapy_kernels_take_error() == 6


def test_extents_whose_products_wrap_round():
    """Lanes, and elements, that 64 bits do not hold are refused, not numbered by what is left of them."""
    L = lib()
    L.musapy_gated_scan_route_v1.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    for shape, axis in (((1 << 31, 1, 1 << 31, 4), 1), ((1 << 31, 9, 1 << 31, 1 << 2), 1), ((1 << 16, 5, 1 << 16, 1 << 32), 1),
                        ((1 << 31, (1 << 32) - 1, 2), 1), (((1 << 32) - 1, (1 << 32) - 1), 0)):
        n = len(shape)
        st = (ctypes.c_ssize_t * n)(*[0] * n)
        for grad in (0, 1):
            a = ScanArgs(kind=0, dtype=F32, gate_dtype=F32, dgate_dtype=F32, ndim=n, axis=axis, shape=(S * n)(*shape), x=64,
                         x_strides=st, gate=64, gate_strides=st, h=64, h_strides=st, dh=64, dh_strides=st, out=64, dgate=64)
            assert L.musapy_gated_scan_route_v1(ctypes.byref(a), grad, ctypes.byref(Route())) == -1, shape
            assert L.musapy_kernels_take_error() == 6
