"""The operators over a vocabulary without a GPU: the 64-bit forms that the GPU tests compare with against central
differences, and the C entry points' refusals (which launch nothing)."""
import ctypes
import os

import numpy as np
import pytest

from tests import vocab_reference as R
from tests.test_blocks_host import BF16, F32, F64, LIB, F, I, P, S

I32, I64 = 3, 4
SS = ctypes.c_ssize_t


def test_embedding_gradient_formula():
    rng = np.random.default_rng(0)
    table, tokens = rng.standard_normal((7, 5)), np.array([[0, 6, 6], [-1, 7, 2]])
    w = rng.standard_normal((2, 3, 5))
    grad, _ = R.embedding_grad(w, tokens, 7, 1.5)
    d = rng.standard_normal((7, 5))
    up, down = (float((w * R.embedding(table + s * d, tokens, 1.5)).sum()) for s in (0.5, -0.5))
    assert abs(up - down - (grad * d).sum()) < 1e-12  # linear: the difference is exact


@pytest.mark.parametrize("temp", [1.0, 2.0, 0.5])
@pytest.mark.parametrize("weight", [1.0, 0.3, 0.0])
def test_distill_gradient_formula(temp, weight):
    rng = np.random.default_rng(1)
    z = rng.standard_normal(13) * 2
    index, teacher = np.array([3, 12, 3, -1, 13, 0]), np.array([2.0, 1.0, 0.5, 9.0, 9.0, -np.inf])
    for label in (5, 3, -100, None):
        _, *sums = R.distill(z, index, teacher, label, temp, weight)
        g = R.distill_grad(1.5, z, sums, index, teacher, label, temp, weight)
        for j in range(13):
            e = np.zeros(13)
            e[j] = 1e-6
            up, down = (1.5 * R.distill(z + s * e, index, teacher, label, temp, weight)[0] for s in (1, -1))
            assert abs((up - down) / 2e-6 - g[j]) < 1e-8 * (1 + temp ** 2)


def test_packed_masks():
    rng = np.random.default_rng(2)
    ok = rng.random((2, 70)) < 0.5
    w = R.pack(ok)
    assert w.shape == (2, 3)
    for r in range(2):
        for c in range(70):
            assert bool((int(w[r, c // 32]) >> (c % 32)) & 1) == ok[r, c]


# ---- the C entry points -----------------------------------------------------------------------------
# The addresses are made up: these run where a call that is not refused cannot launch.
no_gpu = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="made-up addresses, and a GPU that could read them")


class EmbedArgs(ctypes.Structure):
    _fields_ = [("table_dtype", I), ("out_dtype", I), ("id_dtype", I), ("scale", F), ("tokens", S), ("rows", S), ("width", S),
                ("table", P), ("row_stride", SS), ("column_stride", SS), ("ids", P), ("out", P)]


class EmbedGradArgs(ctypes.Structure):
    _fields_ = [("dy_dtype", I), ("out_dtype", I), ("id_dtype", I), ("accumulate", I), ("scale", F), ("tokens", S), ("rows", S),
                ("width", S), ("dy", P), ("dy_pitch", S), ("ids", P), ("out", P)]


class DistillArgs(ctypes.Structure):
    _fields_ = [("dtype", I), ("index_dtype", I), ("teacher_dtype", I), ("label_dtype", I), ("temperature", F), ("weight", F),
                ("rows", S), ("width", S), ("entries", S), ("logits", P), ("pitch", S), ("index", P), ("index_pitch", S),
                ("teacher", P), ("teacher_pitch", S), ("labels", P), ("loss", P), ("sums", P), ("dloss", P), ("dloss_stride", SS),
                ("dlogits", P)]


class AdjustArgs(ctypes.Structure):
    _fields_ = [("dtype", I), ("out_dtype", I), ("history_dtype", I), ("lengths_dtype", I), ("bias_dtype", I), ("index_dtype", I),
                ("allowed_kind", I), ("rows", S), ("width", S), ("length", S), ("entries", S), ("logits", P), ("pitch", S),
                ("history", P), ("history_pitch", S), ("lengths", P), ("repetition", P), ("presence", P), ("frequency", P),
                ("repetition_value", F), ("presence_value", F), ("frequency_value", F), ("bias", P), ("bias_pitch", S),
                ("bias_index", P), ("index_pitch", S), ("allowed", P), ("allowed_pitch", S), ("out", P)]


def lib():
    L = ctypes.CDLL(LIB)
    for n, args in {"musapy_embedding_v1": [P, P], "musapy_embedding_grad_v1": [P, P, S, P], "musapy_distill_loss_v1": [P, P, S, P],
                    "musapy_distill_loss_grad_v1": [P, P], "musapy_adjust_logits_v1": [P, P]}.items():
        getattr(L, n).argtypes, getattr(L, n).restype = args, I
    for n in ("musapy_embedding_grad_scratch_v1", "musapy_distill_loss_scratch_v1"):
        getattr(L, n).argtypes, getattr(L, n).restype = [P], S
    L.musapy_kernels_take_error()
    return L


def made(cls, base, kw):
    a = cls()
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


def refused(fn, L, a, *rest, error=6):
    assert fn(ctypes.byref(a) if a is not None else None, *rest, None) == -1
    assert L.musapy_kernels_take_error() == error


@no_gpu
def test_embedding_refusals():
    L = lib()
    base = dict(table_dtype=F32, out_dtype=BF16, id_dtype=I32, scale=1, tokens=4, rows=8, width=16, table=64, row_stride=16,
                column_stride=1, ids=64, out=64)
    for kw in (dict(table_dtype=F64), dict(out_dtype=I32), dict(id_dtype=F32), dict(tokens=1 << 31), dict(rows=1 << 31),
               dict(width=1 << 31), dict(table=None), dict(ids=None), dict(out=None), dict(rows=0),
               dict(tokens=1 << 30, width=64)):
        refused(L.musapy_embedding_v1, L, made(EmbedArgs, base, kw))
    refused(L.musapy_embedding_v1, L, None)
    for kw in (dict(tokens=0, ids=None, out=None, rows=0, table=None), dict(width=0)):
        assert L.musapy_embedding_v1(ctypes.byref(made(EmbedArgs, base, kw)), None) == 0


@no_gpu
def test_embedding_grad_refusals():
    L = lib()
    base = dict(dy_dtype=F32, out_dtype=BF16, id_dtype=I64, scale=1, tokens=600, rows=8, width=16, dy=64, dy_pitch=16, ids=64, out=64)
    for kw in (dict(dy_dtype=F64), dict(out_dtype=I32), dict(id_dtype=F32), dict(accumulate=2), dict(tokens=1 << 31),
               dict(rows=1 << 31), dict(width=(1 << 22) + 1), dict(width=1 << 31), dict(dy=None), dict(ids=None), dict(out=None)):
        refused(L.musapy_embedding_grad_v1, L, made(EmbedGradArgs, base, kw), 64, 1 << 40)
    refused(L.musapy_embedding_grad_v1, L, None, None, 0)
    a = made(EmbedGradArgs, base, {})
    need = L.musapy_embedding_grad_scratch_v1(ctypes.byref(a))
    assert need > 0
    refused(L.musapy_embedding_grad_v1, L, a, None, 0, error=1)
    refused(L.musapy_embedding_grad_v1, L, a, 64, need - 1, error=1)
    refused(L.musapy_embedding_grad_v1, L, a, 72, need, error=1)  # not 16-byte aligned
    for kw in (dict(rows=0), dict(width=0), dict(tokens=0, accumulate=1)):
        a = made(EmbedGradArgs, base, kw)
        assert L.musapy_embedding_grad_v1(ctypes.byref(a), None, 0, None) == 0
        assert L.musapy_embedding_grad_scratch_v1(ctypes.byref(a)) == 0
    assert L.musapy_embedding_grad_scratch_v1(None) == 0


@no_gpu
def test_distill_refusals():
    L = lib()
    base = dict(dtype=F32, index_dtype=I32, teacher_dtype=BF16, label_dtype=I64, temperature=1, weight=0.5, rows=4, width=100,
                entries=8, logits=64, pitch=100, index=64, index_pitch=8, teacher=64, teacher_pitch=8, labels=64, loss=64, sums=64,
                dloss=64, dloss_stride=1, dlogits=64)
    nan = float("nan")
    for fn, *scratch in ((L.musapy_distill_loss_v1, None, 0), (L.musapy_distill_loss_grad_v1,)):
        for kw in (dict(dtype=F64), dict(index_dtype=F32), dict(teacher_dtype=I32), dict(label_dtype=F32), dict(temperature=0),
                   dict(temperature=-1), dict(temperature=nan), dict(temperature=2e6), dict(weight=-0.1), dict(weight=1.1),
                   dict(weight=nan), dict(rows=1 << 31), dict(width=1 << 31), dict(entries=1025), dict(logits=None),
                   dict(index=None), dict(teacher=None), dict(sums=None)):
            refused(fn, L, made(DistillArgs, base, kw), *scratch)
        refused(fn, L, None, *scratch)
        assert fn(ctypes.byref(made(DistillArgs, base, dict(rows=0, logits=None))), *scratch, None) == 0
    refused(L.musapy_distill_loss_v1, L, made(DistillArgs, base, dict(loss=None)), None, 0)
    # more workgroups than a launch has: a wave a row, eight a row, one for each 4 KB and one more
    for kw in (dict(rows=1 << 26), dict(rows=1 << 23, width=40000)):
        refused(L.musapy_distill_loss_v1, L, made(DistillArgs, base, kw), None, 0)
    refused(L.musapy_distill_loss_grad_v1, L, made(DistillArgs, base, dict(rows=1 << 25)))
    # few long rows go through scratch
    assert L.musapy_distill_loss_scratch_v1(ctypes.byref(made(DistillArgs, base, {}))) == 0
    long = made(DistillArgs, base, dict(width=1 << 20, pitch=1 << 20))
    need = L.musapy_distill_loss_scratch_v1(ctypes.byref(long))
    assert need > 0 and L.musapy_distill_loss_scratch_v1(None) == 0
    refused(L.musapy_distill_loss_v1, L, long, None, 0, error=1)
    refused(L.musapy_distill_loss_v1, L, long, 64, need - 1, error=1)
    refused(L.musapy_distill_loss_v1, L, long, 66, need, error=1)
    for kw in (dict(dloss=None), dict(dlogits=None)):
        refused(L.musapy_distill_loss_grad_v1, L, made(DistillArgs, base, kw))


@no_gpu
def test_adjust_refusals():
    L = lib()
    base = dict(dtype=BF16, out_dtype=F32, history_dtype=I32, lengths_dtype=I32, bias_dtype=F32, index_dtype=I64, allowed_kind=0,
                rows=4, width=100, length=10, entries=3, logits=64, pitch=100, history=64, history_pitch=10, lengths=64,
                repetition_value=1, bias=64, bias_pitch=3, bias_index=64, index_pitch=3, allowed=64, allowed_pitch=100, out=64)
    fn = L.musapy_adjust_logits_v1
    for kw in (dict(dtype=F64), dict(out_dtype=9), dict(history_dtype=F32), dict(lengths_dtype=F32), dict(bias_dtype=I32), dict(dtype=F32, bias_dtype=BF16), dict(rows=1 << 23),
               dict(index_dtype=F32), dict(allowed_kind=2), dict(rows=1 << 31), dict(width=1 << 31), dict(length=1 << 31),
               dict(entries=1025), dict(logits=None), dict(out=None), dict(bias=None), dict(bias_index=None)):
        refused(fn, L, made(AdjustArgs, base, kw))
    refused(fn, L, None)
    for kw in (dict(rows=0, logits=None), dict(width=0)):
        assert fn(ctypes.byref(made(AdjustArgs, base, kw)), None) == 0
