"""Outputs of the distillation loss that live on other streams than the call's: ordered as the recurrent block's are
(tests/test_blocks_streams.py).  On the CPU: host memory in the place of the device, and event calls that are made to fail."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r'''
import ctypes, json, os, sys
import numpy as np
import musapy_amd as ms

lib = ctypes.CDLL(os.path.join(os.path.dirname(ms.__file__), "libmusapy_hip.so"))
EVENT = 5
if lib.mpy_rt_set_backend(1) != 0:
    print(json.dumps({"skip": "the host backend is refused here (a HIP device is present)"}))
    sys.exit(0)
a, b = ms.Stream(), ms.Stream()
results = {}


def on(s, shape, dtype="f32"):
    with ms.stream(s):
        return ms.array(np.zeros(shape), dtype=dtype)


def waits(fn):
    """How many waits between streams a call asks for: the events that it creates (one, one record and one wait each)."""
    n = 0
    while True:
        lib.mpy_rt_inject(EVENT, 1, 3 * n, 1)
        try:
            fn()
            lib.mpy_rt_inject(EVENT, 0, 0, 0)
            return n
        except ms.StreamError:
            n += 1


z, i, t = on(a, (4, 50)), on(a, (4, 3), "i64"), on(a, (4, 3))
loss, at_home, away = on(a, 4), on(a, (4, 3)), on(b, (4, 3))
results["at home"] = waits(lambda: ms.distill_loss(z, i, t, out=(loss, at_home)))
call = lambda: ms.distill_loss(z, i, t, out=(loss, away))
results["away"] = waits(call)
with ms.stream(b):
    read = ms.add(away, away)
lib.mpy_rt_inject(EVENT, 1, 0, 1)
try:
    call()
    results["after a read at home"] = "no wait"
except ms.StreamError:
    results["after a read at home"] = "waits"
lib.mpy_rt_inject(EVENT, 0, 0, 0)
got = call()
with ms.stream(b):
    results["then at home"] = [waits(lambda: ms.add(away, away)), waits(lambda: ms.add(read, read, out=away))]
results["returns"] = [got[1].stream.id == b.id, got[0].stream.id == a.id, got[1].data_ptr == away.data_ptr]
# the other operators: everything on one stream asks for no wait, an input of another stream for one
h = on(b, (4, 9), "i64")
table, tokens = on(a, (7, 5)), on(a, 6, "i64")
results["one stream"] = [waits(lambda: ms.embedding(table, tokens)), waits(lambda: ms.embedding_grad(on(a, (6, 5)), tokens, 7)),
                         waits(lambda: ms.distill_loss_grad(loss, z, at_home, i, t)), waits(lambda: ms.adjust_logits(z))]
with ms.stream(b):
    late = ms.add(on(b, (4, 50)), on(b, (4, 50)))
results["an input of another stream"] = waits(lambda: ms.adjust_logits(late, h, out=on(a, (4, 50))))
print(json.dumps(results))
'''


def test_outputs_and_inputs_of_other_streams():
    env = dict(os.environ)
    env["PYTHONPATH"] = ROOT + os.pathsep + env.get("PYTHONPATH", "")
    r = subprocess.run([sys.executable, "-c", CHILD], env=env, cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    seen = json.loads(r.stdout.strip().splitlines()[-1])
    if "skip" in seen:
        pytest.skip(seen["skip"])
    assert seen["at home"] == 0 and seen["away"] >= 2
    assert seen["after a read at home"] == "waits" and seen["then at home"] == [0, 0]
    assert seen["returns"] == [True, True, True]
    assert seen["one stream"] == [0, 0, 0, 0]
    assert seen["an input of another stream"] >= 1
