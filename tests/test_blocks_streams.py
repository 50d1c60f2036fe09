"""Outputs of the gated recurrent block's operators that live on other streams than the call's: ordered like any other
array's, before the call and behind it.  On the CPU: host memory in the place of the device, and event calls that are made
to fail (tests/test_runtime_injection.py), so that a wait that is asked for shows as a StreamError."""
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


def on(s, shape=(4, 8), dtype="f32"):
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


def calls(home):
    """Calls on stream a, with one output at home on `home` and the others on a."""
    x, g, h0 = on(a), on(a), on(a, (8,))
    w = on(a, (8,))
    one = lambda *s: on(a, s or (4, 8))
    far = lambda *s: on(home, s or (4, 8))
    out = {}
    r, y = one(), far()
    out["norm_residual"] = (y, lambda: ms.norm_residual(x, x, out=(r, y)))
    h, st = one(), far(8)
    out["gated_scan"] = (st, lambda: ms.gated_scan(x, g, h0, axis=0, out=h, state_out=st))
    dx, dg, d0 = one(), far(), one(8)
    out["gated_scan_grad"] = (dg, lambda: ms.gated_scan_grad(x, x, g, x, h0, axis=0, out=(dx, dg, d0)))
    ex, er, ew = one(), one(), far(8)
    out["norm_residual_grad"] = (ew, lambda: ms.norm_residual_grad(x, x, x, x, pre_weight=w, out=(ex, er, None, None, None, ew)))
    return out


for name, (y, call) in calls(a).items():
    results[name + " at home"] = waits(call)
for name, (y, call) in calls(b).items():
    results[name + " away"] = waits(call)
    with ms.stream(b):
        z = ms.add(y, y)                     # read at home: not recorded, the home stream itself is waited for
    lib.mpy_rt_inject(EVENT, 1, 0, 1)
    try:
        call()
        results[name + " after a read at home"] = "no wait"
    except ms.StreamError:
        results[name + " after a read at home"] = "waits"
    lib.mpy_rt_inject(EVENT, 0, 0, 0)
    call()
    # reading or writing it at home comes after the call without a further wait: home waits for the call
    with ms.stream(b):
        results[name + " then at home"] = [waits(lambda: ms.add(y, y)), waits(lambda: ms.add(z, z, out=y))]
    got = call()
    at = [i for i, v in enumerate(got) if v is not None and v.data_ptr == y.data_ptr][0]
    results[name + " returns"] = [got[at].stream.id == b.id, y.stream.id == b.id]
print(json.dumps(results))
'''


@pytest.fixture(scope="module")
def seen():
    env = dict(os.environ)
    env["PYTHONPATH"] = ROOT + os.pathsep + env.get("PYTHONPATH", "")
    r = subprocess.run([sys.executable, "-c", CHILD], env=env, cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    out = json.loads(r.stdout.strip().splitlines()[-1])
    if "skip" in out:
        pytest.skip(out["skip"])
    return out


@pytest.mark.parametrize("name", ["norm_residual", "gated_scan", "gated_scan_grad", "norm_residual_grad"])
def test_an_output_of_another_stream(seen, name):
    assert seen[name + " at home"] == 0
    assert seen[name + " away"] >= 2  # before the call on the output's stream, and there on the call
    assert seen[name + " after a read at home"] == "waits"
    assert seen[name + " then at home"] == [0, 0]
    assert seen[name + " returns"] == [True, True]
