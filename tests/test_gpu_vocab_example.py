"""The gated recurrent example's two ends, in a child process that imports torch first (a process that holds this library's
HIP runtime and then loads torch's copy would hold two)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_example_distils_and_generates():
    r = subprocess.run([sys.executable, "-u", "-m", "tests.vocab_example_checks"], cwd=ROOT, capture_output=True, text=True,
                       timeout=110)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.count(" ok") == 4, r.stdout
