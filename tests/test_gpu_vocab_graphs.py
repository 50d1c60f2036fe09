"""The vocabulary's operators in HIP graphs, in a child process that imports torch first."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_captured_operators_replay():
    r = subprocess.run([sys.executable, "-u", "-m", "tests.vocab_graph_checks"], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.count(" ok") == 2, r.stdout
