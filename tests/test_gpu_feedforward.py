"""The feed-forward operators on torch tensors (feedforward_check.py, in a process of its own)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_torch_tensors(gpu):
    script = os.path.join(os.path.dirname(os.path.abspath(__file__)), "feedforward_check.py")
    r = subprocess.run([sys.executable, "-u", script], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "feed-forward OK" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]
