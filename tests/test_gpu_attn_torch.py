"""The cache-attention binding over torch tensors (attn_torch_child.py, a process of its own)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_torch_tensors(gpu):
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "attn_torch_child.py")
    # torch alone may take two minutes to load at first
    p = subprocess.run([sys.executable, child], capture_output=True, text=True, timeout=240)
    assert p.returncode == 0, p.stdout + p.stderr
    assert p.stdout.splitlines() == ["views ok", "side stream ok", "graph ok", "host tensor refused"]
