"""The block-scaled 8-bit operations on torch tensors, recorded with torch's graphs (torch_graph_program)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_recorded_with_torch():
    program = os.path.join(os.path.dirname(os.path.abspath(__file__)), "torch_graph_program.py")
    run = subprocess.run([sys.executable, "-u", program], capture_output=True, text=True, timeout=110)
    assert run.returncode == 0 and "replays equal the eager calls" in run.stdout, run.stdout[-2000:] + run.stderr[-4000:]
