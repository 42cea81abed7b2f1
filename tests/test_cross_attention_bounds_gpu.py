"""Attention over another sequence in the bounds-checked library, in a process of its own: see tests/_bounds_cross_worker.py."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_bounds_checked_build_covers_lists_of_blocks():
    worker = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_bounds_cross_worker.py")
    res = subprocess.run([sys.executable, worker], capture_output=True, text=True, timeout=900, env=dict(os.environ, FLODL_B200_BOUNDS_CHECK="1"))
    assert res.returncode == 0 and "BOUNDS_OK" in res.stdout, res.stdout[-2000:] + res.stderr[-3000:]
