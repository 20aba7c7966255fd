"""The operators of the shared and pruned cache on the checked build of the kernels (PAE_BOUNDS=1; csrc/common.cuh), which is chosen when the
package is imported: in a process of their own."""

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_the_operators_on_the_checked_build():
    probe = Path(__file__).resolve().parent / "cache_operators_bounds_probe.py"
    done = subprocess.run([sys.executable, str(probe)], capture_output=True, text=True, timeout=600, env=dict(os.environ, PAE_BOUNDS="1"))
    assert done.returncode == 0, (done.stdout[-3000:] + "\n" + done.stderr[-3000:])
    assert "CACHE OPERATORS BOUNDS PROBE OK" in done.stdout
