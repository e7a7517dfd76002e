"""The quantised linear layers' kernels built with their index checks (FMS_B200_DEBUG_BOUNDS=1): their tests run under the flag in
a process of their own, where a fixture in conftest.py fails any that records an index."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_quantized_kernels_stay_inside_their_arrays():
    run = subprocess.run([sys.executable, "-m", "pytest", "tests/test_quantized_gpu.py", "-x", "-q", "-p", "no:cacheprovider"], cwd=ROOT,
                         env=dict(os.environ, FMS_B200_DEBUG_BOUNDS="1"), capture_output=True, text=True, timeout=900)
    assert run.returncode == 0, run.stdout[-4000:] + run.stderr[-2000:]
    assert " passed" in run.stdout and "skipped" not in run.stdout, run.stdout[-1000:]
