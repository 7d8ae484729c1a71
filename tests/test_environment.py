"""What importing the package asks of the HIP runtime."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("before,after", [
    (None, "8"), ("4", "8"), ("8", "8"), ("16", "16"), ("", "8"), ("x", "8")])
def test_hardware_queues(before, after):
    """Eight at least: an environment's smaller number is raised."""
    env = dict(os.environ)
    env.pop("GPU_MAX_HW_QUEUES", None)
    if before is not None:
        env["GPU_MAX_HW_QUEUES"] = before
    out = subprocess.run(
        [sys.executable, "-c", "import gloo_amd, os; "
         "print(os.environ['GPU_MAX_HW_QUEUES'])"],
        cwd=ROOT, env=env, capture_output=True, text=True, check=True)
    assert out.stdout.split()[-1] == after
