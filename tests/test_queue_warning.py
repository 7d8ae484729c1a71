"""Hardware queues that were asked for too late."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("queues,used,warns", [
    ("4", True, True), (None, True, True), ("8", True, False),
    ("4", False, False)])
def test_import_after_the_gpu_was_used(queues, used, warns):
    """HIP reads the number at its first call: an import behind that cannot
    raise it, and says so."""
    env = dict(os.environ)
    env.pop("GPU_MAX_HW_QUEUES", None)
    if queues is not None:
        env["GPU_MAX_HW_QUEUES"] = queues
    out = subprocess.run(
        [sys.executable, "-W", "always", "-c",
         f"import torch; torch.cuda.is_initialized = lambda: {used}; "
         "import gloo_amd"],
        cwd=ROOT, env=env, capture_output=True, text=True, check=True)
    assert ("hardware queues" in out.stderr) == warns, out.stderr
