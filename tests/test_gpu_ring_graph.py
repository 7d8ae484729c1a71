"""The ring allreduce's captured schedule, over processes on one GPU: ranks
that share a device within a process go without it."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)


@pytest.mark.parametrize("size", [2, 4])
def test_ring_graph_replays(tmp_path, size):
    worker = os.path.join(os.path.dirname(__file__), "ring_graph_worker.py")
    env = dict(os.environ, GLOO_AMD_LOG_LEVEL="INFO")
    procs = [subprocess.Popen(
        [sys.executable, worker, str(r), str(size), str(tmp_path)],
        stdout=subprocess.PIPE, stderr=subprocess.STDOUT, env=env)
        for r in range(size)]
    try:
        outs = [p.communicate(timeout=100)[0].decode() for p in procs]
    finally:
        for p in procs:
            if p.poll() is None:
                p.kill()
    for p, out in zip(procs, outs):
        assert p.returncode == 0 and "ALL OK" in out, out[-2000:]
        assert "captured ring schedule graph" in out, out[-2000:]
