"""Windows, several axes and a teacher on two gloo ranks equal the single-process model."""
import json
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_two_ranks(tmp_path):
    out = os.path.join(str(tmp_path), "out")
    env = dict(os.environ, PYTHONPATH=os.pathsep.join((ROOT, os.path.join(ROOT, "tests"))), CUDA_VISIBLE_DEVICES="")
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1",
           "--master-port", "29571", os.path.join(ROOT, "tests", "_long_context_worker.py"), out]
    r = subprocess.run(cmd, env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
    for rank in range(2):
        with open(f"{out}.{rank}") as f:
            res = json.load(f)
        tp, z = res["tp"], res["zero3"]
        assert abs(tp["loss"] - tp["want"]) < 1e-4 and max(tp["grads"]) < 1e-3 and tp["refused"] == 2, tp
        assert max(abs(a - b) for a, b in zip(z["losses"], z["want"])) < 1e-4 and z["diff"] < 2e-5, z
