"""bench.py's guard when rank 0, in whose process the ranks' key-value store lives, is the first to read why a leg
failed: it leaves, and the store with it, before the others have looked."""
import json
import os
import subprocess
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import os, sys
sys.path.insert(0, %r)
import torch.distributed as dist
import bench
rank = int(os.environ["RANK"])
dist.init_process_group("gloo")
extras = {}
def run():
    if rank == 1:
        raise RuntimeError("boom on the second rank")
    dist.barrier()
bench.run_guarded(run, extras, {"metric": "m", "value": 1.0}, rank, 60.0, poll_s=0.1 if rank == 0 else 4.0)
"""


def test_the_others_do_not_wait_for_their_limit():
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29617", WORLD_SIZE="3")
    start = time.time()
    procs = [subprocess.Popen([sys.executable, "-c", SCRIPT % ROOT], env=dict(env, RANK=str(r)), stdout=subprocess.PIPE,
                              stderr=subprocess.PIPE, text=True) for r in range(3)]
    outs = [p.communicate(timeout=110) for p in procs]
    assert time.time() - start < 50, "the ranks waited for their limit"
    assert [p.returncode for p in procs] == [0, 0, 0], [o[1][-1500:] for o in outs]
    lines = [line for line in outs[0][0].splitlines() if line.startswith("{")]
    assert len(lines) == 1 and json.loads(lines[0])["extras_error"] == "rank 1: RuntimeError: boom on the second rank"
    assert not any("{" in o[0] for o in outs[1:])
