"""The attention of groups called by several host threads at once, from their first calls on."""
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

CHILD = """
import sys, threading
import torch
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
from test_gpu_beam_kernels import Groups

# sizes of a kernel that take more and less shared memory: queries of 2 to 64 rows, segments of few and many groups
made = [(Groups([2] * G, [170] * (G * B), 8, 2, D, dtype, seed=G), G, B) for D in (64, 128) for dtype in (torch.bfloat16, torch.float32)
        for G, B in ((1, 1), (2, 16), (60, 2), (1, 4))]
torch.cuda.synchronize()
start, failed, results = threading.Barrier(len(made)), [], [None] * len(made)

def call(i):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            for _ in range(20):
                results[i] = made[i][0].run()
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        failed.append((i, repr(e)))

threads = [threading.Thread(target=call, args=(i,)) for i in range(len(made))]
[t.start() for t in threads]
[t.join() for t in threads]
assert not failed, failed
torch.cuda.synchronize()
for (g, _, _), got in zip(made, results):
    assert torch.equal(g.run(), got)
    g.check()
print("all equal")
"""


def test_first_calls_of_several_threads():
    r = subprocess.run([sys.executable, "-c", CHILD.format(root=str(ROOT))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "all equal" in r.stdout, r.stderr[-2000:]
