"""How the norm cuts a tensor follows from the tensor, not from the calls before it: the same launches in a process whose first call
asked for large tables of groups as in one that began with the tensor itself."""
import json
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

PROGRAM = """
import json, sys
sys.path.insert(0, %r)
import torch
from torch.profiler import ProfilerActivity, profile
from actnn_b200.cpp_extension import group_norm

def both(n, c, h, w, groups):
    x = torch.randn(n, h, w, c, device="cuda").half().movedim(-1, 1)
    y, codes, stats = group_norm.forward(x, groups, activation="silu")
    group_norm.backward(x, codes, stats, groups, activation="silu")

if sys.argv[1] == "after":
    both(300, 2048, 12, 12, 2048)               # 2048 groups a block: 64 KB of tables
with profile(activities=[ProfilerActivity.CUDA]) as p:
    both(7, 192, 95, 95, 32)                   # the same kernels (vectors across groups), 2 KB of tables
    torch.cuda.synchronize()
p.export_chrome_trace(sys.argv[2])
events = json.load(open(sys.argv[2]))["traceEvents"]
print(json.dumps([[e["name"], e["args"]["grid"]] for e in sorted(events, key=lambda e: e.get("ts", 0)) if e.get("cat") == "kernel" and "gn_" in e["name"]]))
"""


def launches(tmp_path, when):
    out = subprocess.run([sys.executable, "-c", PROGRAM % ROOT, when, str(tmp_path / (when + ".json"))], capture_output=True, text=True,
                         timeout=300, cwd=ROOT)
    assert out.returncode == 0, out.stderr[-2000:]
    return json.loads(out.stdout.strip().splitlines()[-1])


def test_the_same_launches(cuda_device, tmp_path):
    first, after = launches(tmp_path, "first"), launches(tmp_path, "after")
    if not first:
        pytest.skip("the profiler records no launches here")
    assert len(first) >= 4 and first == after
