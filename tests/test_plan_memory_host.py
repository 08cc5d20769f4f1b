"""A planner that runs out of host memory reports it; no C++ exception leaves a C entry
(which would end the process)."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

SCRIPT = """
import resource
import numpy as np
from specgrove_amd import ops
make = getattr(ops, {entry!r})
n = 4_000_000
offset, lengths = np.zeros(n + 1, np.int32), np.zeros(n, np.int32)
make([0, 1], [5], 32, 8, 128)
pages = int(open("/proc/self/statm").read().split()[0])
before = resource.getrlimit(resource.RLIMIT_AS)
resource.setrlimit(resource.RLIMIT_AS, (pages * 4096 + (4 << 20), before[1]))
try:
    make(offset, lengths, 32, 8, 128)
except RuntimeError as e:
    print("reported:", e)
resource.setrlimit(resource.RLIMIT_AS, before)
print("units", make([0, 1], [5], 32, 8, 128).units)
"""


@pytest.mark.parametrize("entry", ["plan_attention", "plan_attention_mx4"])
def test_a_planner_without_memory_reports_it(entry):
    run = subprocess.run([sys.executable, "-c", SCRIPT.format(entry=entry)], cwd=ROOT,
                         capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr
    assert "reported: sg_tree_attn_plan" in run.stdout and "no host memory" in run.stdout
    assert "units 8" in run.stdout
