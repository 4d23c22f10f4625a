"""The attention half of a decoder layer on the GPU at the limits of its arguments, where tests of ordinary sizes say
nothing."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


# ---- lines_plan

FRESH = """
import random, sys
sys.path[:0] = [{root!r} + "/tests", {root!r} + "/comfyui-drama3_b200"]
import torch
import lines_ref as ref
from test_lines_gpu import check_plan, fault, lines_case, run_plan
cuda = torch.device("cuda", 0)
for lines in (3007, 3008, 3050, 3071, 3072):
    rng = random.Random(lines)
    lengths = [rng.randrange(0, 40) for _ in range(lines)]
    counts = [rng.randrange(0, 3) for _ in range(lines)]
    table, free, used, tokens = lines_case(lengths, counts, 16, 0, seed=lines)
    _, p = run_plan(cuda, lengths, counts, table, free, used, 16, tokens, 0)
    check_plan(p, ref.plan(lengths, counts, table, free, used, 16, tokens, 0), table)
    assert fault() == 0
print("planned")
"""


def test_plan_of_line_counts_around_48_kb_of_shared_memory(cuda):
    # in a process of its own: a plan of more lines raises the kernel's ceiling for all later ones
    run = subprocess.run([sys.executable, "-c", FRESH.format(root=str(ROOT))], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0 and run.stdout.endswith("planned\n"), run.stderr[-2000:]
