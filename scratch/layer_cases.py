"""Passes over perf/operators.py's listed cases through the kernels, for a profiler (names or parts of them as arguments: only those)."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
os.chdir(ROOT)
from perf import operators as P  # noqa: E402

P.own = True
for case in P.listed():
    if len(sys.argv) < 2 or any(a in case["name"] for a in sys.argv[1:]):
        state = P.prepare(case, 1)
        for _ in range(6):
            P.run(state)
        torch.cuda.synchronize()
        print(case["name"], flush=True)
        del state
