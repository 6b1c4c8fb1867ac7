"""Runs of the cases of perf/operators.py through the framework's kernels.

  python perf/operator_times.py loop CASE PASSES
      passes on one state, for a profiler to look at
  python perf/operator_times.py graph [CASE ...]
      time of a pass among 30 captured into one graph, three sets of inputs in
      turn: median and least of 15 replays (all cases by default)
"""
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))
from perf import operators  # noqa: E402

operators.own = True
CASES = {case["name"]: case for case in operators.listed()}


def loop(name, passes):
    state = operators.prepare(CASES[name], 1)
    for _ in range(passes):
        operators.run(state)
    torch.cuda.synchronize()


def graph(name):
    """(median, least) microseconds of a pass."""
    states = [operators.prepare(CASES[name], seed) for seed in (1, 2, 3)]
    for state in states:
        operators.run(state)
    torch.cuda.synchronize()
    passes = torch.cuda.CUDAGraph()
    with torch.cuda.graph(passes):
        for k in range(30):
            operators.run(states[k % 3])
    times = []
    for _ in range(15):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        passes.replay()
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end) / 30 * 1e3)
    times.sort()
    return times[7], times[0]


if __name__ == "__main__":
    if len(sys.argv) == 4 and sys.argv[1] == "loop" and sys.argv[2] in CASES:
        loop(sys.argv[2], int(sys.argv[3]))
    elif len(sys.argv) > 1 and sys.argv[1] == "graph" and all(a in CASES for a in sys.argv[2:]):
        for name in sys.argv[2:] or CASES:
            print("%-20s median %7.2f us  least %7.2f us" % ((name,) + graph(name)), flush=True)
    else:
        sys.exit(__doc__)
