"""Runs of the cases of perf/operators.py and perf/more_operators.py through the
framework's kernels.

  python perf/operator_times.py loop CASE PASSES
      passes on one state, for a profiler to look at
  python perf/operator_times.py graph [CASE[:SETS] ...]
      time of a pass among 30 captured into one graph, SETS sets of inputs in
      turn (three by default; more where three stay in the last-level cache):
      median and least of 15 replays (all cases by default)
"""
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))
from perf import more_operators, operators  # noqa: E402

operators.own = more_operators.own = True
CASES = {case["name"]: (module, case) for module in (operators, more_operators) for case in module.listed()}


def loop(name, passes):
    module, case = CASES[name]
    state = module.prepare(case, 1)
    for _ in range(passes):
        module.run(state)
    torch.cuda.synchronize()


def graph(name, sets=3):
    """(median, least) microseconds of a pass."""
    module, case = CASES[name]
    states = [module.prepare(case, 1 + seed) for seed in range(sets)]
    for state in states:
        module.run(state)
    torch.cuda.synchronize()
    passes = torch.cuda.CUDAGraph()
    with torch.cuda.graph(passes):
        for k in range(30):
            module.run(states[k % sets])
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


def _asked(text):
    """(case, sets) of CASE or CASE:SETS, or None."""
    name, _, sets = text.partition(":")
    if name in CASES and (not sets or sets.isdigit() and 0 < int(sets) <= 30):
        return name, int(sets or 3)


if __name__ == "__main__":
    if len(sys.argv) == 4 and sys.argv[1] == "loop" and sys.argv[2] in CASES:
        loop(sys.argv[2], int(sys.argv[3]))
    elif len(sys.argv) > 1 and sys.argv[1] == "graph" and all(_asked(a) for a in sys.argv[2:]):
        for asked in sys.argv[2:] or CASES:
            print("%-20s median %7.2f us  least %7.2f us" % ((asked,) + graph(*_asked(asked))), flush=True)
    else:
        sys.exit(__doc__)
