"""Passes of one case, for a profiler to watch: three states of it in turn.

    python3 perf/passes.py operators|more_operators CASE PASSES
"""
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main(module, name, passes):
    cases = importlib.import_module("perf." + module)
    cases.own = True
    case = next(c for c in cases.listed() if c["name"] == name)
    states = [cases.prepare(case, seed) for seed in range(3)]
    torch.cuda.synchronize()
    for _ in range(passes):
        for state in states:
            cases.run(state)
    torch.cuda.synchronize()


if __name__ == "__main__":
    if len(sys.argv) != 4:
        sys.exit(__doc__)
    main(sys.argv[1], sys.argv[2], int(sys.argv[3]))
