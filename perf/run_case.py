"""One case of ``perf/operators.py`` by the framework's kernels, for a profiler: three states of the case, run in turn 24 times.

    python perf/run_case.py                          the cases' names
    python perf/run_case.py "prompt - 2048 tokens"
"""
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch  # noqa: E402

from perf import operators  # noqa: E402


def main():
    cases = {c["name"]: c for c in operators.listed()}
    if len(sys.argv) != 2 or sys.argv[1] not in cases:
        print("\n".join(cases))
        return int(len(sys.argv) > 1)
    operators.own = True
    states = [operators.prepare(cases[sys.argv[1]], seed) for seed in range(3)]
    for i in range(24):
        operators.run(states[i % 3])
    torch.cuda.synchronize()
    return 0


if __name__ == "__main__":
    sys.exit(main())
