"""One case of ``perf/operators.py``, or with ``more`` of ``perf/more_operators.py``, by the framework's kernels, for a profiler: three states of the case, run in turn 24 times.

    python perf/run_case.py                               the cases' names
    python perf/run_case.py "prompt - 2048 tokens"
    python perf/run_case.py more "prompt - 2048 tokens"
"""
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch  # noqa: E402

from perf import more_operators, operators  # noqa: E402


def main():
    args = sys.argv[1:]
    more = args[:1] == ["more"]
    file = more_operators if more else operators
    cases = {c["name"]: c for c in file.listed()}
    if len(args) != 1 + more or args[-1] not in cases:
        print("\n".join(cases))
        return int(len(args) > more)
    file.own = True
    states = [file.prepare(cases[args[-1]], seed) for seed in range(3)]
    for i in range(24):
        file.run(states[i % 3])
    torch.cuda.synchronize()
    return 0


if __name__ == "__main__":
    sys.exit(main())
