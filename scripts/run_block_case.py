"""Runs cases of perf/operators.py on the trainable block operators, for a profiler: ``python3 scripts/run_block_case.py NAME[,NAME] [passes]``."""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from perf import operators  # noqa: E402

if __name__ == "__main__":
    operators.own = True
    cases = {c["name"]: c for c in operators.listed()}
    for name in sys.argv[1].split(","):
        state = operators.prepare(cases[name], 1)
        for _ in range(int(sys.argv[2]) if len(sys.argv) > 2 else 20):
            operators.run(state)
        torch.cuda.synchronize()
        print(name, "done", flush=True)
