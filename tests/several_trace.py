"""A call of several continuations of a sequence, some times over, for a profiler:

    python3 tests/several_trace.py CASE [TIMES]

CASE is one of perf/more_operators.py's listed ones; two states in turn, so that no call finds the last one's data in a cache.
"""
import importlib.util
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
spec = importlib.util.spec_from_file_location("more_operators", os.path.join(ROOT, "perf", "more_operators.py"))
operators = importlib.util.module_from_spec(spec)
spec.loader.exec_module(operators)
operators.own = True

case = next(c for c in operators.listed() if c["name"] == sys.argv[1])
states = [operators.prepare(case, seed) for seed in range(2)]
for k in range(int(sys.argv[2]) if len(sys.argv) > 2 else 40):
    operators.run(states[k % 2])
operators.queue().finish()
print(case["name"], "done", flush=True)
