"""Calls one case of the block-scaled operators (perf/operators.py, by name) over three rotating sets of operands, for a kernel trace:
rocprofv3 --kernel-trace --stats -f csv -d DIR -- python3 tools/scaled_kernel_times.py "product prompt" 300
Prints the time of a call between two events behind the first third of the calls."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from perf import operators  # noqa: E402

operators.own = True
case = next(c for c in operators.listed() if c["name"] == sys.argv[1])
calls = int(sys.argv[2]) if len(sys.argv) > 2 else 300
sets = [operators.prepare(case, seed) for seed in range(3)]
torch.cuda.synchronize()
a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
for i in range(calls):
    if i == calls // 3:
        a.record()
    operators.run(sets[i % 3])
b.record()
torch.cuda.synchronize()
print("%s: %.2f us a call" % (case["name"], a.elapsed_time(b) * 1e3 / (calls - calls // 3)), flush=True)
