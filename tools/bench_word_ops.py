"""Kernel times of the word operators (scan2cap_amd/word_ops.py) on the cases of perf/operators.py:

    python tools/bench_word_ops.py [name,name,...]

Per case: the kernels of one pass with their times (torch.profiler), their sum, what the pass has to read and
write, and the rate.  Three sets of inputs in turn, so that a pass does not find its logits in the caches.
"""
import collections
import os
import re
import sys

import torch
from torch.profiler import ProfilerActivity, profile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "perf")]
import operators  # noqa: E402

PASSES = 15


def main():
    operators.own = True
    names = sys.argv[1].split(",") if len(sys.argv) > 1 else None
    for case in operators.listed():
        if names and case["name"] not in names:
            continue
        states = [operators.prepare(case, seed) for seed in (1, 2, 3)]
        for s in states:
            operators.run(s)
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            for i in range(PASSES):
                operators.run(states[i % 3])
            torch.cuda.synchronize()
        kernels = collections.OrderedDict()
        for e in p.events():
            if e.device_type == torch.autograd.DeviceType.CUDA:
                m = re.search(r"(\w+_kernel)(<[^>]*>)?", e.name)
                name = "".join(g or "" for g in m.groups()) if m else e.name
                kernels[name] = kernels.get(name, 0.0) + e.device_time / PASSES
        total = sum(kernels.values())
        size = operators.work(case)["bytes"]
        print("%-20s %8.1f us %8.1f MB %6.0f GB/s   %s" % (
            case["name"], total, size / 1e6, size / total / 1e3,
            ", ".join("%s %.1f" % kv for kv in kernels.items())), flush=True)
        del states


if __name__ == "__main__":
    main()
