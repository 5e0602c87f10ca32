#!/usr/bin/env python3
"""Times of the drafted-decoding operators (manual_whisper_amd.paged) on the cases of perf/operators.py.

    python tools/drafted_times.py [out.csv]        per case: us a call as a program makes it (calls one after another, Python included) and
                                                   us of GPU time a call (the same calls in a graph), medians of 15 rounds in turn
    python tools/drafted_times.py --trace          the graphs alone, for `rocprofv3 --kernel-trace`
    python tools/drafted_times.py --calls N TEXT   N calls of the cases whose names hold TEXT, for `rocprofv3 --pmc`
    python tools/drafted_times.py --summary kernel_trace.csv out.csv        per kernel and grid: launches, smallest, median and mean us

Three input sets of a case take turns, so that no call finds its own inputs in the caches (256 MB of one set stay in the last level)."""
import collections
import csv
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def short(name):
    """paged_plan_kernel, tree_attn_wide_kernel<f16, true, 128>: plain and mangled names alike (the demangler knows no f16)."""
    m = re.match(r"_ZN2mw12_GLOBAL__N_1\d+(\w+?_kernel)I(\w+?)EEv", name)
    if not m:
        return re.sub(r"\(.*", "", name.replace("mw::(anonymous namespace)::", "").replace("void ", ""))
    args = re.findall(r"DF16b|DF16_|Lb[01]|Li\d+", m.group(2))
    plain = {"DF16b": "bf16", "DF16_": "f16", "Lb0": "false", "Lb1": "true"}
    return f"{m.group(1)}<{', '.join(plain.get(a, a[2:]) for a in args)}>"


def summary(trace, out):
    times = collections.OrderedDict()
    with open(trace, newline="") as f:
        for r in csv.DictReader(f):
            name = r["Kernel_Name"]
            if any(k in name for k in ("tree_attn", "tree_join", "paged_", "accept_")):
                grid = "x".join(r[k] for k in ("Grid_Size_X", "Grid_Size_Y", "Grid_Size_Z"))
                times.setdefault((short(name), grid), []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
    with open(out, "w", newline="") as f:
        w = csv.writer(f)
        w.writerow(["kernel", "grid_threads", "launches", "min_us", "median_us", "mean_us"])
        for (name, grid), v in times.items():
            v.sort()
            w.writerow([name, grid, len(v), f"{v[0]:.2f}", f"{v[len(v) // 2]:.2f}", f"{sum(v) / len(v):.2f}"])


if sys.argv[1:2] == ["--summary"]:
    summary(*sys.argv[2:4])
    sys.exit()

sys.path[:0] = [ROOT, os.path.join(ROOT, "perf")]
import manual_whisper_amd  # noqa: E402,F401  (before torch: it sets the number of hardware queues)
import operators  # noqa: E402
import torch  # noqa: E402

CALLS = 45          # of a graph, and of a round
operators.own = True


def graph_of(states):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for i in range(CALLS):
            operators.run(states[i % 3])
    return g


def timed(work):
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    work()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) * 1e3 / CALLS


def eager(states):
    for i in range(CALLS):
        operators.run(states[i % 3])


def main():
    calls, only, out = 0, "", None
    if sys.argv[1:2] == ["--calls"]:
        calls, only = int(sys.argv[2]), sys.argv[3]
    elif len(sys.argv) > 1 and not sys.argv[1].startswith("--"):
        out = sys.argv[1]
    rows = []
    for case in operators.listed():
        if only not in case["name"]:
            continue
        states = [operators.prepare(dict(case), seed) for seed in range(3)]
        if calls:
            for i in range(calls):
                operators.run(states[i % 3])
            torch.cuda.synchronize()
            print(case["name"], flush=True)
            continue
        for s in states:
            operators.run(s)
        torch.cuda.synchronize()
        g = graph_of(states)
        for _ in range(3):
            g.replay()
            eager(states)
        torch.cuda.synchronize()
        if "--trace" in sys.argv:
            for _ in range(5):
                g.replay()
            torch.cuda.synchronize()
            print(case["name"], flush=True)
        else:
            both = [(timed(lambda: eager(states)), timed(g.replay)) for _ in range(15)]
            call, gpu = (sorted(x)[7] for x in zip(*both))
            rows.append([case["name"], f"{call:.2f}", f"{gpu:.2f}"])
            print(f"{case['name']:28s} call {call:8.2f} us  gpu {gpu:8.2f} us", flush=True)
        del states, g
        torch.cuda.empty_cache()
    if out:
        with open(out, "w", newline="") as f:
            w = csv.writer(f)
            w.writerow(["case", "call_us", "gpu_us"])
            w.writerows(rows)


main()
