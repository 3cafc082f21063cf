"""The cases of perf/operators.py in a loop, for a kernel trace of them, and the
table of such a trace.

    rocprofv3 --kernel-trace --stats --output-format csv -d kt -- python3 profiles/run_operators.py [case,...]
    python3 profiles/run_operators.py --table kt

Each case runs twelve times over three sets of inputs, with the library's
kernels.  The table: every kernel and grid in the order of its first launch, the
median and the shortest of its durations, and the identity of the sources.
"""
import csv
import glob
import os
import re
import statistics
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def run(names):
    import torch

    from perf import operators

    operators.own = True
    for case in operators.listed():
        if names and case["name"] not in names:
            continue
        states = [operators.prepare(case, seed) for seed in range(3)]
        torch.cuda.synchronize()
        for i in range(12):
            operators.run(states[i % 3])
        torch.cuda.synchronize()
        print(case["name"], flush=True)


def table(folder):
    import bench

    rows = []
    for f in glob.glob(os.path.join(folder, "**", "*kernel_trace.csv"), recursive=True):
        with open(f) as lines:
            rows += [r for r in csv.DictReader(lines) if "bsq::" in r["Kernel_Name"]]
    times = {}
    for r in sorted(rows, key=lambda r: int(r["Start_Timestamp"])):
        name = re.sub(r"\(anonymous namespace\)::|void |bsq::", "", r["Kernel_Name"])
        name = re.sub(r"\(.*", "", re.sub(r"\((Mx4Type|Mode)\)", "", name))
        groups = [int(r["Grid_Size_" + d]) // int(r["Workgroup_Size_" + d]) for d in "XYZ"]
        grid = " x ".join(str(g) for g in groups if g > 1) or "1"
        times.setdefault((name, grid, r["Workgroup_Size_X"]), []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
    print("sources_sha256 =", bench.operators_sha256())
    for (name, grid, threads), t in times.items():
        print(f"| `{name}` | {grid} x {threads} | {len(t)} | {statistics.median(t):.1f} | {min(t):.1f} |")


if __name__ == "__main__":
    if sys.argv[1:2] == ["--table"]:
        table(sys.argv[2])
    else:
        run(sys.argv[1].split(",") if sys.argv[1:] else None)
