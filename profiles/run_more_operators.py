"""The cases of perf/more_operators.py in a loop, for a kernel trace of them, and the
table of such a trace.

    rocprofv3 --kernel-trace --stats --output-format csv -d kt -- python3 profiles/run_more_operators.py [case,...]
    python3 profiles/run_more_operators.py --table kt

Each case runs twelve times over three sets of inputs, with the library's
kernels.  The table: every kernel and grid in the order of its launches, twelve to
a line, the median and the shortest of their durations, and the identity of the
sources.

    python3 profiles/run_more_operators.py --further

Times of cases beside those: other sizes of heads, types, numbers of queries, and
attention that is not causal; a pass among others over three sets of inputs, the
median of seven blocks of passes.
"""
import csv
import glob
import os
import re
import statistics
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
RUNS = 12


def run(names):
    import torch

    from perf import more_operators

    more_operators.own = True
    for case in more_operators.listed():
        if names and case["name"] not in names:
            continue
        states = [more_operators.prepare(case, seed) for seed in range(3)]
        torch.cuda.synchronize()
        for i in range(RUNS):
            more_operators.run(states[i % 3])
        torch.cuda.synchronize()
        print(case["name"], flush=True)


def further_cases(M):
    cases = [M._attention(f"64 requests of 4096 keys, {q} heads on {h} of {d}", 64, 4096, 4096, q, h, d) for q, h, d in
             ((32, 8, 64), (32, 8, 96), (32, 8, 128), (32, 8, 192), (32, 8, 256), (8, 8, 128), (32, 2, 128))]
    cases += [M._attention(f"64 requests of 4096 keys, {t}", 64, 4096, 4096, 32, 8, 128, type=t, out=t) for t in ("f16", "f32")]
    cases += [M._attention(f"64 requests of 4096 keys, {n} queries each", 64, 4096, 4096, 32, 8, 128, new=n, chunks=64)
              for n in (4, 8, 16)]
    cases += [M._attention(f"prompt of 4096, heads of {d}, {t}", 1, 0, 0, 32, 8, d, page=64, new=4096, chunks=1, type=t, out=t)
              for d, t in ((64, "bf16"), (128, "bf16"), (256, "bf16"), (128, "f16"), (128, "f32"))]
    cases += [M._attention("512 queries on 64 thousand keys", 1, 65024, 65024, 32, 8, 128, page=64, new=512, chunks=1)]
    cases += [M._attention(f"{what}, not causal", *a, 32, 8, 128, page=64, **k) for what, a, k in
              (("prompt of 4096", (1, 0, 0), dict(new=4096, chunks=1)), ("64 requests of 4096 keys", (64, 4096, 4096), {}))]
    cases += [M._rope(f"rope of 8192 tokens, 32 heads of 128, {t}, forward and gradient", 8192, 32, 128, 128, type=t, train=True)
              for t in ("bf16", "f32")]
    return cases + [M._append(f"append of 8191 tokens, 32 and 8 heads of 128, {t}, and back", 8191, 32, 8, 128, 64, type=t)
                    for t in ("bf16", "f32")]


def not_causal(M, state):
    import bitsqz_amd as B
    import torch

    case, q = state["case"], state["q"]
    if "work" not in state:
        M.run(state)  # its buffers
    B.check(B.lib().bsq_kv4_attention(
        state["handle"], state["table"].data_ptr(), state["table"].shape[1], state["lengths"].data_ptr(),
        state["starts"].data_ptr(), case["requests"], q.data_ptr(), 1, q.shape[0], case["new"] if case["chunks"] else 1,
        case["queries"], case["queries"] * case["dim"], state["scale"], 0, 0, state["out"].data_ptr(), 1,
        case["queries"] * case["dim"], state["lse"].data_ptr(), state["work"].data_ptr(), state["work"].numel(),
        torch.cuda.current_stream().cuda_stream), "kv4 attention")


def further():
    import torch

    import bench
    from perf import more_operators as M

    M.own = True
    print("sources_sha256 =", bench.more_operators_sha256())
    for case in further_cases(M):
        states, causal, work = [M.prepare(case, seed) for seed in range(3)], "not causal" not in case["name"], M.work(case)
        if not causal:  # every query sees every key
            seen = sum(m * (p + m) for p, m in M._lengths(case))
            work["flops"] = 4 * seen * case["queries"] * case["dim"]

        def block(n):
            torch.cuda.synchronize()
            begin = time.perf_counter()
            for i in range(n):
                M.run(states[i % 3]) if causal else not_causal(M, states[i % 3])
            torch.cuda.synchronize()
            return (time.perf_counter() - begin) / n

        n = max(10, min(500, int(0.1 / block(10))))
        block(3 * n)
        s = statistics.median(block(n) for _ in range(7))
        print(f"| {case['name']} | {s * 1e6:.1f} | {work['bytes'] / s / 1e12:.2f} | {work['flops'] / s / 1e12:.0f} |", flush=True)
        del states
        torch.cuda.empty_cache()


def table(folder):
    import bench

    rows = []
    for f in glob.glob(os.path.join(folder, "**", "*kernel_trace.csv"), recursive=True):
        with open(f) as lines:
            rows += [r for r in csv.DictReader(lines) if "bsq::" in r["Kernel_Name"]]
    times, seen = {}, {}
    for r in sorted(rows, key=lambda r: int(r["Start_Timestamp"])):
        name = re.sub(r"\(anonymous namespace\)::|void |bsq::", "", r["Kernel_Name"])
        name = re.sub(r"\(.*", "", re.sub(r"\((Mx4Type|Mode)\)", "", name))
        groups = [int(r["Grid_Size_" + d]) // int(r["Workgroup_Size_" + d]) for d in "XYZ"]
        grid = " x ".join(str(g) for g in groups if g > 1) or "1"
        key = name, grid, r["Workgroup_Size_X"]
        seen[key] = seen.get(key, -1) + 1
        times.setdefault((*key, seen[key] // RUNS), []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
    print("sources_sha256 =", bench.more_operators_sha256())
    for (name, grid, threads, _), t in times.items():
        print(f"| `{name}` | {grid} x {threads} | {len(t)} | {statistics.median(t):.1f} | {min(t):.1f} |")


if __name__ == "__main__":
    if sys.argv[1:2] == ["--table"]:
        table(sys.argv[2])
    elif sys.argv[1:2] == ["--further"]:
        further()
    else:
        run(sys.argv[1].split(",") if len(sys.argv) > 1 else [])
