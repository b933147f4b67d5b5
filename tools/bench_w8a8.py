#!/usr/bin/env python3
"""The W8A8 operators at the workloads of perf/operators.py and at further sizes and forms.

  python3 tools/bench_w8a8.py [--passes 30]        us a call among others (host included), the best of three runs of 60 ms or `passes` calls
  rocprofv3 --kernel-trace --stats -f csv -d DIR -o NAME -- python3 tools/bench_w8a8.py --trace-run
  python3 tools/bench_w8a8.py --summary DIR/.../NAME_kernel_trace.csv        median and minimum time of each workload's kernels

Two states of each workload in turn.  DS_HIP_LIBRARY selects another build of the library."""
import argparse
import csv
import importlib.util
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
KERNEL = re.compile(r"gemm_i8_few_kernel|gemm_i8_tile_kernel|rows_team_kernel|rows_long_kernel|dequant_any_kernel|dequant_kernel|align_rows_kernel")


def workloads():
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True

    def product(m, n, k, out="f16", residual=None, act="none"):
        return {"op": "product", "m": m, "k": k, "n": n, "out": out, "residual": residual, "bias": True, "act": act, "lda_extra": 0,
                "name": f"product {m} x {n} x {k} {act if act != 'none' else ''} {out} {'+ ' + residual if residual else ''}"}

    def norm(m, n, x, residual, out):
        return {"op": "norm", "m": m, "n": n, "x": x, "residual": residual, "out": out, "name": f"norm {m} x {n} {x} {'+ ' + residual if residual else ''} -> {out}"}

    further = [product(8192, 8192, 8192), product(4096, 4096, 4096), product(163840, 640, 640, "f32", "f32"), product(40960, 1280, 5120, "f32", "f32"),
               product(40960, 10240, 1280, "f32", act="geglu"), product(97866, 8704, 464, "f32", act="geglu"), product(117446, 5617, 407, act="silu"),
               product(100001, 2001, 1001), product(2048, 1280, 1280), product(283, 2288, 6512), product(73, 173, 4215), product(3276, 757, 4627),
               norm(655360, 320, "f16", None, "f16"), norm(655360, 320, "f16", None, "f32"), norm(655360, 320, "f16", "f32", "f16"), norm(655360, 320, "f32", "f16", "f16"),
               norm(3001, 1283, "f16", None, "f16"), norm(3001, 1280, "f16", "f32", "i8"), norm(300, 20011, "f16", "f32", "i8")]
    return ops, ops.listed() + further


def run(passes, timed):
    import torch
    ops, cases = workloads()
    for case in cases:
        states = [ops.prepare(case, seed) for seed in (1, 2)]
        torch.cuda.synchronize()
        for i in range(5 if timed else passes):
            ops.run(states[i % 2])
        torch.cuda.synchronize()
        if timed:
            best = None
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            n = passes
            for _ in range(4):
                begin.record()
                for i in range(n):
                    ops.run(states[i % 2])
                end.record()
                torch.cuda.synchronize()
                us = begin.elapsed_time(end) * 1e3 / n
                best = us if best is None else min(best, us)
                n = max(passes, int(60e3 / us))
            print(f"{best:10.2f} us  {case['name']}", flush=True)
        else:
            print(case["name"], flush=True)
        del states


def summary(path):
    """A workload's kernels follow one another without another kernel between them (its inputs are made before)."""
    _, cases = workloads()
    runs, inside = [], False
    rows = sorted(csv.DictReader(open(path)), key=lambda r: int(r["Start_Timestamp"]))
    for r in rows:
        if not KERNEL.search(r["Kernel_Name"]):
            inside = False
            continue
        if not inside:
            runs.append({})
            inside = True
        name = re.sub(r"\(anonymous namespace\)::|\(.*$|^void |_ZN12_GLOBAL__N_1\d+|EEvNS_.*$|EvPK.*$", "", r["Kernel_Name"])
        key = (name, r["Grid_Size_X"], r["Workgroup_Size_X"])
        runs[-1].setdefault(key, []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
    assert len(runs) == len(cases), f"{len(runs)} runs of kernels, {len(cases)} workloads"
    print("# rocprofv3 --kernel-trace of tools/bench_w8a8.py --trace-run on one MI355X: median and minimum us of each workload's kernels")
    for case, kernels in zip(cases, runs):
        print(case["name"].strip())
        for (name, grid, group), us in kernels.items():
            us.sort()
            print(f"  {us[len(us) // 2]:9.2f} (least {us[0]:9.2f}) x {len(us):3d}  {name}  {grid} / {group} threads")


if __name__ == "__main__":
    a = argparse.ArgumentParser()
    a.add_argument("--passes", type=int, default=30)
    a.add_argument("--trace-run", action="store_true")
    a.add_argument("--summary")
    a = a.parse_args()
    if a.summary:
        summary(a.summary)
    else:
        run(a.passes, not a.trace_run)
