#!/usr/bin/env python
"""The workloads of perf/operators.py through the framework's own calls: one pass eagerly (host included) and replayed from a hipGraph
(what the kernels take one behind the other), or passes alone for a profiler.

    python tools/operators_probe.py [NAME,NAME]                                    # a line per case
    rocprofv3 --kernel-trace --stats -d out -o o -- python tools/operators_probe.py NAME --passes 13
"""
import argparse
import os
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "perf")]


def replayed(M, s, passes=10):
    """us per pass inside a graph of `passes` of them, the best of eight replays."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            M.run(s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(passes):
            M.run(s)
    best = float("inf")
    for _ in range(8):
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3 / passes)
    return best


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("names", nargs="?", default="")
    ap.add_argument("--passes", type=int, default=0)
    args = ap.parse_args()
    import operators as M
    M.own = True
    for case in M.listed():
        if args.names and case["name"] not in args.names.split(","):
            continue
        s = M.prepare(case, 1)
        for _ in range(args.passes or 5):
            M.run(s)
        torch.cuda.synchronize()
        if args.passes:
            continue
        t = time.perf_counter()
        for _ in range(20):
            M.run(s)
        host = (time.perf_counter() - t) * 5e4
        torch.cuda.synchronize()
        eager = (time.perf_counter() - t) * 5e4
        print(f"{case['name']:<20} eager {eager:8.1f} us a pass (host {host:7.1f})   replayed {replayed(M, s):8.1f} us", flush=True)
