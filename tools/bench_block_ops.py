#!/usr/bin/env python3
"""Times the layer-level operators for blocks of language models (include/qcnn.h: qcnn_op_matvec_w4, qcnn_op_grouped_matmul,
qcnn_op_norm_res) on the cases of perf/operators.py.  Not the headline benchmark (bench.py is).

Inputs are cold: copies of a case's buffers are used in turn, so many that what a call reads is 1 GiB in all, at most 64 (those of
the smallest calls do fit into the L2s and the 256 MB last cache).  With --warm two copies are used in turn.  For each case,
medians of nine runs:
  device  one call of a captured graph of calls
  call    one call of a loop of calls made from Python, launches on their way ahead of the GPU
  plain   with --plain: the plain form of perf/operators.py (elementary 32-bit operations), in a loop
  floor   what the case reads, writes and computes at the rates of a 1 GiB copy and an 8192^3 product, both timed here first
          (int8 taken as twice bfloat16)

    python tools/bench_block_ops.py [--warm] [--plain] [--only NAME[,NAME]]
"""
import argparse
import importlib.util
import os
import statistics
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
operators = importlib.util.module_from_spec(spec)
spec.loader.exec_module(operators)

ap = argparse.ArgumentParser()
ap.add_argument("--warm", action="store_true")
ap.add_argument("--plain", action="store_true")
ap.add_argument("--only", default="")
a = ap.parse_args()


def device_us(go):
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    ev[0].record()
    go()
    ev[1].record()
    torch.cuda.synchronize()
    return ev[0].elapsed_time(ev[1]) * 1e3


def median(f, n=9):
    f()
    return statistics.median(f() for _ in range(n))


src = torch.zeros(1 << 30, dtype=torch.uint8, device="cuda")
dst = torch.empty_like(src)
rate = {"copy": 2 * src.numel() / median(lambda: device_us(lambda: dst.copy_(src))) * 1e6}
for t in ("bf16", "f16", "f32"):
    m = torch.randn(8192, 8192, device="cuda").to(operators.TYPES[t])
    rate[t] = 2 * 8192 ** 3 / median(lambda: device_us(lambda: m @ m.t())) * 1e6
rate["i8"] = 2 * rate["bf16"]
del src, dst, m
print("copy %.0f GB/s; products %s TFLOP/s" % (rate["copy"] / 1e9, ", ".join("%s %.0f" % (t, rate[t] / 1e12) for t in ("bf16", "f16", "f32"))), flush=True)
print("%-24s %10s %10s %10s %10s  %s" % ("case", "floor us", "device us", "call us", "plain us" if a.plain else "", "copies"), flush=True)
for case in operators.listed():
    if a.only and case["name"] not in a.only.split(","):
        continue
    work = operators.work(case)
    operators.own = True
    first = operators.prepare(case, 0)
    written = sum(t.numel() * t.element_size() for t in (first["h"], first["n"])) if case["op"] == "norm" else first["y"].numel() * first["y"].element_size()
    copies = 2 if a.warm else max(2, min(64, -(-(1 << 30) // max(1, work["bytes"] - written))))
    states = [first] + [operators.prepare(case, i) for i in range(1, copies)]
    floor = max(work["bytes"] / rate["copy"], work["flops"] / rate[case["type"]] if case["op"] != "norm" else 0) * 1e6
    n = max(copies, 24)

    def calls():
        for i in range(n):
            operators.run(states[i % copies])
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    device = median(lambda: device_us(graph.replay)) / n

    def wall():
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        calls()
        torch.cuda.synchronize()
        return (time.perf_counter() - t0) * 1e6
    call = median(wall) / n
    plain = ""
    if a.plain:
        operators.own = False
        plain = "%10.0f" % median(lambda: device_us(lambda: [operators.run(s) for s in states[:4]]) / min(4, copies), 3)
    print("%-24s %10.2f %10.2f %10.2f %10s  %d" % (case["name"], floor, device, call, plain, copies), flush=True)
    del graph, states, first
