"""Device times of the attention operators on the listed cases of perf/operators.py.

    python perf/device_time.py [name,...]

For each case, in microseconds:

floor     the case's bytes at the copy rate or its flops at the bf16 rate of MEASURED_PEAKS.json, whichever is longer
plain     the plain form's pass, without the append's dequantised view of the cache that `run` returns
chain     the library's call in a chain captured as a graph: 12 calls over three sets of inputs, median of 7 replays
launched  the library's call in ordinary launches over the same sets for about a second, the mean; and the median
          SM clock sampled meanwhile (MHz)

The sets of the large cases exceed L2; the small cases' stay in it, as between the layers of a step.
"""
import json
import os
import statistics
import subprocess
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

from perf import operators as o  # noqa: E402

CALLS, SETS, SECONDS = 12, 3, 1.0


def events(f):
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    f()
    b.record()
    b.synchronize()
    return a.elapsed_time(b) * 1e3


def chain(sets):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        for i in range(CALLS):
            o._call(sets[i % SETS])
    for _ in range(3):
        graph.replay()
    return statistics.median(events(graph.replay) for _ in range(7)) / CALLS


def launched(sets, guess):
    n = max(30, int(SECONDS * 1e6 / max(guess, 8.0)))

    def calls():
        for i in range(n):
            o._call(sets[i % SETS])

    clocks = subprocess.Popen(["nvidia-smi", "-i", str(torch.cuda.current_device()), "--query-gpu=clocks.sm",
                               "--format=csv,noheader,nounits", "-lms", "100"], stdout=subprocess.PIPE, text=True)
    try:
        events(calls)  # the clock settles
        t = events(calls) / n
    finally:
        clocks.terminate()
    seen = [int(x) for x in clocks.communicate()[0].split() if x.isdigit()]
    return t, statistics.median(seen[len(seen) // 2:]) if seen else 0


def main():
    only = sys.argv[1].split(",") if len(sys.argv) > 1 else None
    peaks = {"hbm_gbs": 6552.0, "bf16_tflops": 1679.3}  # of one B200, where none were measured beside the tree
    if os.path.exists(os.path.join(ROOT, "MEASURED_PEAKS.json")):
        with open(os.path.join(ROOT, "MEASURED_PEAKS.json")) as f:
            peaks = json.load(f)
    print("%-26s %9s %9s %9s %9s %9s" % ("case", "floor", "plain", "chain", "launched", "MHz"))
    for c in o.listed():
        if only and c["name"] not in only:
            continue
        sets = [o.prepare(c, i) for i in range(SETS)]
        plain = {"append": o._append, "decode": o._decode, "prompt": o._prompt}[c["op"]]
        plain(sets[0])
        p = statistics.median(events(lambda: plain(s)) for s in sets)
        for s in sets:
            o._call(s)
        torch.cuda.synchronize()
        w, t = o.work(c), chain(sets)
        floor = max(w["bytes"] / peaks["hbm_gbs"] / 1e3, w["flops"] / peaks["bf16_tflops"] / 1e6)
        print("%-26s %9.2f %9.1f %9.2f %9.2f %9d" % ((c["name"], floor, p, t) + launched(sets, t)), flush=True)
        del sets, plain, s
        torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
