"""Runs cases of the sequence operators (perf/operators.py's listed ones and the further shapes that comments in csrc/ quote),
for profiling; and sums up what the profiler wrote.

    python tools/seq_cases.py --list
    python tools/seq_cases.py "scan prompt 1 x 8192" [runs]
    python tools/seq_cases.py --summary <folder of one sub-folder per case> > profiles/seq_kernel_stats.csv
"""

import csv
import glob
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def cases():
    from perf import operators
    scan = dict(op="scan", dtype="bf16", channels=2048, groups=1)
    norm = dict(op="norm", form="full")
    further = [dict(scan, name="scan prompt 16 x 1024, {} states".format(n), mode="prompt", batch=16, length=1024, state=n, ragged=False) for n in (4, 8, 16)]
    further += [dict(scan, name="scan train 8 x 2048, {} states".format(n), mode="train", batch=8, length=2048, state=n) for n in (4, 8, 32, 64)]
    further += [dict(scan, name="scan token 256 streams, {} states".format(n), mode="token", batch=256, slots=320, state=n) for n in (61, 64)]
    further += [dict(norm, name="norm train 16387 rows", mode="train", dtype="bf16", rows=16387, channels=2048),
                dict(norm, name="norm train 16032 rows bf16", mode="train", dtype="bf16", rows=16032, channels=1285),
                dict(norm, name="norm train 4096 rows of 8192", mode="train", dtype="bf16", rows=4096, channels=8192),
                dict(norm, name="norm train 4096 rows of 8192 fp32", mode="train", dtype="fp32", rows=4096, channels=8192),
                dict(norm, name="norm prompt 4096 rows of 5000", mode="infer", dtype="bf16", rows=4096, channels=5000)]
    further += [dict(op="conv", name="conv train 8 x 4096", mode="train", dtype="bf16", batch=8, length=4096, channels=2048, taps=4)]
    return operators, operators.listed() + further


def run(name, runs):
    import torch
    operators, known = cases()
    operators.own = True
    case, = (c for c in known if c["name"] == name)
    states = [operators.prepare(case, seed) for seed in range(3)]
    for k in range(runs):
        operators.run(states[k % 3])
    torch.cuda.synchronize()
    print("ran", name, flush=True)


def short(kernel):
    """_ZN6unetmi15scan_fwd_kernelIDF16bLi4ELNS_8ScanPassE2EEEv.. -> scan_fwd_kernel<bf16, 4, marks>"""
    m = re.match(r"_ZN6unetmi(\d+)", kernel)
    at = m.end()
    name, rest = kernel[at:at + int(m[1])], kernel[at + int(m[1]):]
    if rest[0] != "I":
        return name
    words = {"DF16b": "bf16", "f": "float", "Lb0E": "false", "Lb1E": "true", "LNS_8ScanPassE0E": "states", "LNS_8ScanPassE1E": "outputs",
             "LNS_8ScanPassE2E": "marks"}
    args = re.match(r"I((?:DF16b|f|L[ib]\d+E|LNS_8ScanPassE\dE)*)E", rest)[1]
    return "{}<{}>".format(name, ", ".join(words.get(a, a[2:-1]) for a in re.findall(r"DF16b|f|L[ib]\d+E|LNS_8ScanPassE\dE", args)))


def summary(folder):
    _, known = cases()
    out = csv.writer(sys.stdout, lineterminator="\n")
    out.writerow(["case", "kernel", "grid", "calls", "median_us", "min_us", "vector_busy", "vector_instructions_per_wave"])
    for case in known:
        here = os.path.join(folder, re.sub(r"\W+", "_", case["name"]))
        times, counters = {}, {}
        for path in glob.glob(here + "/**/*kernel_trace.csv", recursive=True):
            for r in csv.DictReader(open(path)):
                if "unetmi" in r["Kernel_Name"]:
                    grid = "x".join(str(int(r["Grid_Size_" + a]) // int(r["Workgroup_Size_" + a])) for a in "XYZ")
                    size = 1
                    for a in "XYZ":
                        size *= int(r["Grid_Size_" + a])
                    times.setdefault((short(r["Kernel_Name"]), grid, size), []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
        for path in glob.glob(here + "/**/*counter_collection.csv", recursive=True):
            for r in csv.DictReader(open(path)):
                if "unetmi" in r["Kernel_Name"]:
                    counters.setdefault((short(r["Kernel_Name"]), int(r["Grid_Size"])), {}).setdefault(r["Counter_Name"], []).append(float(r["Counter_Value"]))
        for (kernel, grid, size), t in times.items():
            t.sort()
            c = {k: sorted(v)[len(v) // 2] for k, v in counters.get((kernel, size), {}).items()}
            busy = "{:.2f}".format(c["SQ_ACTIVE_INST_VALU"] / c["SQ_BUSY_CU_CYCLES"]) if c.get("SQ_BUSY_CU_CYCLES") else ""
            per_wave = "{:.0f}".format(c["SQ_INSTS_VALU"] / c["SQ_WAVES"]) if c.get("SQ_WAVES") else ""
            out.writerow([case["name"], kernel, grid, len(t), "{:.1f}".format(t[len(t) // 2]), "{:.1f}".format(t[0]), busy, per_wave])


if __name__ == "__main__":
    if sys.argv[1] == "--list":
        print("\n".join(c["name"] for c in cases()[1]))
    elif sys.argv[1] == "--summary":
        summary(sys.argv[2])
    else:
        run(sys.argv[1], int(sys.argv[2]) if len(sys.argv) > 2 else 15)
