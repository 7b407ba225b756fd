#!/bin/bash
# Kernel times and vector-unit counters of the sequence operators, case by case (run on the GPU from the repository root).
# Two rocprofv3 runs a case, in a folder of its own under $OUT; tools/seq_cases.py --summary $OUT makes the table of them.
R=$(pwd); OUT=$R/gpurun_out/seq; mkdir -p "$OUT"
python3 tools/seq_cases.py --list > "$OUT/cases.txt" || exit 1
cd /tmp; export TMPDIR=/tmp
while read -r name; do
  d="$OUT/$(echo "$name" | sed 's/[^A-Za-z0-9_][^A-Za-z0-9_]*/_/g')"
  timeout -k 10 60 rocprofv3 --kernel-trace --stats --mangled-kernels --output-format csv -d "$d/time" -- python3 $R/tools/seq_cases.py "$name" 15 > "$d.log" 2>&1 < /dev/null || { echo "$name: trace failed"; tail -n 5 "$d.log"; exit 1; }
  timeout -s KILL 60 rocprofv3 --mangled-kernels --output-format csv --pmc SQ_INSTS_VALU SQ_ACTIVE_INST_VALU SQ_BUSY_CU_CYCLES SQ_WAVES -d "$d/counters" -- python3 $R/tools/seq_cases.py "$name" 3 > "$d.pmc.log" 2>&1 < /dev/null || { echo "$name: counters failed"; tail -n 5 "$d.pmc.log"; exit 1; }
  echo "$name"
done < "$OUT/cases.txt"
