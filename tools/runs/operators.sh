#!/bin/bash
# perf/operators.py's listed cases: eager and replayed time of a pass, then a kernel trace of 13 passes of each (averages per launch)
set -eu
OUT=gpurun_out/${1:-operators}; mkdir -p $OUT
export TMPDIR=/tmp
timeout -k 10 200 python3 -u tools/operators_probe.py > $OUT/times.txt
: > $OUT/kernels.txt
for n in $(python3 -c 'import sys; sys.path.insert(0, "perf"); import operators as M; print(*[c["name"] for c in M.listed()])'); do
  timeout -s KILL 90 rocprofv3 --kernel-trace --stats -d /tmp/op_$n -o o --output-format csv -- python3 tools/operators_probe.py $n --passes 13 > $OUT/$n.log 2>&1 || [ -f /tmp/op_$n/o_kernel_stats.csv ]
  python3 - $n /tmp/op_$n/o_kernel_stats.csv >> $OUT/kernels.txt <<'PY'
import csv, re, sys
print(sys.argv[1])
for r in sorted(csv.DictReader(open(sys.argv[2])), key=lambda r: -float(r["TotalDurationNs"])):
    name = re.search(r"k_(diff_(fwd|few|join|delta|bwd|dlam)|sandwich_(fwd|bwd|cols)|adamw8_values|adamw8|sqnorm8)", r["Name"])
    if name:
        print("    %-18s %4d launches  %9.1f us" % (name.group(0), int(r["Calls"]), float(r["AverageNs"]) / 1e3))
PY
  tail -1 $OUT/kernels.txt
done
cat $OUT/times.txt
