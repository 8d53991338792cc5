#!/bin/bash
# Times and counters of the layer norm and AdamW (from the repository root, on a machine with the GPU): profile_operators.sh <output folder>
# Each counter in a run of its own, kernel trace only.
mkdir -p "$1"; R=$PWD; OUT=$(cd "$1" && pwd)
timeout -k 10 120 python3 tools/bench_operators.py > $OUT/cases.log 2>&1 || exit 1
timeout -k 10 180 python3 tools/bench_operators.py --kernels > $OUT/kernels.log 2>&1 || exit 1
cd /tmp && export TMPDIR=/tmp
timeout -s KILL 120 rocprofv3 --kernel-trace --output-format csv -d $OUT -o time -- python3 $R/tools/bench_operators.py --passes 12 > $OUT/time.log 2>&1 || exit 1
timeout -s KILL 120 rocprofv3 --kernel-trace --pmc FETCH_SIZE --output-format csv -d $OUT -o fetch -- python3 $R/tools/bench_operators.py --passes 12 > $OUT/fetch.log 2>&1 || exit 1
timeout -s KILL 120 rocprofv3 --kernel-trace --pmc WRITE_SIZE --output-format csv -d $OUT -o write -- python3 $R/tools/bench_operators.py --passes 12 > $OUT/write.log 2>&1 || exit 1
python3 $R/tools/bench_operators.py --table $OUT > $OUT/operators_kernels.csv
