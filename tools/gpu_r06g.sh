#!/bin/bash
# r06: the LU graph-capture tests with the captured look-ahead / split; sched_bwd batch loads
set -o pipefail
mkdir -p gpurun_out
export TMPDIR=/tmp
timeout -k 10 900 python3 -u -m pytest -x -v --timeout 600 --timeout-method thread \
  tests/test_abi_concurrency_gpu.py tests/test_train_gpu.py tests/test_window_grads_gpu.py > gpurun_out/r06g_tests.log 2>&1
rc=$?
grep -E "PASS|FAIL|ERROR|passed|failed" gpurun_out/r06g_tests.log | tail -30
exit $rc
