#!/bin/bash
# r06: panels' staged loads double-buffered for real (inline-asm stage reads) -- LU tests, A/B against
# the previous build; recipe epoch time with cached synthetic instances
set -o pipefail
mkdir -p gpurun_out
export TMPDIR=/tmp
timeout -k 10 900 python3 -u -m pytest -x -q --timeout 600 --timeout-method thread \
  tests/test_stage2_gpu.py tests/test_abi_concurrency_gpu.py tests/test_lu_hbm_gpu.py > gpurun_out/r06f_lu_tests.log 2>&1 || { tail -n 40 gpurun_out/r06f_lu_tests.log; exit 1; }
tail -n 2 gpurun_out/r06f_lu_tests.log
timeout -k 10 600 python3 tools/lu_ab.py --libs tools/var_lu_before.so i-admm-lstm_amd/iadmm/libiadmm.so \
  tools/var_lu_before.so i-admm-lstm_amd/iadmm/libiadmm.so --batch 1024 --N 2000 > gpurun_out/r06f_lu_ab_panel.txt 2>&1 || exit 2
grep '^{' gpurun_out/r06f_lu_ab_panel.txt | cut -c1-200
bash tools/train_reference_recipe.sh r06u 3 || exit 3
grep -h "Epoch" gpurun_out/r06u_recipe/train.log | head -12
exit 0
