#!/bin/bash
# r06: LU batch-split stagger A/B; the recipe's epoch time at HEAD (main.py train mode, batch 2, fresh run for two minutes)
set -o pipefail
mkdir -p gpurun_out
export TMPDIR=/tmp
timeout -k 10 600 python3 tools/lu_ab.py --libs i-admm-lstm_amd/iadmm/libiadmm.so tools/var_stagger1.so tools/var_stagger2.so \
  i-admm-lstm_amd/iadmm/libiadmm.so tools/var_stagger1.so tools/var_stagger2.so --batch 1024 --N 2000 > gpurun_out/r06e_lu_ab_stagger.txt 2>&1 || exit 1
grep lib gpurun_out/r06e_lu_ab_stagger.txt | cut -c1-300
bash tools/train_reference_recipe.sh r06t 2 || exit 1
grep -h "Epoch" gpurun_out/r06t_recipe/train.log | head -12
exit 0
