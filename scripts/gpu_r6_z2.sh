#!/bin/bash
# round 6, call 37: GroupNorm per-shape sweep of the sample groups (experiments build), the as-shipped step: two-launch | one-launch, tests, the headline
cd $GRAFT_REPO_ROOT; mkdir -p gpurun_out
timeout 600 python -u scripts/exp_gn_groups.py 2>&1 | grep -v "Warning\|amdgpu.ids" | tee gpurun_out/r06_z2_gn_groups.txt
timeout 600 python -m pytest tests/test_stem_kernels_gpu.py -q -m gpu 2>&1 | grep -v Warning | tail -6 | cut -c1-300 | tee gpurun_out/r06_z2_tests.txt
for mode in two fused fused two; do
  if [ $mode = fused ]; then extra="--gn-fused"; else extra=""; fi
  timeout 240 python bench.py --native-yaml --no-cpu-baseline --steps 6 --warmup 3 $extra 2>/dev/null | tee gpurun_out/r06_z2_bench_native_$mode.json | python -c "import sys,json; d=json.loads(sys.stdin.read()); print('$mode', round(d['value'],1), 'seg/s', round(d['ms_per_step'],1), 'ms', 'loss', d['config'].get('final_loss'))"
done
timeout 900 python -m pytest tests/test_kernels_gpu.py tests/test_native_yaml_gpu.py tests/test_stem_model_gpu.py -q -m gpu -k "attention or native or shipped or stem" 2>&1 | grep -v Warning | tail -4 | cut -c1-300 | tee -a gpurun_out/r06_z2_tests.txt
timeout 300 python bench.py --no-cpu-baseline 2>/dev/null | tee gpurun_out/r06_z2_bench.json | python -c "import sys,json; d=json.loads(sys.stdin.read()); print('headline', round(d['value'],1), 'seg/s', round(d['ms_per_step'],1), 'ms')"
