#!/bin/bash
# Builds libstylemesh_hip.so for gfx950 (cross-compiles without a GPU). Usage: build.sh [extra hipcc flags]
set -euo pipefail
cd "$(dirname "$0")"
OUT=../libstylemesh_hip.so
# packed fp32 instructions stay off: hipcc forms them by itself and some have given wrong results now and then
FLAGS="--offload-arch=gfx950 -Xclang -target-feature -Xclang -packed-fp32-ops -O3 -std=c++17 -munsafe-fp-atomics -fPIC -Wall -Wno-unused-function"
mkdir -p ../../build
# the host extension that reads lists of tensors: against torch's headers, with the host compiler
EXT=../_tensor_list.so
if [ ! -f $EXT ] || [ tensor_list.cpp -nt $EXT ] || [ build.sh -nt $EXT ]; then
  rm -f $EXT
  TORCH=$(python3 -c "import importlib.util, os; print(os.path.dirname(importlib.util.find_spec('torch').origin))")
  g++ -O2 -std=c++17 -fPIC -shared -Wall -I"$TORCH/include" -I"$(python3 -c "import sysconfig; print(sysconfig.get_paths()['include'])")" \
    tensor_list.cpp -o $EXT -L"$TORCH/lib" -ltorch_python -ltorch_cpu -lc10 &
  EXT_PID=$!
fi
objs=()
pids=()
for f in conv texture gram prep comm eval raster scatter_plan exchange replay fp8 gradnorm; do
  o=../../build/$f.o
  stale=0
  for dep in "$f.hip" *.h ../../include/stylemesh_hip.h; do
    if [ ! -f "$o" ] || [ "$dep" -nt "$o" ]; then stale=1; fi
  done
  if [ $stale = 1 ]; then
    rm -f "$o"
    /opt/rocm/bin/hipcc $FLAGS "$@" -c $f.hip -o $o &
    pids+=($!)
  fi
  objs+=("$o")
done
for p in "${pids[@]:-}"; do [ -z "$p" ] || wait "$p"; done   # (a failed compile ends the build here)
[ -z "${EXT_PID:-}" ] || wait "$EXT_PID"
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o $OUT "${objs[@]}" -L/opt/rocm/lib -lrccl
echo "built $(realpath $OUT)"
