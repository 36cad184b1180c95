#!/bin/bash
# Builds libstylemesh_hip.so for gfx950 (cross-compiles without a GPU). Usage: build.sh [extra hipcc flags]
set -euo pipefail
cd "$(dirname "$0")"
OUT=../libstylemesh_hip.so
# packed fp32 instructions stay off: hipcc forms them by itself and some have given wrong results now and then
FLAGS="--offload-arch=gfx950 -Xclang -target-feature -Xclang -packed-fp32-ops -O3 -std=c++17 -munsafe-fp-atomics -fPIC -Wall -Wno-unused-function"
mkdir -p ../../build
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
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o $OUT "${objs[@]}" -L/opt/rocm/lib -lrccl
# host extensions that read torch's tensors: against its headers, with the host compiler
TORCH=$(python3 -c "import importlib.util, os; print(os.path.dirname(importlib.util.find_spec('torch').origin))")
PYINC=$(python3 -c "import sysconfig; print(sysconfig.get_paths()['include'])")
pids=()
for e in tensor_list fp8_host; do
  so=../_$e.so
  if [ ! -f $so ] || [ $e.cpp -nt $so ] || [ build.sh -nt $so ] || [ ../../include/stylemesh_hip.h -nt $so ]; then
    rm -f $so
    g++ -O2 -std=c++17 -fPIC -shared -Wall -I"$TORCH/include" -I"$PYINC" $e.cpp -o $so -L"$TORCH/lib" -ltorch_python -ltorch_cpu -lc10 \
      -L.. -l:libstylemesh_hip.so '-Wl,-rpath,$ORIGIN' &
    pids+=($!)
  fi
done
for p in "${pids[@]:-}"; do [ -z "$p" ] || wait "$p"; done
echo "built $(realpath $OUT)"
