#!/bin/bash
# Build libt2mi.so for gfx950 (MI355X).  Cross-compiles without a GPU.  Arguments go to every compile step.
# Packed fp32 instructions are switched off for the device code; hipcc's host pass says that it does not know the feature.
set -euo pipefail
cd "$(dirname "$0")"
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
FLAGS=(--offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wall -Wno-unused-function -Wno-unused-value
       -Xclang -target-feature -Xclang -packed-fp32-ops)
UNITS=(t2mi recurrence adamw)
mkdir -p build
pids=()
for u in "${UNITS[@]}"; do
    $HIPCC "${FLAGS[@]}" -c "$u.hip" -o "build/$u.o" "$@" &
    pids+=($!)
done
for p in "${pids[@]}"; do wait "$p"; done
objs=("${UNITS[@]/#/build/}")
$HIPCC --offload-arch=gfx950 -shared -fPIC -o ../libt2mi.so "${objs[@]/%/.o}"
echo "built $(cd .. && pwd)/libt2mi.so"
