#!/bin/bash
# Build libsad.so for gfx950 (MI355X), in-tree.  hipcc cross-compiles without a GPU.
set -euo pipefail
HERE="$(cd "$(dirname "${BASH_SOURCE[0]}")" && pwd)"
OUT="$HERE/../_native"
mkdir -p "$OUT"
HIPCC="${HIPCC:-/opt/rocm/bin/hipcc}"
# No packed FP32 instructions (v_pk_add/mul/fma_f32): some of their forms have given wrong results now and then on
# gfx950, with no error, and hipcc -O3 makes them from ordinary float code by itself.  The host pass warns that it
# does not know the feature; that warning is harmless.
# SAD_OUT: another name for the library (A/B builds).
LIB="${SAD_OUT:-$OUT/libsad.so}"
OBJ="$(mktemp -d)"
trap 'rm -r "$OBJ"' EXIT
pids=()
for src in sad_api scan_api; do
    "$HIPCC" --offload-arch=gfx950 -O3 -std=c++17 -fPIC -c \
        -Xclang -target-feature -Xclang -packed-fp32-ops \
        -Wall -Wno-unused-function \
        ${SAD_EXTRA_FLAGS:-} \
        -o "$OBJ/$src.o" "$HERE/$src.hip" &
    pids+=($!)
done
for pid in "${pids[@]}"; do wait "$pid"; done
"$HIPCC" --offload-arch=gfx950 -shared -fPIC -o "$LIB" "$OBJ/sad_api.o" "$OBJ/scan_api.o"
echo "built $LIB"
