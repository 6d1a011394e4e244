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
"$HIPCC" --offload-arch=gfx950 -O3 -std=c++17 -fPIC -shared \
    -Xclang -target-feature -Xclang -packed-fp32-ops \
    -Wall -Wno-unused-function \
    ${SAD_EXTRA_FLAGS:-} \
    -o "$OUT/libsad.so" "$HERE/sad_api.hip"
echo "built $OUT/libsad.so"
