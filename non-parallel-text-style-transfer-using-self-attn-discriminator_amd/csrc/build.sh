#!/bin/bash
# Build libsad.so for gfx950 (MI355X), in-tree.  hipcc cross-compiles without a GPU.
set -euo pipefail
HERE="$(cd "$(dirname "${BASH_SOURCE[0]}")" && pwd)"
OUT="$HERE/../_native"
mkdir -p "$OUT"
HIPCC="${HIPCC:-/opt/rocm/bin/hipcc}"
# No packed FP32 instructions (v_pk_add/mul/fma_f32), which hipcc -O3 makes from ordinary float code by itself: a precaution, as
# a silent wrong result of some of their forms would not show in tests.  The batch-1024 training step takes 1.19 ms with
# and without them.  The host pass warns that it does not know the feature; that warning is harmless.
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
# Autograd nodes for torch's dispatcher (plain C++ against torch's headers; not built for a renamed library)
if [ -z "${SAD_OUT:-}" ]; then
    TORCH="$(python3 -c 'import importlib.util, os; print(os.path.dirname(importlib.util.find_spec("torch").origin))')"
    "${CXX:-g++}" -O2 -std=c++17 -fPIC -shared -Wall -D__HIP_PLATFORM_AMD__=1 -DUSE_ROCM=1 \
        -I"$TORCH/include" -I"$TORCH/include/torch/csrc/api/include" -I"${ROCM_PATH:-/opt/rocm}/include" \
        -o "$OUT/libsad_torch.so" "$HERE/torch_ops.cpp" \
        -L"$TORCH/lib" -ltorch -ltorch_cpu -ltorch_hip -lc10 -lc10_hip &
    pids+=($!)
fi
for pid in "${pids[@]}"; do wait "$pid"; done
"$HIPCC" --offload-arch=gfx950 -shared -fPIC -o "$LIB" "$OBJ/sad_api.o" "$OBJ/scan_api.o"
echo "built $LIB"
