#!/bin/bash
# Builds libmtk_hip.so for gfx950 in-tree (hipcc cross-compiles without a GPU).
set -euo pipefail
cd "$(dirname "$0")"
INC=../../include
# no packed fp32 instructions: some of their forms have given wrong results on this hardware (the host pass warns that it does not know
# the feature)
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -I$INC -I. -Wall -Wno-unused-function -Xclang -target-feature -Xclang -packed-fp32-ops"
mkdir -p _build
pids=()
# the diffusion kernels mirror eager fp32 op sequences: no fused multiply-add contraction
hipcc $FLAGS -ffp-contract=off -c mtk_diffusion.hip -o _build/mtk_diffusion.o & pids+=($!)
hipcc $FLAGS -ffp-contract=off -c mtk_tf.hip -o _build/mtk_tf.o & pids+=($!)
hipcc $FLAGS -ffp-contract=off -c mtk_train.hip -o _build/mtk_train.o & pids+=($!)
hipcc $FLAGS -c mtk_capi.hip -o _build/mtk_capi.o & pids+=($!)
hipcc $FLAGS -c mtk_mlp_f32.hip -o _build/mtk_mlp_f32.o & pids+=($!)
hipcc $FLAGS -c mtk_mlp_bf16.hip -o _build/mtk_mlp_bf16.o & pids+=($!)
hipcc $FLAGS -c mtk_mlp_bf16_layered.hip -o _build/mtk_mlp_bf16_layered.o & pids+=($!)
hipcc $FLAGS -ffp-contract=off -c mtk_transform.hip -o _build/mtk_transform.o & pids+=($!)
hipcc $FLAGS -c mtk_rows.hip -o _build/mtk_rows.o & pids+=($!)
hipcc $FLAGS -c mtk_adapter.hip -o _build/mtk_adapter.o & pids+=($!)
# AdamW: each product and sum rounded by itself, so the update is the one torch's elementary operations give
hipcc $FLAGS -ffp-contract=off -c mtk_optim.hip -o _build/mtk_optim.o & pids+=($!)
# torch's side of the small entry points (host code only; the library's functions reach it by address)
read -r TORCH PYINC CXX11 < <(python3 -c "import os, sysconfig, torch; print(os.path.dirname(torch.__file__), sysconfig.get_paths()['include'], int(torch._C._GLIBCXX_USE_CXX11_ABI))")
g++ -O2 -std=c++17 -fPIC -shared -Wall -D_GLIBCXX_USE_CXX11_ABI=$CXX11 -D__HIP_PLATFORM_AMD__=1 -DUSE_ROCM -I$INC -isystem $TORCH/include -isystem $TORCH/include/torch/csrc/api/include -isystem $PYINC -isystem /opt/rocm/include \
    mtk_torch.cpp -o ../_mtk_torch.so -L$TORCH/lib -lc10 -lc10_hip -ltorch_cpu -ltorch_python & pids+=($!)
for p in "${pids[@]}"; do wait "$p"; done
hipcc --offload-arch=gfx950 -shared -fPIC _build/*.o -o ../libmtk_hip.so
echo "built $(cd .. && pwd)/libmtk_hip.so"
