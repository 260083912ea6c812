#!/bin/sh
# builds tools/cbench/cbench against hallo_amd/libhallo_amd.so (run `python __graft_entry__.py` first)
set -e
cd "$(dirname "$0")"
# no packed fp32 instructions, as in the library (hallo_amd/build.py)
/opt/rocm/bin/hipcc --offload-arch=gfx950 -O2 -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops cbench.hip -o cbench -L../../hallo_amd -lhallo_amd -Wl,-rpath,'$ORIGIN/../../hallo_amd'
