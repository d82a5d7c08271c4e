#!/bin/sh
# Builds tests/cpp/test_epilogue_frontend against the in-tree library.
set -e
here="$(cd "$(dirname "$0")" && pwd)"
root="$(dirname "$(dirname "$here")")"
pkg="$root/rocm_wmma_gemm_b200"
cuda="${CUDA_HOME:-/usr/local/cuda}"
g++ -O2 -std=c++17 -Wall -I"$root/include" -I"$cuda/include" "$here/test_epilogue_frontend.cpp" -o "$here/test_epilogue_frontend" \
    -L"$pkg" -lrocm_wmma_gemm_sm100a -Wl,-rpath,"$pkg" -L"$cuda/lib64" -lcudart
echo "$here/test_epilogue_frontend"
