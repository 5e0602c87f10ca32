#!/bin/bash
# builds tools/gemv_bench from the library's kernel sources (decode projections + the LayerNorm they call), with the library's
# device flags (manual-whisper_amd/build.py); HIPCC: another compiler driver
set -e
cd "$(dirname "$0")/.."
flags=$(cd manual-whisper_amd && python3 -c 'import build; print(*build.ARCH_FLAGS)')
${HIPCC:-/opt/rocm/bin/hipcc} -O3 -std=c++17 $flags -Imanual-whisper_amd/csrc "$@" tools/gemv_bench.hip manual-whisper_amd/csrc/kernels_dec.hip manual-whisper_amd/csrc/kernels_enc.hip -o tools/gemv_bench
