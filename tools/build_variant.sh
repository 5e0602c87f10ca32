#!/bin/bash
# A/B builds: tools/build_variant.sh <name> [-DFLAG=1 ...]  ->  tools/ab/<name>/libmwhip.so (select with MW_LIB_PATH)
# Sources and flags are the library's own (manual-whisper_amd/build.py); HIPCC: another compiler driver.
set -e
name=$1; shift
root=$(cd "$(dirname "$0")/.." && pwd)
out=$root/tools/ab/$name
hipcc=${HIPCC:-/opt/rocm/bin/hipcc}
mkdir -p $out
cd $root/manual-whisper_amd
recipe=$(python3 -c 'import build
for s in build.SOURCES: print(s, *build.FLAGS, *build.EXTRA_FLAGS.get(s, []))')
cd csrc
pids=()
objects=()
while read -r src flags; do
  objects+=($out/${src%.hip}.o)
  $hipcc $flags "$@" -c $src -o $out/${src%.hip}.o &
  pids+=($!)
done <<< "$recipe"
for p in "${pids[@]}"; do wait $p; done
$hipcc -shared -fPIC --offload-arch=gfx950 -o $out/libmwhip.so "${objects[@]}"
rm -f "${objects[@]}"
echo $out/libmwhip.so
