#!/bin/bash
# Build a variant of the library with extra compile flags for ONE translation unit and link it beside the shipped objects:
#   tools/build_variant.sh w12 gemm_big -DFACT_EXPERIMENTAL_W12      -> tools/bin/libfact_w12.so
#   tools/build_variant.sh pm2 gemm_big -DBIG_DMA_IN_MFMA=2
# tools/bin/ is git-ignored but travels to the GPU box; A/B against the tree's library with tools/attic/ab_libs.sh, or load it
# with FACT_LIB=tools/bin/libfact_w12.so (mint_amd/_lib.py) for tools/bench_r2.py.
set -e
R=$(cd "$(dirname "$0")/.." && pwd)
CSRC=$R/mint_amd/csrc
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
if [ $# -lt 2 ]; then echo "usage: $0 NAME UNIT [FLAGS]" >&2; exit 2; fi
name=$1; unit=$2; shift 2
. <(grep -E '^(UNITS|FLAGS)=' "$CSRC/build.sh")
# (the variant is a test / bench build: engine.hip / probe.hip with the debug surface)
found=""
for f in $UNITS engine probe; do [ "$f" = "$unit" ] && found=1; done
if [ -z "$found" ]; then echo "unknown unit $unit (units: $UNITS engine probe)" >&2; exit 2; fi
TMP=$(mktemp -d)
trap 'rm -rf "$TMP"' EXIT
mkdir -p "$R/tools/bin"
fresh=1
objs=""
for f in $UNITS engine_dbg probe_dbg; do
  o=$R/mint_amd/lib/obj/$f.o
  if [ ! -f "$o" ] || [ "$CSRC/${f%_dbg}.hip" -nt "$o" ] || [ -n "$(find "$CSRC" "$R/include" -name '*.h' -newer "$o")" ]; then fresh=""; fi
  if [ "${f%_dbg}" = "$unit" ]; then o=$TMP/$unit.o; fi
  objs="$objs $o"
done
[ -n "$fresh" ] || "$CSRC/build.sh"
$HIPCC $FLAGS -DFACT_DEBUG_ABI "$@" -c "$CSRC/$unit.hip" -o "$TMP/$unit.o"
$HIPCC --offload-arch=gfx950 -shared -fPIC -Wl,-z,defs -Wl,--version-script="$CSRC/exports.map" -o "$R/tools/bin/libfact_$name.so" $objs
echo "built tools/bin/libfact_$name.so"
