#!/bin/bash
# Build a kernel variant of libtsdiff_hip.so for A/B timing:   tools/build_variant.sh NAME "-DFLAG ..." [TU ...]
# Recompiles the listed translation units (default: kernels_combo.hip) as the Makefile does, with the extra flags behind its own,
# takes the other objects from tsdiff_amd/csrc (run `make -C tsdiff_amd/csrc` first) and links tools/bin/lib_NAME.so (git-ignored).
set -e
NAME=$1; FLAGS=$2; shift 2 || true
TUS=${@:-kernels_combo.hip}
ROOT=$(cd $(dirname $0)/.. && pwd)
SRC=$ROOT/tsdiff_amd/csrc
OUT=$ROOT/tools/bin/obj_$NAME
mkdir -p $OUT
MAKE="make -C $SRC --no-print-directory -n -B"
LINK=$($MAKE ../libtsdiff_hip.so | grep -- "-shared" | tail -1)  # hipcc .. a.o b.o .. -o ../libtsdiff_hip.so
LINK=${LINK/ -o ..\/libtsdiff_hip.so/ -o $ROOT/tools/bin/lib_$NAME.so}
PIDS=""
for tu in $TUS; do
  f=${tu%.hip}
  CMD=$($MAKE $f.o | grep -- " -c $f.hip ")
  (cd $SRC && ${CMD/ -o $f.o/ $FLAGS -o $OUT/$f.o}) &
  PIDS="$PIDS $!"
  LINK=${LINK/ $f.o / $OUT/$f.o }
done
for p in $PIDS; do wait $p; done
(cd $SRC && $LINK)
echo built tools/bin/lib_$NAME.so
