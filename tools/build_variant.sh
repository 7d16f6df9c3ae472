#!/bin/bash
# usage: tools/build_variant.sh <name> <extra hipcc flags...>   -> transformer_vae_amd/variants/libtvae_<name>.so
# (A/B builds of single constants; the GPU tools load one with TVAE_LIB_OVERRIDE)
set -e
NAME=$1; shift
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
cd "$(dirname "$0")/../transformer_vae_amd/csrc"
OUT=../variants; mkdir -p $OUT/obj_$NAME
for f in $(sed -n 's/^SRCS = //p' Makefile); do
  f=${f%.hip}
  # only the files the flags can touch are recompiled, by the Makefile's own line; the rest are the product objects
  if grep -q "TVAE_" <<< "$*" && grep -qE "$(echo "$*" | grep -oE 'TVAE_[A-Z_0-9]+' | paste -sd'|')" $f.hip; then
    LINE=$(make -s -n -B HIPCC="$HIPCC" $f.o | grep -- "-c $f.hip")
    ${LINE% -o *} "$@" -o $OUT/obj_$NAME/$f.o &
  else
    cp $f.o $OUT/obj_$NAME/$f.o
  fi
done
wait
"$HIPCC" -shared -fPIC --offload-arch=gfx950 $OUT/obj_$NAME/*.o -o $OUT/libtvae_$NAME.so
rm -rf $OUT/obj_$NAME
ls -la $OUT/libtvae_$NAME.so
