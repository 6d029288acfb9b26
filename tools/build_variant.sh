#!/bin/bash
# Development aid: builds build_variants/libomnihip_<name>.so with extra compiler flags for ONE kernel file
# (flags and object list are the Makefile's, all other objects the in-tree ones).
# usage: [HIPCC=compiler] [OUT=folder] tools/build_variant.sh <name> <file.hip> <flags...>
set -e
ROOT="$(cd "$(dirname "$0")/.." && pwd)"
NAME="$1"; FILE="$2"; shift 2
HIPCC="${HIPCC:-/opt/rocm/bin/hipcc}"; OUT="${OUT:-$ROOT/build_variants}"
mkdir -p "$OUT"
cd "$ROOT/omni-video_amd/csrc"
BASE="${FILE%.hip}"
"$HIPCC" $(make -s "flags-$BASE") "$@" -c "$FILE" -o "$OUT/${BASE}_${NAME}.o"
OBJS=""
for o in $(make -s objects); do
  if [ "$o" = "$BASE.o" ]; then OBJS="$OBJS $OUT/${BASE}_${NAME}.o"; else OBJS="$OBJS $o"; fi
done
"$HIPCC" --offload-arch=gfx950 -shared -fPIC -o "$OUT/libomnihip_${NAME}.so" $OBJS
echo "$OUT/libomnihip_${NAME}.so"
