#!/bin/bash
# Code-placement / scheduler sweep of fused.hip (the launch over 500 graphs of 200 vertices moves by 4 % with its code placement): one libdgcn_<tag>.so per
# flag set under build/sweep/, every other object taken from build/obj as built by __graft_entry__.build().  tools/ab_libs.py times them.
#   tools/placement_sweep.sh tag "flags" [tag "flags" ...]
set -e
. "$(dirname "$0")/library_build.sh"
cd "$ROOT/distgcn_amd/csrc"
mkdir -p "$ROOT/build/sweep"
OTHERS=""; for s in $SRCS; do [ "$s" = fused ] || OTHERS="$OTHERS $ROOT/build/obj/$s.o"; done
PIDS=""
while [ $# -ge 2 ]; do
  tag="$1"; flags="$2"; shift 2
  ( "$HIPCC" $FLAGS $flags -c fused.hip -o "$ROOT/build/sweep/fused_$tag.o" &&
    "$HIPCC" $FLAGS -shared -Wl,-z,defs -o "$ROOT/build/sweep/libdgcn_$tag.so" "$ROOT/build/sweep/fused_$tag.o" $OTHERS &&
    echo "built $tag: $flags" ) &
  PIDS="$PIDS $!"
done
for p in $PIDS; do wait $p; done
