#!/bin/bash
# The -DDGCN_DIAG profiling build of the library (phase clocks / ablation switches in k_fused; tools/stamp_fused.py).
# Not part of the product: built on demand (hipcc cross-compiles), selected with
# DGCN_LIB=distgcn_amd/libdgcn_diag.so.  One object per source, side by side, like __graft_entry__.build().
set -e
. "$(dirname "$0")/library_build.sh"
cd "$ROOT/distgcn_amd/csrc"
OBJ="$ROOT/build/obj_diag"
mkdir -p "$OBJ"
for s in $SRCS; do
  if [ ! -f "$OBJ/$s.o" ] || [ -n "$(find $s.hip *.h ../../include/dgcn.h ../../__graft_entry__.py -newer "$OBJ/$s.o" 2>/dev/null | head -1)" ]; then
    rm -f "$OBJ/$s.o"  # (a source that does not compile must not leave its old object to the link)
    "$HIPCC" $FLAGS -DDGCN_DIAG -c $s.hip -o "$OBJ/$s.o" &
  fi
done
wait
OBJS=""; for s in $SRCS; do OBJS="$OBJS $OBJ/$s.o"; done
"$HIPCC" $FLAGS -shared -Wl,-z,defs -o ../libdgcn_diag.so $OBJS
