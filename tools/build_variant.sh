#!/bin/bash
# Build libiadmm.so from an alternative copy of the sources (variant studies; load it with
# IADMM_LIB_PATH=<out.so>), by the library's own Makefile: its flags and its list of sources.
# Usage: [EXTRA="-DNAME=VAL ..."] bash tools/build_variant.sh <dir with csrc/> <out.so>
set -euo pipefail
src=$(realpath "$1"); out=$(realpath -m "$2")
obj=$(mktemp -d /tmp/var_obj_XXXX)
make -s -j8 -C "$(dirname "$0")/../i-admm-lstm_amd" CSRC="$src/csrc" BLD="$obj" OUT="$out" EXTRA="${EXTRA:-}" "$out"
rm -rf "$obj"
echo "built $out"
