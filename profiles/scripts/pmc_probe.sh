#!/bin/bash
# HBM-traffic passes (FETCH_SIZE, WRITE_SIZE: one rocprofv3 run each) over bench.py --probe-hbm-only -> probe_pmc.json.
#   bash profiles/scripts/pmc_probe.sh OUT_DIR   (writes OUT_DIR/probe_pmc.json, or nothing if a group is empty)
set -u
ROOT=$(cd "$(dirname "$0")/../.." && pwd)
mkdir -p "$1" || exit 1
DEST=$(cd "$1" && pwd)
export TMPDIR=/tmp
OUT=/tmp/pmc_probe
rm -rf $OUT; mkdir -p $OUT
for c in FETCH_SIZE WRITE_SIZE; do
  ( cd /tmp && timeout -k 10 400 rocprofv3 --pmc $c --kernel-trace --output-format csv -d $OUT/pmc_$c -- python3 "$ROOT/bench.py" --probe-hbm-only > "$DEST/pmc_probe_$c.log" 2>&1 )
  rc=$?; echo "$c rc $rc"; [ $rc -eq 0 ] || exit $rc
done
if python3 "$ROOT/profiles/scripts/pmc_summary.py" $OUT > "$DEST/probe_pmc.json.tmp"; then
  mv "$DEST/probe_pmc.json.tmp" "$DEST/probe_pmc.json"
else
  echo "pmc_summary failed: no probe_pmc.json written"; rm -f "$DEST/probe_pmc.json.tmp"; exit 1
fi
