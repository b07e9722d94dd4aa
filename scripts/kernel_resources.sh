#!/bin/bash
# Kernel resource record: VGPRs / AGPRs / scratch / LDS / occupancy of every kernel of the shipped build, from the compiler's own
# remarks (hipcc -Rpass-analysis=kernel-resource-usage, same flags as friedrich_amd/build.py).  Runs without a GPU.
#   scripts/kernel_resources.sh [out.txt]      (default profiles/r06/kernel_resources.txt; also writes kernel_resources.sources.json next
#   to it: the content hashes of friedrich_amd/csrc the record was made from -- tests/test_profiles_fresh.py holds it to the tree)
set -e
cd "$(dirname "$0")/.."
OUT=${1:-profiles/r06/kernel_resources.txt}
mkdir -p "$(dirname "$OUT")"
TMP=$(mktemp -d)
{
  echo "# kernel | VGPRs | AGPRs | scratch B/lane | LDS B (static) | occupancy waves/SIMD | SGPRs | VGPRs spilled | SGPRs spilled"
  echo "# hipcc $(/opt/rocm/bin/hipcc --version | grep -m1 'HIP version'); flags: --offload-arch=gfx950 -O3 -packed-fp32-ops (friedrich_amd/build.py); generated by scripts/kernel_resources.sh"
  for f in friedrich_amd/csrc/*.hip; do  # the compilations run side by side, the records are read in the order of the files
    /opt/rocm/bin/hipcc -x hip --offload-arch=gfx950 -O3 -std=c++17 -fPIC -fno-gpu-rdc -Xclang -target-feature -Xclang -packed-fp32-ops -Iinclude -Ifriedrich_amd/csrc -I/opt/rocm/include \
      -Rpass-analysis=kernel-resource-usage -c "$f" -o "$TMP/$(basename "$f").o" 2> "$TMP/$(basename "$f").txt" && touch "$TMP/$(basename "$f").ok" &
  done
  wait
  for f in friedrich_amd/csrc/*.hip; do
    R="$TMP/$(basename "$f").txt"
    [ -e "$TMP/$(basename "$f").ok" ] || { cat "$R" >&2; exit 1; }
    python3 - "$R" "$(basename "$f")" <<'PY'
import re, sys
txt = open(sys.argv[1]).read()
cur = None
rows = {}
for line in txt.splitlines():
    m = re.search(r"remark: .*Function Name: (\S+)", line)
    if m:
        cur = m.group(1); rows[cur] = {}
        continue
    m = re.search(r"remark: .*?\s{2,}([A-Za-z ]+(?:\[[^\]]*\])?[A-Za-z /]*): (\S+)", line)
    if m and cur:
        rows[cur][m.group(1).strip()] = m.group(2)
import subprocess
for name, r in rows.items():
    dem = subprocess.run(["c++filt", name], capture_output=True, text=True).stdout.strip()
    dem = re.sub(r"\(.*", "", dem)
    print(f"{sys.argv[2]}: {dem} | {r.get('VGPRs','?')} | {r.get('AGPRs','?')} | {r.get('ScratchSize [bytes/lane]','?')} | "
          f"{r.get('LDS Size [bytes/block]','?')} | {r.get('Occupancy [waves/SIMD]','?')} | {r.get('TotalSGPRs','?')} | {r.get('VGPRs Spill','?')} | {r.get('SGPRs Spill','?')}")
PY
  done
} > "$OUT"
rm -rf "$TMP"
python3 scripts/source_hash.py > "${OUT%.txt}.sources.json"
echo "wrote $OUT ($(grep -c '|' "$OUT") lines)"
