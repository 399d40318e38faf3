"""Kernel resource usage of libr3det_hip.so as compiled (VGPRs, LDS, occupancy, scratch), from the
`-Rpass-analysis=kernel-resource-usage` remarks the Makefile keeps next to each object (csrc/*.ru.txt).

    python tools/kernel_resources.py            table of every kernel (demangled)
    python tools/kernel_resources.py --check    exit 1 when a kernel outside the allow-list uses scratch memory

"0 scratch" was claimed and false for one kernel; this is the build-time check behind the claim
(tests/test_kernel_resources.py runs it in the CPU suite)."""
import glob
import os
import re
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "r3det-pytorch_amd", "csrc")
# kernels that may use scratch, with the reason (substring of the demangled name)
ALLOW_SCRATCH = {
    "fr_forward_points_kernel<5, 4>": "points = 5 sampler with four positions per thread (40 sample-point registers): 16 B / lane, "
                                      "not a shipped configuration (DESIGN 7)",
    # SURVEY 8f rank 4 (convex / polygon_geo helpers, not on the detector's path): Sutherland-Hodgman on per-lane vertex
    # arrays that are indexed dynamically, as the reference's own polygon code does (polygon_geo_cpu.cpp) -- they live in
    # scratch by construction
    "polygon_iou_kernel": "per-lane polygon vertex arrays, dynamically indexed (rank-4 helper op)",
    "poly_mask_kernel": "per-lane polygon vertex arrays, dynamically indexed (rank-4 helper op)",
    "poly_iou_mat_kernel": "per-lane polygon vertex arrays, dynamically indexed (rank-4 helper op)",
}


def demangle(names):
    try:
        for tool in ("/opt/rocm/lib/llvm/bin/llvm-cxxfilt", "c++filt"):
            try:
                out = subprocess.run([tool], input="\n".join(names), capture_output=True, text=True, check=True).stdout
                return out.split("\n")[:len(names)]
            except (OSError, subprocess.CalledProcessError):
                continue
        return names
    except Exception:  # noqa: BLE001
        return names


def parse(path):
    txt = open(path).read()
    rows = []
    for block in re.split(r"remark: [^\n]*Function Name: ", txt)[1:]:
        name = block.split("\n")[0].split(" [-Rpass")[0].strip()

        def g(key):
            m = re.search(re.escape(key) + r": (\d+)", block)
            return int(m.group(1)) if m else -1
        rows.append(dict(file=os.path.basename(path).replace(".ru.txt", ".hip"), name=name, vgpr=g("VGPRs"), agpr=g("AGPRs"),
                         sgpr=g("SGPRs"), scratch=g("ScratchSize [bytes/lane]"), occupancy=g("Occupancy [waves/SIMD]"),
                         lds=g("LDS Size [bytes/block]")))
    return rows


def collect(csrc=CSRC):
    rows = []
    for p in sorted(glob.glob(os.path.join(csrc, "*.ru.txt"))):
        rows += parse(p)
    names = demangle([r["name"] for r in rows])
    for r, d in zip(rows, names):
        r["demangled"] = re.sub(r"^void ", "", d).replace("(anonymous namespace)::", "")
        r["short"] = r["demangled"].split("(")[0]
    return rows


def offenders(rows):
    return [r for r in rows if r["scratch"] > 0 and not any(k in r["demangled"] for k in ALLOW_SCRATCH)]


def main():
    rows = collect() + collect(os.path.join(CSRC, "train"))
    if not rows:
        print("no csrc/*.ru.txt: build the library first (make -C r3det-pytorch_amd/csrc)")
        return 2
    if "--check" in sys.argv:
        bad = offenders(rows)
        for r in bad:
            print(f"SCRATCH {r['scratch']} B/lane: {r['file']}: {r['demangled'][:160]}")
        print(f"{len(rows)} kernels, {len(bad)} with scratch outside the allow-list")
        return 1 if bad else 0
    print(f"{'file':14s} {'VGPR':>4s} {'AGPR':>4s} {'LDS':>7s} {'occ':>3s} {'scr':>3s}  kernel")
    for r in sorted(rows, key=lambda r: (r["file"], r["short"])):
        print(f"{r['file']:14s} {r['vgpr']:4d} {r['agpr']:4d} {r['lds']:7d} {r['occupancy']:3d} {r['scratch']:3d}  {r['short'][:120]}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
