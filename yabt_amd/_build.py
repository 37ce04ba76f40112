"""Compile the gfx950 HIP library in-tree (yabt_amd/_lib/libyabt_hip.so).

The library is plain C-ABI (include/yabt_hip.h); it links only the HIP runtime.
Each source is compiled to its own object in parallel, then linked.
"""

from __future__ import annotations

import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OUT_DIR = os.path.join(HERE, "_lib")
OBJ_DIR = os.path.join(OUT_DIR, "obj")
LIB = os.path.join(OUT_DIR, "libyabt_hip.so")
SOURCES = ["grow.hip", "grow_batch.hip", "grow_level.hip", "grow_ref.hip", "ops.hip", "leaf.hip", "slots.hip",
           "boost.hip", "binner.hip", "noalloc.hip", "norm.hip", "route.hip",
           "experts.hip"]
ARCH = "gfx950"

# -ffp-contract=off: no fused multiply-add may change a rounding that the
#   fixed-point contract shares with the CPU oracle.
# -packed-fp32-ops off: packed fp32 VALU forms are avoided on this target.
#   hipcc forwards -Xclang options to the host and the device pass alike (its
#   -Xarch_device form refuses options that take an argument), so the host
#   pass reports the feature as unknown and ignores it; that one line is
#   dropped from the build output below.
FLAGS = [
    "-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}",
    "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-result",
]
_HOST_PASS_NOTE = "'-packed-fp32-ops' is not a recognized feature for this target"


def hipcc() -> str:
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    return "hipcc"


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    p = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    text = "\n".join(line for line in p.stdout.splitlines() if _HOST_PASS_NOTE not in line)
    if text.strip():
        print(text, flush=True)
    if p.returncode != 0:
        raise subprocess.CalledProcessError(p.returncode, cmd, output=text)


def build(verbose: bool = False, jobs: int | None = None) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    objs = []
    cmds = []
    for s in SOURCES:
        obj = os.path.join(OBJ_DIR, os.path.splitext(s)[0] + ".o")
        objs.append(obj)
        cmds.append([hipcc(), *FLAGS, "-I", CSRC, "-I", INCLUDE, "-c", os.path.join(CSRC, s), "-o", obj])
    jobs = jobs or min(len(cmds), max(1, min(os.cpu_count() or 1, 16)))
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        for f in [ex.submit(_run, c, verbose) for c in cmds]:
            f.result()
    tmp = LIB + ".tmp"
    _run([hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp], verbose)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
