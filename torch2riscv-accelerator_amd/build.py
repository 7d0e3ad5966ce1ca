"""Builds libt2r.so (the C-ABI of include/t2r.h) for gfx950 with hipcc, in-tree.

    python -m t2r_amd.build            (or __graft_entry__.build())

Flags: -O3, -ffp-contract=off (no fused multiply-add: every fp32 step rounds once, as the
reference's vector engine), the default f32 denormal mode (IEEE, as NumPy float32), and packed
fp32 instructions switched off.
"""
import os
import subprocess
import sys
import tempfile
import time

HERE = os.path.dirname(os.path.abspath(__file__))
SRCS = [os.path.join(HERE, "csrc", n) for n in ("t2r.hip", "t2r_block.hip")]
LIB = os.path.join(HERE, "libt2r.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = os.environ.get("T2R_ARCH", "gfx950")
FLAGS = ["-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}", "-ffp-contract=off",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-unused-result"]


def build(verbose=False):
    """Compiles the sources side by side, each a unit with device code of its own, and links them into LIB."""
    t0 = time.time()
    noise = "is not a recognized feature for this target"
    err = ""

    def run(cmds):
        nonlocal err
        ps = [subprocess.Popen(c, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for c in cmds]
        outs = [p.communicate()[0] for p in ps]
        for c, p, out in zip(cmds, ps, outs):
            err += "".join(l + "\n" for l in out.splitlines() if noise not in l)
            if p.returncode != 0:
                raise RuntimeError(f"hipcc failed ({p.returncode}):\n{' '.join(c)}\n{err}")

    with tempfile.TemporaryDirectory() as d:
        objs = [os.path.join(d, os.path.basename(s) + ".o") for s in SRCS]
        run([[HIPCC, *FLAGS, "-c", s, "-o", o] for s, o in zip(SRCS, objs)])
        run([[HIPCC, "-shared", "-fPIC", f"--offload-arch={ARCH}", *objs, "-o", LIB + ".tmp"]])
    os.replace(LIB + ".tmp", LIB)
    if verbose:
        print(f"built {LIB} in {time.time() - t0:.1f} s" + (f"\n{err}" if err.strip() else ""), flush=True)
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
