"""Build libinet_nr.so (the engines' C-ABI HIP library) and libinet_policy.so (the policy operators') in-tree for gfx950.

    python isaac-net_amd/build.py            # or __graft_entry__.build(): both
    python isaac-net_amd/build.py --policy   # libinet_policy.so alone
    python isaac-net_amd/build.py --phase-clocks   # libinet_nr_phase.so: the step kernels with per-phase clocks

The step-kernel instantiations are split over translation units (one per subband count) that compile in parallel
and link into one shared library. Flags: -ffp-contract=off keeps every float multiply and add separately rounded
(the op order mirrors the reference's torch expressions), and packed FP32 instructions are disabled for this target.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libinet_nr.so")
PHASE_LIB = os.path.join(HERE, "libinet_nr_phase.so")
# (the units with the most and the largest instantiations first: the pool's last unit sets the build's wall time)
UNITS = [f"nr_step_mc{c}.hip" for c in (7, 6, 5, 4)] + \
        ["nr_step_s13.hip", "nr_step_w2.hip", "nr_step_w4.hip", "nr_step_mc.hip", "nr_step_mc2.hip", "nr_step_s8.hip"] + \
        [f"nr_step_s{s}.hip" for s in (10, 11, 12, 14, 16, 17, 18)] + ["inet_nr.hip", "wifi.hip"]
# the policy operators: a library of their own, so that either is rebuilt without the other
POLICY_CSRC = os.path.join(CSRC, "policy")
POLICY_LIB = os.path.join(HERE, "libinet_policy.so")
POLICY_HEADER = "inet_policy.h"
POLICY_UNITS = ["delta_backward.hip", "delta_split.hip", "delta_forward.hip", "delta_step.hip", "ffn.hip", "norm.hip", "policy.hip"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wall", "-Wno-unused-function"]
# (the policy operators mirror no other implementation's rounding: multiplies and adds may fuse)
POLICY_FLAGS = [f for f in FLAGS if f != "-ffp-contract=off"]


def _hash(files):
    import hashlib
    h = hashlib.sha256()
    for f in sorted(files) + [os.path.abspath(__file__)]:
        h.update(os.path.basename(f).encode())
        with open(f, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()[:16]


def source_hash():
    """SHA-256 over libinet_nr.so's sources (csrc/*.h, csrc/*.hip, include/*.h, this file), in name order."""
    import glob
    return _hash(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip")) +
                 [f for f in glob.glob(os.path.join(HERE, "..", "include", "*.h"))
                  if os.path.basename(f) != POLICY_HEADER])


def policy_hash():
    """The same over libinet_policy.so's (csrc/policy/, include/inet_policy.h, this file)."""
    import glob
    return _hash(glob.glob(os.path.join(POLICY_CSRC, "*.h")) + glob.glob(os.path.join(POLICY_CSRC, "*.hip")) +
                 [os.path.join(HERE, "..", "include", POLICY_HEADER)])


def _compile(units, csrc, obj_dir, flags, src, lib, verbose):
    os.makedirs(obj_dir, exist_ok=True)

    def compile_unit(u):
        obj = os.path.join(obj_dir, u.replace(".hip", ".o"))
        cmd = [HIPCC, *flags, f'-DINET_SRC_HASH="{src}"', "-c", "-o", obj, os.path.join(csrc, u)]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        return obj

    with cf.ThreadPoolExecutor(min(len(units), os.cpu_count() or 8)) as ex:
        objs = list(ex.map(compile_unit, units))
    tmp = lib + ".tmp"
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, lib)
    return lib


def build_policy(verbose=False):
    """Compile and link libinet_policy.so."""
    return _compile(POLICY_UNITS, POLICY_CSRC, os.path.join(HERE, "_build", "policy"), POLICY_FLAGS, policy_hash(),
                    POLICY_LIB, verbose)


def build(verbose=False, out_dir=None, phase_clocks=False):
    """Compile every unit and link the libraries. phase_clocks: libinet_nr.so's sources with INET_PHASE_CLOCKS defined
    (every step-kernel wavefront records the shader clock spent in each phase of the step), linked as
    libinet_nr_phase.so for bench.py --phase-clocks; the product libraries are not touched."""
    obj_dir = out_dir or os.path.join(HERE, "_build_phase" if phase_clocks else "_build")
    extra = ["-DINET_PHASE_CLOCKS"] if phase_clocks else []
    if not phase_clocks:
        build_policy(verbose)
    return _compile(UNITS, CSRC, obj_dir, FLAGS + extra, source_hash(), PHASE_LIB if phase_clocks else LIB, verbose)


if __name__ == "__main__":
    verb = "-v" in sys.argv
    print(build_policy(verb) if "--policy" in sys.argv else build(verb, phase_clocks="--phase-clocks" in sys.argv))
