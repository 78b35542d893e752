"""Build libstreamvbyte.so.2 (HIP, gfx950) in-tree.

    python -m streamvbyte_amd.build [--force]

The translation units of csrc/ side by side, then one link; the library lands next to this file
so that it travels with the source tree.
"""
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libstreamvbyte.so.2")
LINK = os.path.join(HERE, "libstreamvbyte.so")
# the same library with the look-back's stress hooks compiled in (csrc/svb_lookback.h: lb_stress_delay);
# loaded only by the tests of it (test_gpu_lookback_stress.py, test_gpu_grad_stress.py), through SVB_LIB_PATH
STRESS_LIB = os.path.join(HERE, "libstreamvbyte_stress.so.2")
# No packed float32 arithmetic: some forms of v_pk_{add,mul,fma}_f32 have given wrong results now and then on these
# cards, and the compiler makes them by itself from ordinary float code.  (The host pass does not know the feature and
# says so: harmless.)
DEVICE_FLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


UNITS = ["svb_api", "svb_grad"]  # translation units: csrc/<unit>.hip
OBJ = os.path.join(HERE, "obj")


def with_includes(path, seen=None):
    """The file and every file of this repository that it includes."""
    seen = set() if seen is None else seen
    path = os.path.normpath(path)
    if path not in seen and os.path.exists(path):
        seen.add(path)
        for name in re.findall(r'^#include "([^"]+)"', open(path).read(), flags=re.M):
            for base in (os.path.dirname(path), os.path.join(ROOT, "include")):
                with_includes(os.path.join(base, name), seen)
    return sorted(seen)


def stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(s) > t for s in deps)


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    return subprocess.Popen(cmd)


def _wait(jobs):
    codes = [(j.wait(), j.args) for j in jobs]
    for rc, args in codes:
        if rc != 0:
            raise subprocess.CalledProcessError(rc, args)


def build(force=False, verbose=True):
    """Both libraries: every stale unit compiled side by side, then linked."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    os.makedirs(OBJ, exist_ok=True)
    objects = {LIB: [], STRESS_LIB: []}
    jobs = []
    for lib, extra, tag in ((LIB, [], ""), (STRESS_LIB, ["-DSVB_LB_STRESS"], ".stress")):
        for unit in UNITS:
            src, obj = os.path.join(CSRC, unit + ".hip"), os.path.join(OBJ, unit + tag + ".o")
            objects[lib].append(obj)
            if force or stale(obj, with_includes(src)):
                jobs.append(_run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function",
                                  *DEVICE_FLAGS, *extra, "-I", os.path.join(ROOT, "include"), "-c", src, "-o", obj], verbose))
    _wait(jobs)
    jobs = [_run([hipcc, "--offload-arch=gfx950", "-fPIC", "-shared", "-Wl,-soname,libstreamvbyte.so.2", "-o", lib, *objs, "-ldl"], verbose)
            for lib, objs in objects.items() if force or stale(lib, objs)]
    _wait(jobs)
    if jobs:
        if os.path.lexists(LINK):
            os.remove(LINK)
        os.symlink(os.path.basename(LIB), LINK)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
