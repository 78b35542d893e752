"""Build libstreamvbyte.so.2 (HIP, gfx950) in-tree.

    python -m streamvbyte_amd.build [--force]
    python -m streamvbyte_amd.build --variant OUT [hipcc flags]

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
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", *DEVICE_FLAGS]

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


def _compiles(extra, tag):
    """(object, its dependencies, the command that makes it) of every unit."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    out = []
    for unit in UNITS:
        src, obj = os.path.join(CSRC, unit + ".hip"), os.path.join(OBJ, unit + tag + ".o")
        out.append((obj, with_includes(src), [hipcc, *FLAGS, "-fPIC", "-Wall", "-Wno-unused-function", *extra,
                                              "-I", os.path.join(ROOT, "include"), "-c", src, "-o", obj]))
    return out


def _link(lib, objects):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    return [hipcc, "--offload-arch=gfx950", "-fPIC", "-shared", "-Wl,-soname,libstreamvbyte.so.2", "-o", lib, *objects, "-ldl"]


def build(force=False, verbose=True):
    """Both libraries, where a source is newer: every stale unit compiled side by side, then linked."""
    os.makedirs(OBJ, exist_ok=True)
    plans = [(LIB, _compiles([], "")), (STRESS_LIB, _compiles(["-DSVB_LB_STRESS"], ".stress"))]
    if not force:  # by the sources alone: a built tree may have been copied without its objects
        plans = [(lib, units) for lib, units in plans if any(stale(lib, deps) for _, deps, _ in units)]
    _wait([_run(cmd, verbose) for _, units in plans for obj, deps, cmd in units if force or stale(obj, deps)])
    _wait([_run(_link(lib, [obj for obj, *_ in units]), verbose) for lib, units in plans])
    if plans:
        if os.path.lexists(LINK):
            os.remove(LINK)
        os.symlink(os.path.basename(LIB), LINK)
    return LIB


def build_variant(out, extra, verbose=True):
    """The library with extra compiler flags, as `out`: for A/B comparisons through SVB_LIB_PATH."""
    os.makedirs(OBJ, exist_ok=True)
    units = _compiles(list(extra), "." + os.path.basename(out))
    _wait([_run(cmd, verbose) for *_, cmd in units])
    _wait([_run(_link(out, [obj for obj, *_ in units]), verbose)])


if __name__ == "__main__":
    if "--variant" in sys.argv:
        at = sys.argv.index("--variant")
        build_variant(os.path.abspath(sys.argv[at + 1]), sys.argv[at + 2:])
    else:
        build(force="--force" in sys.argv)
