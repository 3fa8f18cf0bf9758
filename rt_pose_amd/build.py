"""Build librtp_hip.so (all HIP kernels + the C ABI) for gfx950 with hipcc, in-tree.

    python -m rt_pose_amd.build            # what is older than its source or was made by another command (flags, compiler)
    python -m rt_pose_amd.build --force    # everything

hipcc cross-compiles without a GPU, so this also runs in the CPU-only authoring container.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "lib", "obj")
LIB = os.path.join(HERE, "lib", "librtp_hip.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function", "-Wno-inline-asm",
         "-Wno-int-to-pointer-cast",
         # no SLP vectoriser: it packs the epilogues' fp32 adds / multiplies into v_pk_add_f32 / v_pk_fma_f32, which cost more issue
         # time beside the matrix pipe than the scalar pairs they replace (fused data gradient of conv_tiled: 77.6 -> 72.8 us)
         "-fno-slp-vectorize",
         # no packed fp32 at all (hipcc also forms v_pk_add / mul / fma_f32 from plain float code): some of their forms have given
         # wrong results now and then.  The host pass does not know the feature and says so; harmless.
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"] + os.environ.get("RTP_HIPCC_EXTRA", "").split()
LIB = os.environ.get("RTP_BUILD_LIB", LIB)   # A/B builds: another output library (load it with RTP_LIB)
OBJ = os.environ.get("RTP_BUILD_OBJ", OBJ)


def sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))


def _deps_mtime():
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")]
    hdrs.append(os.path.join(os.path.dirname(HERE), "include", "rtp.h"))
    return max(os.path.getmtime(h) for h in hdrs)


def _made_by(out, cmd):
    """Whether `out` is there and this very command made it (recorded beside it once it had succeeded)."""
    try:
        with open(out + ".cmd") as f:
            return os.path.exists(out) and f.read() == cmd
    except OSError:
        return False


def _run(cmd, out, what):
    if os.path.exists(out + ".cmd"):
        os.remove(out + ".cmd")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("%s failed:\n%s\n%s" % (what, r.stdout, r.stderr))
    with open(out + ".cmd", "w") as f:
        f.write(_record(cmd))


def _record(cmd):
    """The command and the compiler that it stands for: another release, or another file at the same place, is another command."""
    real = os.path.realpath(cmd[0])
    return "\n".join([real, str(os.path.getmtime(real)) if os.path.exists(real) else "", *cmd])


def _compile(src, force, hdr_m):
    """An object is taken as it is if it is newer than its source and the headers and was made by the same command: other flags make other code."""
    obj = os.path.join(OBJ, src[:-4] + ".o")
    srcp = os.path.join(CSRC, src)
    cmd = [HIPCC, *FLAGS, "-c", srcp, "-o", obj]
    if not force and _made_by(obj, _record(cmd)) and os.path.getmtime(obj) > max(os.path.getmtime(srcp), hdr_m):
        return obj
    _run(cmd, obj, "hipcc for %s" % src)
    return obj


def build(force=False, verbose=True):
    os.makedirs(OBJ, exist_ok=True)
    hdr_m = _deps_mtime()
    with ThreadPoolExecutor(max_workers=4) as ex:
        objs = list(ex.map(lambda s: _compile(s, force, hdr_m), sources()))
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB, *objs]
    if force or not _made_by(LIB, _record(cmd)) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        _run(cmd, LIB, "link")
        if verbose:
            print("built", LIB)
    elif verbose:
        print("up to date:", LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
