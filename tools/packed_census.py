"""tools/packed_census.py -- per kernel of a built library: packed-fp32 instructions (v_pk_*_f32, with / without op_sel), K-doubled 16-bit
MFMAs, vector registers.  `python tools/packed_census.py [lib.so]` on a library built here from source (installed libraries are refused:
their code is not read); tests/test_capi_symbols.py imports census() for the static half of the
co-residency rule: a kernel that does not itself issue bf16 MFMAs carries no packed-fp32 instruction."""
import os
import re
import shutil
import subprocess
import sys
import tempfile

LLVM = "/opt/rocm/lib/llvm/bin"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEFAULT = os.path.join(ROOT, "self-corr-pose_amd", "lib", "libscp_hip.so")
PK = re.compile(r"\bv_pk_(mul|add|fma)_f32\b")
# the erratum form (csrc/selftest.hip): op_sel exactly [0,1] / [0,1,0] -- low half = src0.lo (x) src1.hi
BAD = re.compile(r"op_sel:\[0,1(,0)?\]")
MFMA16 = re.compile(r"\bv_mfma_f32_(32x32x16|16x16x32)_(bf16|f16)\b")
SYM = re.compile(r"^[0-9a-f]+ <([^>]+)>:$")


def census(lib=DEFAULT):
    """{kernel symbol: dict(packed, op_sel, bad, mfma16)} over every gfx950 code object embedded in `lib` (a .so or a .o built here)"""
    real = os.path.realpath(lib)
    if real.startswith(("/opt/", "/usr/", "/lib")) or "site-packages" in real or "dist-packages" in real:
        raise RuntimeError("packed_census: %s is an installed library; only objects built here from source are read" % lib)
    out = {}
    tmp = tempfile.mkdtemp(prefix="scp_census_")
    try:
        so = os.path.join(tmp, os.path.basename(lib))
        shutil.copy(lib, so)
        subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", so], check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
        for f in sorted(os.listdir(tmp)):
            if "amdgcn" not in f:
                continue
            text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", os.path.join(tmp, f)], check=True, capture_output=True, text=True).stdout
            cur = None
            for line in text.splitlines():
                m = SYM.match(line)
                if m:
                    cur = out.setdefault(m.group(1), dict(packed=0, op_sel=0, bad=0, mfma16=0))
                    continue
                if cur is None:
                    continue
                if PK.search(line):
                    cur["packed"] += 1
                    cur["op_sel"] += int("op_sel:[" in line)
                    cur["bad"] += int(bool(BAD.search(line)))
                elif MFMA16.search(line):
                    cur["mfma16"] += 1
    finally:
        shutil.rmtree(tmp, ignore_errors=True)
    return out


def demangle(names):
    r = subprocess.run([shutil.which("c++filt") or "cat"], input="\n".join(names), capture_output=True, text=True)
    return r.stdout.splitlines()


if __name__ == "__main__":
    c = census(sys.argv[1] if len(sys.argv) > 1 else DEFAULT)
    names = sorted(c)
    print("%-8s %-8s %-8s %-8s kernel" % ("packed", "op_sel", "erratum", "mfma16"))
    for n, d in zip(names, demangle(names)):
        k = c[n]
        if k["packed"] or k["mfma16"]:
            print("%-8d %-8d %-8d %-8d %s" % (k["packed"], k["op_sel"], k["bad"], k["mfma16"], d[:150]))
    bad = [n for n in names if c[n]["packed"] and not c[n]["mfma16"]]
    print("%d kernels, %d with packed fp32, %d of those WITHOUT bf16 MFMA" % (len(c), sum(1 for n in names if c[n]["packed"]), len(bad)))
