"""tools/library_gemm_scan.py -- the stamp of the installed fp32 library GEMMs (names and sizes of their gfx950 files, torch / HIP version).

    python tools/library_gemm_scan.py

scp_amd/streams.py compares it with tuning/coresidency_stamp.json: an installation other than the one whose co-residency was screened
(tests/test_coresidency_gpu.py) defaults to the one-stream schedule.  The files themselves are not opened: what an installed library
holds is established by running beside it, never by reading its code."""
import hashlib
import os
import sys


def torch_lib_dir():
    import torch
    return os.path.join(os.path.dirname(torch.__file__), "lib")


def code_objects():
    """paths of the fp32 gfx950 GEMM files rocBLAS / hipBLASLt ship inside torch, and their helper-kernel files"""
    lib = torch_lib_dir()
    out = []
    for sub in ("rocblas/library", "hipblaslt/library"):
        d = os.path.join(lib, sub)
        for f in sorted(os.listdir(d)) if os.path.isdir(d) else ():
            if "gfx950" in f and (f.endswith(".co") or f.endswith(".hsaco")) and (f.startswith("Kernels.so") or "Type_SS_" in f):
                out.append(os.path.join(d, f))
    return out


def stamp(files=None):
    """the torch build and a digest over the names + sizes of those files"""
    import torch
    files = code_objects() if files is None else files
    h = hashlib.sha256()
    for f in files:
        h.update(("%s:%d;" % (os.path.basename(f), os.path.getsize(f))).encode())
    return {"torch": torch.__version__, "hip": str(torch.version.hip), "code_objects": len(files), "digest": h.hexdigest()[:16]}


if __name__ == "__main__":
    print("stamp %r" % (stamp(),))
    sys.exit(0)
