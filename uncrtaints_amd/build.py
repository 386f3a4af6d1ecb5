"""Build libuncr_hip.so (hand-written HIP for gfx950) in-tree with hipcc.

`python -m uncrtaints_amd.build` or `build_lib()`.  hipcc cross-compiles without a GPU; the .so is
git-ignored but travels to the GPU box with the working tree."""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libuncr_hip.so")
DEV_LIB = os.path.join(LIBDIR, "libuncr_dev.so")     # development probes (include/uncr_dev.h): never loaded by the product path
# (source stem, extra flags, object stem); the split GEMM is compiled once per prologue kind (compile-time PRO)
SOURCES = [(s, [], s) for s in ["norm", "ew", "pw_gemm", "pw_wgrad_split", "pw_wgrad_a16", "dwconv", "dwconv_row", "se", "ltae", "ltae_fused", "aggregate", "mgnll", "metrics", "conv3", "attn_rows", "rotary", "packed_attn", "packed_attn_rows", "packed_attn_planes", "packed_attn_bwd", "optim", "inconv", "anysize"]] + \
          [("pw_gemm_split", [f"-DPWS_PRO={p}"], f"pw_gemm_split_p{p}") for p in range(5)]
# -fno-slp-vectorize: the SLP vectoriser packs neighbouring scalar FMAs into v_pk_fma_f32 and pays for it with
# register-pair moves (depthwise row kernel: 370 vs 282 VALU instructions per row; whole step +1 %)
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 at all; some of their forms have given wrong results on these parts now and then
# (hipcc's host pass warns that it does not know the feature, which is harmless)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fno-slp-vectorize", "-Xclang", "-target-feature", "-Xclang",
         "-packed-fp32-ops"]


def source_sha() -> str:
    """sha256 (first 16 hex digits) over the kernel sources and the flags they are compiled with: measurements that depend on the kernels'
    code (the PMC traffic file under profiles/) record it, and bench.py only attaches them while it still matches."""
    import hashlib
    h = hashlib.sha256()
    for f in sorted(os.listdir(CSRC)):
        if f.endswith((".hip", ".h")) and f != "dev_probes.hip":
            h.update(f.encode())
            h.update(open(os.path.join(CSRC, f), "rb").read())
    h.update(repr((FLAGS, SOURCES)).encode())
    return h.hexdigest()[:16]


def _newer(src, dst):
    return (not os.path.exists(dst)) or os.path.getmtime(src) > os.path.getmtime(dst)


def _made_by(out):
    """The flags that made a built file, as recorded beside it (None: not known)"""
    try:
        with open(out + ".flags") as f:
            return f.read()
    except FileNotFoundError:
        return None


def build_lib(force: bool = False, verbose: bool = False) -> str:
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    os.makedirs(LIBDIR, exist_ok=True)
    objdir = os.path.join(LIBDIR, "obj")
    os.makedirs(objdir, exist_ok=True)
    hdrs = [os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith(".h")]

    def stale(out, sources, flags):
        """A file is made again if a source is newer or if other flags made it: objects of two sets of flags are not linked together"""
        return force or any(_newer(s, out) for s in sources) or _made_by(out) != " ".join(flags)

    def run(job):
        out, flags, inputs = job
        cmd = [hipcc, *flags, *inputs, "-o", out]
        if verbose:
            print(" ".join(cmd), flush=True)
        if os.path.exists(out + ".flags"):
            os.remove(out + ".flags")
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("hipcc failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
        with open(out + ".flags", "w") as f:
            f.write(" ".join(flags))

    jobs = []
    for s, extra, o in SOURCES:
        src, obj, flags = os.path.join(CSRC, s + ".hip"), os.path.join(objdir, o + ".o"), [*FLAGS, *extra, "-c"]
        if stale(obj, [src, *hdrs], flags):
            jobs.append((obj, flags, [src]))
    if jobs:
        with ThreadPoolExecutor(max_workers=min(13, len(jobs))) as ex:
            list(ex.map(run, jobs))
    objs, link = [os.path.join(objdir, o + ".o") for _, _, o in SOURCES], ["--offload-arch=gfx950", "-shared", "-fPIC"]
    if jobs or stale(LIB, objs, link):
        run((LIB, link, objs))
    dsrc, flags = os.path.join(CSRC, "dev_probes.hip"), [*FLAGS, "-shared"]
    if stale(DEV_LIB, [dsrc, *hdrs], flags):
        run((DEV_LIB, flags, [dsrc]))
    return LIB


if __name__ == "__main__":
    print(build_lib(force="--force" in sys.argv, verbose=True))
