"""Build libpixelhip.so (HIP kernels + C-ABI + network executor) for gfx950 and _pxlnode.so (its autograd nodes: host C++
against torch's headers), in-tree.

    python -m pixelssl_amd.build            # incremental
    python -m pixelssl_amd.build --force
    python -m pixelssl_amd.build --library  # libpixelhip.so alone: what a user of the C ABI needs (no g++, no torch headers)

hipcc cross-compiles without a GPU; the resulting .so is git-ignored but travels with the
snapshot to the GPU box (it is NOT listed in .gpurunignore).
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJDIR = os.path.join(CSRC, "_obj")
LIB = os.path.join(HERE, "libpixelhip.so")
HEADERS = [os.path.join(CSRC, "common.h"), os.path.join(CSRC, "conv_dma_kernel.h"), os.path.join(CSRC, "conv_halo_kernel.h"),
           os.path.join(os.path.dirname(HERE), "include", "pixelhip.h"),
           os.path.abspath(__file__)]           # (the flags above)
ARCH = "gfx950"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# (-packed-fp32-ops: no v_pk_add / mul / fma_f32 -- hipcc -O3 forms them from ordinary float code, and some of their forms have given
# wrong results on gfx950 now and then; the host pass does not know the feature and says so: -Wno-... has no name for that warning)
CFLAGS = ["--offload-arch=" + ARCH, "-O3", "-std=c++17", "-fPIC", "-munsafe-fp-atomics",
          "-Wno-unused-result", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-x", "hip"]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp")))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src, force):
    obj = os.path.join(OBJDIR, os.path.basename(src) + ".o")
    if force or _stale(obj, [src] + HEADERS):
        cmd = [HIPCC] + CFLAGS + ["-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("hipcc failed for %s:\n%s\n%s" % (src, r.stdout, r.stderr))
        return obj, True
    return obj, False


NODE_SRC = os.path.join(HERE, "node", "layer_norm_node.cpp")
NODE_LIB = os.path.join(HERE, "_pxlnode.so")


NODE_STAMP = os.path.join(OBJDIR, "_pxlnode.cmd")       # what _pxlnode.so was compiled with: torch's version among it


def _build_node(force):
    """host code only: the kernels are reached through addresses that functional.py hands over, so libpixelhip.so is loaded once"""
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    libdir = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI, NODE_SRC, "-o", NODE_LIB]
    for d in cpp_extension.include_paths() + [sysconfig.get_paths()["include"], "/opt/rocm/include"]:
        cmd += ["-isystem", d]
    cmd += ["-L" + libdir] + ["-l" + n for n in ("c10", "torch_cpu", "torch_python", "c10_hip", "torch_hip")]
    stamp = "torch %s\n%s\n" % (torch.__version__, "\n".join(cmd))
    if not force and not _stale(NODE_LIB, [NODE_SRC] + HEADERS) and _read(NODE_STAMP) == stamp:
        return False
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("compiling %s failed:\n%s\n%s" % (NODE_SRC, r.stdout, r.stderr))
    with open(NODE_STAMP, "w") as f:
        f.write(stamp)
    return True


def _read(path):
    try:
        with open(path) as f:
            return f.read()
    except OSError:
        return None


def build(force=False, verbose=True, node=True):
    """the library, and with `node` the autograd nodes: compiled beside it, but nothing that goes wrong with them keeps the library from being linked"""
    os.makedirs(OBJDIR, exist_ok=True)
    srcs = sources()
    with ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
        nodes = ex.submit(_build_node, force) if node else None
        results = list(ex.map(lambda s: _compile(s, force), srcs))
        objs = [o for o, _ in results]
        if force or any(c for _, c in results) or _stale(LIB, objs):
            cmd = [HIPCC, "--offload-arch=" + ARCH, "-shared", "-fPIC", "-o", LIB] + objs
            r = subprocess.run(cmd, capture_output=True, text=True)
            if r.returncode != 0:
                raise RuntimeError("link failed:\n%s\n%s" % (r.stdout, r.stderr))
            if verbose:
                print("built", LIB)
        elif verbose:
            print("up to date:", LIB)
        if nodes is not None and nodes.result() and verbose:
            print("built", NODE_LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, node="--library" not in sys.argv)
