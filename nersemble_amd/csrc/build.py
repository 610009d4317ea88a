"""Builds nersemble_amd/csrc/libnsx.so for gfx950 with hipcc (in-tree; the .so is git-ignored but
travels to the GPU box with the gpurun snapshot).  hipcc cross-compiles without a GPU."""
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
INCLUDE = os.path.join(ROOT, "include")
OBJ = os.path.join(HERE, "_obj")
SO = os.path.join(HERE, "libnsx.so")
BINDING = os.path.join(HERE, "_experts.so")
STAMP = os.path.join(OBJ, "_experts.txt")          # what BINDING was built against
ARCH = "gfx950"


def _hipcc() -> str:
    for c in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("hipcc not found: libnsx.so cannot be built")


def _sources():
    return sorted(os.path.join(HERE, f) for f in os.listdir(HERE) if f.endswith(".hip"))


def _headers():
    hs = [os.path.join(HERE, f) for f in os.listdir(HERE) if f.endswith(".h")]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return hs


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    hipcc = _hipcc()
    os.makedirs(OBJ, exist_ok=True)
    flags = [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-I", INCLUDE, "-I", HERE,
             "-Wall", "-Wno-unused-function",
             # no packed fp32 instructions: some of their forms have given wrong results on this hardware now and then
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
    hdrs = _headers()
    jobs = []
    objs = []
    for src in _sources():
        obj = os.path.join(OBJ, os.path.basename(src)[:-4] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + hdrs + [__file__]):
            jobs.append([hipcc, *flags, "-c", src, "-o", obj])

    def run(cmd):
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"hipcc failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        if verbose and r.stderr.strip():
            print(r.stderr, file=sys.stderr)

    if jobs:
        with ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            list(ex.map(run, jobs))
    if force or jobs or _stale(SO, objs):
        run([hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", SO, *objs])
    src = os.path.join(HERE, "experts_torch.cpp")
    if force or binding_is_stale(BINDING, STAMP, [src, os.path.join(INCLUDE, "nsx.h"), __file__]):
        if os.path.exists(STAMP):
            os.remove(STAMP)
        run(_binding(src))
        with open(STAMP, "w") as f:
            f.write(_built_against())
    return SO


def _built_against() -> str:
    """The torch and the interpreter whose classes BINDING is compiled with."""
    import torch
    return f"{torch.__version__} {torch.version.git_version} {sys.version}"


def binding_is_stale(binding, stamp, deps) -> bool:
    if _stale(binding, deps) or not os.path.exists(stamp):
        return True
    with open(stamp) as f:
        return f.read() != _built_against()


def _binding(src):
    """The one source that sees torch's headers: host code only, calls libnsx.so beside it."""
    import sysconfig
    import torch
    root = os.path.join(os.path.dirname(torch.__file__))
    inc = os.path.join(root, "include")
    return [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DNSX_TORCH="{torch.__version__}"', "-I", INCLUDE, "-I", inc,
            "-I", os.path.join(inc, "torch", "csrc", "api", "include"), "-I", sysconfig.get_paths()["include"], "-I", "/opt/rocm/include",
            src, "-o", BINDING, "-L", os.path.join(root, "lib"), "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip", "-ltorch_python",
            "-L", HERE, "-lnsx", "-Wl,-rpath,$ORIGIN"]


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
