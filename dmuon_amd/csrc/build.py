"""Builds libdmuon_amd.so (gfx950) in-tree with hipcc, and the extension module of the autograd
operators on it (_dmuon_torch.so, host code only; left out where there is no torch to build against).

    python -m dmuon_amd.csrc.build          # or: python dmuon_amd/csrc/build.py

Every call recompiles (the in-tree .so travels with the source tree to the GPU host).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent.parent
SOURCES = ["ns_gemm.hip", "gram_small.hip", "ew_kernels.hip", "adamw.hip", "clip.hip",
           "head_gemm.hip", "head_rows.hip", "head_loss.hip", "residual_norm.hip", "attention_fwd.hip",
           "attention_bwd.hip", "attention.hip", "rotary_heads.hip", "embedding.hip", "abi.hip"]
LIB_NAME = "libdmuon_amd.so"
ARCH = "gfx950"

# -packed-fp32-ops: keep hipcc from emitting v_pk_{add,mul,fma}_f32 (some forms have given wrong
# results on the target machines); the host pass prints a harmless "not a recognized feature" warning for it.
FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # no a*b+c contraction: the momentum and weight updates round each op like the reference
    "-ffp-contract=off",
    # leading scalar kernel arguments arrive in SGPRs instead of by a load from memory
    "-mllvm", "-amdgpu-kernarg-preload-count=8",
    "-Wall",
    "-Wno-unused-function",
]


BINDING = "torch_binding.cpp"
BINDING_NAME = "_dmuon_torch.so"


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (need ROCm in /opt/rocm)")


def lib_path() -> Path:
    return HERE / LIB_NAME


def binding_path() -> Path:
    return HERE / BINDING_NAME


def _run(cmd, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in (proc.stderr or "").splitlines() if noise not in l)
    if proc.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({proc.returncode}):\n{err}")
    if err.strip() and verbose:
        print(err, file=sys.stderr)


def build(verbose: bool = False) -> Path:
    out = lib_path()
    tmp = out.with_suffix(".so.tmp")
    compile_flags = [f for f in FLAGS if f != "-shared"]
    with tempfile.TemporaryDirectory() as d:
        objects = [str(Path(d) / (s + ".o")) for s in SOURCES]
        jobs = [[hipcc(), *compile_flags, "-I", str(ROOT / "include"), "-c", str(HERE / s), "-o", o]
                for s, o in zip(SOURCES, objects)]
        module = str(Path(d) / (BINDING + ".o"))
        try:
            module_job = _binding_compile(module)
        except ImportError as e:
            module_job = None
            print(f"{BINDING_NAME} is not built: {e}", file=sys.stderr)
        # the files are independent code objects: one compiler each
        with ThreadPoolExecutor(max_workers=min(len(jobs) + 1, os.cpu_count() or 1, 8)) as pool:
            compiled = pool.submit(_run, module_job, verbose) if module_job else None
            list(pool.map(lambda cmd: _run(cmd, verbose), jobs))
        _run([hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *objects, "-o", str(tmp)], verbose)
        _check_launch_stubs(tmp)
        os.replace(tmp, out)
        # the library needs no torch: the module's errors come after it
        if compiled:
            compiled.result()
            tmp = binding_path().with_suffix(".so.tmp")
            _run(_binding_link(module, str(tmp)), verbose)
            os.replace(tmp, binding_path())
    return out


def _cxx() -> str:
    return shutil.which("g++") or hipcc()


def _binding_compile(obj: str) -> list:
    """The extension module is compiled against this interpreter's torch."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    return [_cxx(), "-O2", "-std=c++17", "-fPIC", "-Wall",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", f'-DDMUON_TORCH="{torch.__version__}"',
            *[x for d in cpp_extension.include_paths() for x in ("-isystem", d)],
            "-isystem", "/opt/rocm/include", "-isystem", sysconfig.get_paths()["include"],
            "-c", str(HERE / BINDING), "-o", obj]


def _binding_link(obj: str, out: str) -> list:
    """It finds the library beside itself."""
    from torch.utils import cpp_extension

    return [_cxx(), "-shared", obj, "-o", out,
            *[f"-L{d}" for d in cpp_extension.library_paths()],
            "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip",
            f"-L{HERE}", f"-l:{LIB_NAME}", "-Wl,-rpath,$ORIGIN"]


def _check_launch_stubs(so: Path) -> None:
    """clang can silently skip a kernel template's host launch stub (the library then fails
    to load with an undefined __device_stub__ symbol); catch that at build time."""
    nm = shutil.which("nm")
    if not nm:
        return
    proc = subprocess.run([nm, "-D", "--undefined-only", str(so)], capture_output=True, text=True)
    missing = [l.split()[-1] for l in proc.stdout.splitlines() if "__device_stub__" in l]
    if missing:
        so.unlink(missing_ok=True)
        raise RuntimeError("hipcc dropped kernel launch stubs: " + ", ".join(missing[:4]))


if __name__ == "__main__":
    p = build(verbose=True)
    print(f"built {p}")
