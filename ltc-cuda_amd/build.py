"""Compile libltc_hip.so (the C-ABI library) for gfx950 with hipcc, in-tree.

Usage:  python ltc-cuda_amd/build.py [--verbose]

The library is linked against the HIP runtime by SONAME only (no rpath), so
a process that has already imported torch resolves it to torch's bundled
libamdhip64.so.7 and only one HIP runtime is ever mapped.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_NAME = "libltc_hip.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
SOURCES = ("ltc_device.hip", "ltc_capi.hip", "ltc_scan_device.hip", "ltc_token_device.hip",
           "ltc_seq_capi.hip", "ltc_conv_device.hip", "ltc_ssm_device.hip",
           "ltc_vocab_device.hip", "ltc_model_capi.hip")
HEADERS = ("ltc_internal.h", "ltc_seq_internal.h", "ltc_model_internal.h", "ltc_capi_util.h",
           "ltc_vec.h", "ltc_tokens.h", "ltc_torch_checks.h", "ltc_torch_util.h")
ARCH = os.environ.get("LTC_OFFLOAD_ARCH", "gfx950")


def hipcc_path() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.isfile(cand):
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def source_files() -> list:
    """Every file the library and the torch extension are built from."""
    inc = os.path.join(os.path.dirname(HERE), "include", "ltc_capi.h")
    return [os.path.join(CSRC, s) for s in SOURCES] + [
        *[os.path.join(CSRC, s) for s in HEADERS + EXT_SOURCES], inc]


def _flags(arch: str) -> list:
    return [f"--offload-arch={arch}", "-O3", "-std=c++17", "-fPIC", "-mcode-object-version=5",
            # No packed-FP32 (v_pk_*_f32) instructions anywhere in device code.
            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
            "-Wall", "-Wno-unused-command-line-argument"]


def compile_command(source: str, out: str, arch: str = ARCH) -> list:
    """One source of the library to an object."""
    return [hipcc_path(), *_flags(arch), "-c", os.path.join(CSRC, source), "-o", out]


def command(out: str = LIB_PATH, arch: str = ARCH, inputs=None) -> list:
    """The library from its sources, or from their objects."""
    return [hipcc_path(), *_flags(arch), "-shared",
            # Resolve libamdhip64.so.7 by SONAME (torch's copy once torch is loaded).
            "-fno-rtlib-add-rpath",
            # Fixed SONAME: the torch extension and ctypes then share one instance.
            "-Wl,-soname," + LIB_NAME, "-o", out,
            *(inputs or [os.path.join(CSRC, s) for s in SOURCES])]


EXT_SOURCES = ("ltc_torch_ext.cpp", "ltc_torch_seq.cpp", "ltc_torch_model.cpp")
EXT_NAME = "_ltc_torch"


def ext_path() -> str:
    import sysconfig
    return os.path.join(HERE, EXT_NAME + sysconfig.get_config_var("EXT_SUFFIX"))


def ext_commands(objects, out: str) -> tuple:
    """Host-only C++ build of the torch glue (the autograd nodes of the fused module path and
    of the sequence, token and model operators): a command for each of its sources, and the
    one that links them against libltc_hip.so through $ORIGIN."""
    import sysconfig
    import torch
    from torch.utils import cpp_extension as ce
    incs = ce.include_paths("cuda") + [sysconfig.get_paths()["include"]]
    libs = ce.library_paths("cuda")[:1]
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    cxx = os.environ.get("CXX", "g++")
    flags = [
        "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-w",
        # The HIP headers torch includes select their AMD half with this macro.
        "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
        f"-D_GLIBCXX_USE_CXX11_ABI={abi}", f"-DTORCH_EXTENSION_NAME={EXT_NAME}",
        "-DTORCH_API_INCLUDE_EXTENSION_H",
        *[f"-I{d}" for d in incs]]
    compiles = [[cxx, *flags, "-c", os.path.join(CSRC, s), "-o", o] for s, o in zip(EXT_SOURCES, objects)]
    link = [cxx, "-shared", *objects, "-o", out, f"-L{HERE}", "-lltc_hip", *[f"-L{d}" for d in libs],
            "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_python",
            "-Wl,-rpath,$ORIGIN", "-Wl,--no-as-needed"]
    return compiles, link


def _run(cmd, what: str, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    msgs = [ln for ln in (proc.stdout + proc.stderr).splitlines() if noise not in ln]
    if proc.returncode != 0:
        raise RuntimeError(f"{what} failed:\n" + "\n".join(msgs))
    if verbose and msgs:
        print("\n".join(msgs), flush=True)


def build(verbose: bool = False, arch: str = ARCH) -> str:
    """Compile libltc_hip.so for `arch` and the torch extension, several sources at once;
    returns the library path."""
    with tempfile.TemporaryDirectory() as tmp:
        objects = [os.path.join(tmp, s + ".o") for s in SOURCES]
        ext_objects = [os.path.join(tmp, s + ".o") for s in EXT_SOURCES]
        lib_tmp, ext_tmp = LIB_PATH + ".tmp", ext_path() + ".tmp"
        ext_compiles, ext_link = ext_commands(ext_objects, ext_tmp)
        jobs = [(compile_command(s, o, arch), "hipcc") for s, o in zip(SOURCES, objects)]
        jobs += [(c, "torch extension build") for c in ext_compiles]
        with concurrent.futures.ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
            for done in [pool.submit(_run, cmd, what, verbose) for cmd, what in jobs]:
                done.result()
        _run(command(lib_tmp, arch, objects), "hipcc", verbose)
        os.replace(lib_tmp, LIB_PATH)
        _run(ext_link, "torch extension build", verbose)
        os.replace(ext_tmp, ext_path())
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose="--verbose" in sys.argv))
