"""In-tree native build driver.

``python -m triton_client_amd._build [targets...]`` compiles the native pieces
into ``triton_client_amd/_lib`` (shared objects loaded by Python) and
``build/`` (C++ client library, examples and tests).  Everything targets
gfx950 only; ``hipcc`` cross-compiles without a GPU so the same command works
on a CPU-only build host.

Targets
-------
core   : libtca_core.so      (g++   – system shm, codec, base64, image decoding C ABI)
pyext  : _tca_pyext*.so      (g++   – CPython BYTES pack/unpack, native gRPC serving front)
torch  : _tca_torch*.so       (g++   – the 8-bit operators' calls on torch tensors; where torch is installed)
hip    : libtca_hip.so       (hipcc – hipshm + CDNA4 kernels)
cpp    : build/libtcaclient.{a,so}, C++ examples, tests and the perf driver
all    : everything above (default)

A target is rebuilt only when one of its sources is newer than its output.
"""

from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "csrc"
LIBDIR = Path(__file__).resolve().parent / "_lib"
BUILD = ROOT / "build"
ROCM = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))
GFX = "gfx950"

CXXFLAGS = ["-O2", "-std=c++17", "-fPIC", "-Wall", "-Wextra", "-I", str(CSRC / "include")]


def _stale(out: Path, srcs) -> bool:
    if not out.exists():
        return True
    t = out.stat().st_mtime
    deps = list(srcs) + list((CSRC / "include" / "tca").glob("*.h"))
    return any(Path(s).stat().st_mtime > t for s in deps)


def _run(cmd):
    cmd = [str(c) for c in cmd]
    print("[build]", " ".join(cmd), flush=True)
    subprocess.check_call(cmd)


def _compile_atomic(cmd, out: Path):
    """Run a compile that writes ``out`` via a temp name then renames, so that
    a concurrently importing process never maps a half-written library."""
    tmp = out.with_name(out.name + f".tmp{os.getpid()}")
    _run([tmp if c is out else c for c in cmd])
    os.replace(tmp, out)


def build_core(force=False):
    out = LIBDIR / "libtca_core.so"
    srcs = [CSRC / "core" / "base64.cc", CSRC / "core" / "codec.cc", CSRC / "core" / "shm_utils.cc",
            CSRC / "core" / "common.cc", CSRC / "core" / "image_io.cc", CSRC / "core" / "jpeg.cc",
            CSRC / "capi" / "core_capi.cc"]
    if force or _stale(out, srcs):
        LIBDIR.mkdir(exist_ok=True)
        _compile_atomic(["g++", *CXXFLAGS, "-shared", "-o", out, *srcs, "-lrt", "-lz", "-pthread"], out)
    return out


def build_pyext(force=False):
    suffix = sysconfig.get_config_var("EXT_SUFFIX")
    out = LIBDIR / f"_tca_pyext{suffix}"
    srcs = [CSRC / "capi" / "pyext.cc", CSRC / "capi" / "py_grpc_front.cc", CSRC / "capi" / "py_http_front.cc",
            CSRC / "capi" / "py_native_executor.cc", CSRC / "server" / "native_executor.cc",
            CSRC / "grpc" / "grpc_server.cc", CSRC / "http" / "http_server.cc",
            CSRC / "grpc" / "grpc_compress.cc", CSRC / "h2" / "hpack.cc", CSRC / "h2" / "connection.cc",
            CSRC / "net" / "tls.cc"]
    if force or _stale(out, srcs):
        LIBDIR.mkdir(exist_ok=True)
        inc = sysconfig.get_paths()["include"]
        _compile_atomic(["g++", *CXXFLAGS, "-I", inc, "-shared", "-o", out, *srcs, "-pthread", "-lssl", "-lcrypto",
                         "-lz"], out)
    return out


def build_torch(force=False):
    """``_tca_torch``: needs torch's headers, so it is built where torch is installed (client-only hosts go without)."""
    import importlib.util

    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        return None
    home = Path(list(spec.submodule_search_locations)[0])
    out = LIBDIR / f"_tca_torch{sysconfig.get_config_var('EXT_SUFFIX')}"
    src = CSRC / "capi" / "torch_ops.cc"
    version = (home / "version.py").read_text()
    # as _native.torch_ops() puts it together from the imported torch
    torch = " ".join("".join(re.findall(rf"^{name} = ['\"](.*)['\"]", version, re.M))
                     for name in ("__version__", "git_version"))
    built_for = LIBDIR / "_tca_torch.torch"
    if (force or _stale(out, [src, CSRC / "hip" / "kernels.h", home / "version.py"])
            or not built_for.exists() or built_for.read_text() != torch):
        LIBDIR.mkdir(exist_ok=True)
        _compile_atomic(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
                         f'-DTCA_TORCH="{torch}"', "-isystem", home / "include", "-isystem",
                         home / "include" / "torch" / "csrc" / "api" / "include", "-isystem", ROCM / "include",
                         "-isystem", sysconfig.get_paths()["include"], "-I", CSRC / "hip", "-o", out, src, f"-L{home / 'lib'}",
                         "-ltorch_python", "-ltorch_hip", "-ltorch_cpu", "-ltorch", "-lc10_hip", "-lc10"], out)
        built_for.write_text(torch)
    return out


def hip_sources():
    return sorted((CSRC / "hip").glob("*.hip")) + sorted((CSRC / "hip").glob("*.cc"))


def build_hip(force=False):
    out = LIBDIR / "libtca_hip.so"
    srcs = hip_sources()
    hdrs = list((CSRC / "hip").glob("*.h")) + list((CSRC / "hip").glob("*.hpp")) + [Path(__file__)]  # the flags
    if not srcs:
        return None
    if force or _stale(out, srcs + hdrs):
        LIBDIR.mkdir(exist_ok=True)
        hipcc = shutil.which("hipcc") or str(ROCM / "bin" / "hipcc")
        objs = []
        objdir = BUILD / "hip_obj"
        objdir.mkdir(parents=True, exist_ok=True)
        for s in srcs:
            o = objdir / (s.name + ".o")
            if force or _stale(o, [s] + hdrs):
                # packed fp32 instructions stay off: some of their forms have given wrong results on this hardware
                _run([hipcc, f"--offload-arch={GFX}", "-O3", "-std=c++17", "-fPIC", "-x", "hip",
                      "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                      "-I", CSRC / "include", "-I", CSRC / "hip", "-c", s, "-o", o])
            objs.append(o)
        _compile_atomic([hipcc, f"--offload-arch={GFX}", "-shared", "-fPIC", "-o", out, *objs,
                         f"-L{ROCM / 'lib'}", "-lamdhip64", f"-Wl,-rpath,{ROCM / 'lib'}"], out)
    return out


def build_cpp(force=False):
    mk = CSRC / "Makefile"
    if not mk.exists():
        return None
    BUILD.mkdir(exist_ok=True)
    _run(["make", "-C", CSRC, "-j8", f"BUILD={BUILD}"] + (["-B"] if force else []))
    # programs needed at run time (bench.py, perf --native, GPU tests of the C++ image client): keep
    # copies next to the shared objects, which is the directory that travels with the package
    for built, installed in (("tca_loadgen", "tca_loadgen"), ("image_client", "tca_image_client")):
        src = BUILD / "bin" / built
        if not src.exists():
            continue
        LIBDIR.mkdir(exist_ok=True)
        tmp = LIBDIR / f"{installed}.tmp{os.getpid()}"
        shutil.copy2(src, tmp)
        if shutil.which("strip"):
            subprocess.call(["strip", str(tmp)])
        os.replace(tmp, LIBDIR / installed)
    return BUILD


TARGETS = {"core": build_core, "pyext": build_pyext, "torch": build_torch, "hip": build_hip, "cpp": build_cpp}


def build(targets=None, force=False):
    targets = list(targets or ["all"])
    if "all" in targets:
        targets = list(TARGETS)
    outs = {}
    for t in targets:
        outs[t] = TARGETS[t](force=force)
    return outs


def main(argv=None):
    argv = list(sys.argv[1:] if argv is None else argv)
    force = "--force" in argv
    targets = [a for a in argv if not a.startswith("-")]
    outs = build(targets, force=force)
    for k, v in outs.items():
        print(f"[build] {k}: {v}")


if __name__ == "__main__":
    main()
