"""Build recipe of ``libwisp_b200.so`` (sm_100a), in-tree.

``python -m wisp_b200.build`` compiles every CUDA/C++ source under ``csrc/`` with
``nvcc -gencode arch=compute_100a,code=sm_100a`` into ``wisp_b200/_lib``.  The
static CUDA runtime is linked in, so the library does not depend on the
runtime version another extension in the same process loaded.

Objects are rebuilt when the content of their source, of any header or of the
compile flags changes (a sha256 per object, not file times), the sources compile
in parallel, and the library is stamped with a hash of everything it was built
from: ``wisp_b200_version()`` returns ``"wisp_b200 <version> sm_100a src:<hash>"``,
so a run can show which sources the loaded library came from (``source_hash()``
computes the same hash from the tree).
"""

from __future__ import annotations

import hashlib
import os
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "_lib"
LIB = LIB_DIR / "libwisp_b200.so"
OBJ_DIR = ROOT / "_build" / "obj"
VERSION = "0.2.0"
# the Python binding of the paged cache's calls: a module of its own, against torch
BINDING_SRC = "torch_binding.cpp"
BINDING = LIB_DIR / "_paged_torch.so"

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O3,-Wall,-Wno-unused-function",
          f"-I{ROOT / 'include'}", f"-I{CSRC}"]
SOURCES = ["moe_kernels.cu", "dense_ffn.cu", "prefill.cu", "expert_layout.cu", "quantize.cu",
           "ref_launchers.cu", "decoder.cu", "paged.cu", "paged_plan.cu", "paged_attn.cu", "paged_mma.cu", "paged_few.cu",
           "page_pool.cpp", "engine.cpp", "tiers.cpp", "stream_cache.cpp", "multi_gpu.cpp"]
HEADERS = ["internal.h", "tiers.h", "route_common.cuh", "dense_ffn.h", "paged.h", "paged_math.cuh", "paged_tma.cuh"]


def _headers() -> list[Path]:
    return [CSRC / h for h in HEADERS] + [ROOT / "include" / "wisp_b200.h"]


def source_hash() -> str:
    """sha256 (first 16 hex digits) over every source, header and the flags."""
    h = hashlib.sha256()
    for p in [CSRC / s for s in SOURCES] + _headers():
        h.update(p.name.encode())
        h.update(p.read_bytes())
    h.update(" ".join(ARCH + COMMON).encode())
    return h.hexdigest()[:16]


def _compile(src: Path, obj: Path, hdr_bytes: bytes, force: bool, ptxas_info: bool,
             verbose: bool) -> None:
    cmd = [NVCC, *ARCH, *COMMON, "-c", str(src), "-o", str(obj)]
    if ptxas_info and src.suffix == ".cu":
        cmd.insert(1, "-Xptxas=-v")
    digest = hashlib.sha256(src.read_bytes() + hdr_bytes + " ".join(cmd).encode()).hexdigest()
    stamp = obj.with_suffix(obj.suffix + ".sha256")
    if not force and obj.exists() and stamp.exists() and stamp.read_text() == digest:
        return
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    if ptxas_info or verbose:
        print(r.stderr, file=sys.stderr)
    stamp.write_text(digest)


def build(verbose: bool = False, ptxas_info: bool = False) -> Path:
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    binding = ThreadPoolExecutor(max_workers=1).submit(build_binding, verbose)
    hdr_bytes = b"".join(p.read_bytes() for p in _headers())
    objs = [OBJ_DIR / (s + ".o") for s in SOURCES]
    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 4)) as ex:
        list(ex.map(lambda so: _compile(CSRC / so[0], so[1], hdr_bytes, ptxas_info, ptxas_info,
                                        verbose), zip(SOURCES, objs)))
    # the identity stamp: a generated translation unit holding the source hash
    src_hash = source_hash()
    ident = f"wisp_b200 {VERSION} sm_100a src:{src_hash}"
    stamp_src = OBJ_DIR / "version_stamp.cpp"
    text = ('// generated by wisp_b200/build.py: the identity of this build\n'
            f'extern "C" const char* wisp_b200_version(void) {{ return "{ident}"; }}\n')
    if not stamp_src.exists() or stamp_src.read_text() != text:
        stamp_src.write_text(text)
    stamp_obj = OBJ_DIR / "version_stamp.o"
    _compile(stamp_src, stamp_obj, b"", False, False, verbose)
    objs.append(stamp_obj)
    lib_stamp = LIB.with_suffix(".so.sha256")
    link_key = hashlib.sha256(b"".join(o.read_bytes() for o in objs)).hexdigest()
    if not LIB.exists() or not lib_stamp.exists() or lib_stamp.read_text() != link_key:
        cmd = [NVCC, *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-lpthread", "-ldl"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        lib_stamp.write_text(link_key)
    try:
        binding.result()
    except BindingUnavailable as e:  # the C library stands without it
        warnings.warn(f"built without the torch binding of wisp_b200.paged: {e}", RuntimeWarning)
    return LIB


class BindingUnavailable(RuntimeError):
    """What the torch binding is built against is not installed."""


def build_binding(verbose: bool = False) -> Path:
    """``_paged_torch.so`` (host code only), rebuilt when its source, the ABI header, torch or
    the flags change."""
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    src, stamp = CSRC / BINDING_SRC, BINDING.with_suffix(".so.sha256")
    src_key = hashlib.sha256(src.read_bytes() +
                             (ROOT / "include" / "wisp_b200.h").read_bytes()).hexdigest()

    def missing(what: str):
        # (a binding of another source does not fit the library: it must not be loaded)
        if BINDING.exists() and not (stamp.exists() and stamp.read_text().startswith(src_key + " ")):
            BINDING.unlink()
        return BindingUnavailable(what)

    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError as e:
        raise missing(f"no torch ({e})") from None
    torch_lib = Path(torch.__file__).parent / "lib"
    inc = [*cpp_extension.include_paths(device_type="cuda"), sysconfig.get_paths()["include"],
           str(ROOT / "include")]
    for header in ("Python.h", "ATen/ATen.h"):
        if not any((Path(i) / header).exists() for i in inc):
            raise missing(f"no {header}")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{i}" for i in inc), str(src), "-o", str(BINDING), f"-L{torch_lib}",
           f"-Wl,-rpath,{torch_lib}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    key = src_key + " " + hashlib.sha256((torch.__version__ + " ".join(cmd)).encode()).hexdigest()
    if BINDING.exists() and stamp.exists() and stamp.read_text() == key:
        return BINDING
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {BINDING_SRC}:\n{r.stdout}\n{r.stderr}")
    stamp.write_text(key)
    return BINDING


if __name__ == "__main__":
    build(verbose="-v" in sys.argv, ptxas_info="--ptxas" in sys.argv)
    print(LIB)
