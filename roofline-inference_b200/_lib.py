"""Loader of the C-ABI library librib_attention.so (CUDA kernels for sm_100a), and of the native Python
binding of its paged-cache entry points (_paged_binding.so).

The library is built in-tree from csrc/ with nvcc.  `load()` rebuilds it when
its sources changed (content hash, not mtimes, so a copied tree is recognised
correctly) and then binds the entry points declared in
include/rib_attention.h with ctypes.  There is no fallback: if the library
cannot be built or loaded, every call raises.
"""
from __future__ import annotations

import ctypes
import fcntl
import hashlib
import importlib.util
import os
import shutil
import subprocess
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
HEADER = REPO_DIR / "include" / "rib_attention.h"
LIB_PATH = PKG_DIR / "librib_attention.so"
STAMP = PKG_DIR / "librib_attention.so.srchash"
MAIN_SOURCE = CSRC / "rib_attention.cu"
BINDING_SOURCE = CSRC / "paged_binding.cpp"
BINDING_PATH = PKG_DIR / "_paged_binding.so"
BINDING_STAMP = PKG_DIR / "_paged_binding.so.srchash"

EXPORTS = CSRC / "exports.map"
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "-Xlinker", f"--version-script={EXPORTS}",
]

# status codes (include/rib_attention.h)
RIB_OK, RIB_EINVAL, RIB_ECAPACITY, RIB_EALIGN, RIB_ECUDA, RIB_ETIMEOUT = range(6)

_lib: ctypes.CDLL | None = None
_binding_module = None


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [HEADER, EXPORTS]


def source_hash() -> str:
    h = hashlib.sha256()
    for p in _sources():
        h.update(p.name.encode())
        h.update(p.read_bytes())
    h.update(" ".join(f for f in NVCC_FLAGS if not f.startswith("--version-script")).encode())
    return h.hexdigest()


def is_current() -> bool:
    return LIB_PATH.exists() and STAMP.exists() and STAMP.read_text().strip() == source_hash()


def _nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: cannot build librib_attention.so")


def _run(cmd: list[str], tool: str, verbose: bool) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{tool} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    if verbose:
        print(res.stdout + res.stderr)


def _binding_command() -> list[str]:
    import torch
    root = Path(torch.__file__).parent
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
            f"-I{sysconfig.get_paths()['include']}", f"-I{root / 'include'}",
            f"-I{root / 'include/torch/csrc/api/include'}", f"-I{Path(_nvcc()).resolve().parent.parent / 'include'}",
            str(BINDING_SOURCE), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-lc10",
            "-lc10_cuda"]


def binding_hash() -> str:
    import torch
    h = hashlib.sha256(f"{torch.__version__} {sysconfig.get_python_version()}".encode())
    for p in (BINDING_SOURCE, HEADER):
        h.update(p.read_bytes())
    return h.hexdigest()


def binding_is_current() -> bool:
    return BINDING_PATH.exists() and BINDING_STAMP.exists() and BINDING_STAMP.read_text().strip() == binding_hash()


def _build_locked(current, make, force: bool) -> None:
    """Runs `make` unless `current()`.  Serialised with a file lock so that several ranks importing the
    package at once build only once."""
    if not force and current():
        return
    with open(PKG_DIR / ".librib_attention.lock", "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        try:
            if force or not current():
                make()
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compiles csrc/rib_attention.cu for sm_100a into librib_attention.so."""
    def make():
        tmp = LIB_PATH.with_name(f"{LIB_PATH.name}.{os.getpid()}.tmp")
        cmd = [_nvcc(), *NVCC_FLAGS, "-o", str(tmp), str(MAIN_SOURCE)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        _run(cmd, "nvcc", verbose)
        tmp.replace(LIB_PATH)
        STAMP.write_text(source_hash() + "\n")
    _build_locked(is_current, make, force)
    return LIB_PATH


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """Compiles csrc/paged_binding.cpp against this process's torch into _paged_binding.so."""
    def make():
        tmp = BINDING_PATH.with_name(f"{BINDING_PATH.name}.{os.getpid()}.tmp")
        _run([*_binding_command(), "-o", str(tmp)], "g++", verbose)
        tmp.replace(BINDING_PATH)
        BINDING_STAMP.write_text(binding_hash() + "\n")
    _build_locked(binding_is_current, make, force)
    return BINDING_PATH


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compiles the library and the binding where their sources changed (or `force`)."""
    path = build_library(force, verbose)
    build_binding(force, verbose)
    return path


def _bind(L: ctypes.CDLL) -> None:
    vp, i, d, f, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_double, ctypes.c_float, ctypes.c_size_t
    ll = ctypes.c_longlong
    sig = {
        "rib_version": ([], i),
        "rib_status_string": ([i], ctypes.c_char_p),
        "rib_last_error_string": ([], ctypes.c_char_p),
        "rib_take_device_status": ([ctypes.POINTER(ctypes.c_int)], i),
        "rib_set_wait_limit_ns": ([ctypes.c_ulonglong], i),
        "rib_get_wait_limit_ns": ([ctypes.POINTER(ctypes.c_ulonglong)], i),
        "rib_qk_norm_rope": ([vp, vp, vp, i, i, i, d, vp, vp, vp], i),
        "rib_qk_norm_rope_prefill": ([vp, i, vp, vp, i, i, i, d, i, vp, vp, vp], i),
        "rib_qk_norm_rope_append": ([vp, i, vp, vp, i, i, i, d, i, vp, vp, i, vp], i),
        "rib_decode_workspace_bytes": ([i, i, i], sz),
        "rib_decode_kernel_choice": ([i, i, i], i),
        "rib_decode_workspace_init": ([vp, sz, vp], i),
        "rib_decode_attention": ([vp, vp, i, i, i, i, f, vp, vp, sz, vp], i),
        "rib_decode_attention_noalloc": ([vp, vp, i, i, i, i, f, vp, vp], i),
        "rib_decode_attention_batched": ([vp, vp, vp, i, i, i, i, i, f, vp, vp, sz, vp], i),
        "rib_prefill_workspace_bytes": ([i, i], sz),
        "rib_prefill_attention": ([vp, vp, vp, i, i, i, i, i, i, f, vp, vp, sz, vp], i),
        "rib_qk_norm_rope_append_dev": ([vp, i, vp, vp, vp, i, i, d, i, vp, vp, i, vp], i),
        "rib_qk_norm_rope_prefill_dev": ([vp, i, vp, vp, vp, i, i, d, i, vp, vp, vp], i),
        "rib_gemv": ([vp, i, i, vp, vp, vp, i, i, vp, vp], i),
        "rib_add_rms": ([vp, vp, vp, i, i, vp, vp, vp], i),
        "rib_rms_norm": ([vp, vp, i, i, vp, vp], i),
        "rib_swiglu": ([vp, i, i, vp, vp], i),
        "rib_embed": ([vp, i, i, vp, i, vp, vp], i),
        "rib_argmax_workspace_bytes": ([], sz),
        "rib_argmax_f32": ([vp, i, vp, vp, vp], i),
        "rib_qwen3_step_workspace_bytes": ([vp, i], sz),
        "rib_qwen3_step_workspace_init": ([vp, sz, vp], i),
        "rib_qwen3_decode_step": ([vp, vp, i, vp, vp, vp, vp, vp, sz, vp], i),
        "rib_decode_attention_ragged": ([vp, vp, vp, vp, i, i, i, i, f, vp, vp, sz, vp], i),
        "rib_qk_norm_rope_append_batched": ([vp, vp, vp, vp, vp, vp, i, i, i, d, vp, vp], i),
        "rib_argmax_rows_f32": ([vp, i, i, vp, vp], i),
        "rib_decode_attention_qkv": ([vp, vp, vp, d, vp, vp, i, i, i, i, i, f, vp, vp, sz, vp], i),
        "rib_rotary_apply": ([vp, vp, ll, ll, vp, ll, ll, vp, i, i, i, i, vp], i),
        "rib_paged_append": ([vp, vp, vp, ll, ll, vp, ll, ll, vp, ll, ll, vp, ll, ll, vp, vp, vp, i, i, vp, vp, f,
                              vp], i),
        "rib_paged_decode_workspace_bytes": ([i, i, i, i, i], sz),
        "rib_paged_decode_attention": ([vp, vp, ll, ll, vp, i, i, i, f, vp, vp, ll, ll, vp, ll, ll, vp, sz, vp], i),
        "rib_paged_evict": ([vp, vp, ll, i, vp, i, i, vp, ll, ll, i, i, i, vp, vp, vp, ll, ll, i, vp], i),
    }
    for name, (args, res) in sig.items():
        fn = getattr(L, name)
        fn.argtypes = args
        fn.restype = res


def load() -> ctypes.CDLL:
    """Builds if needed, loads and binds the library (once per process).  The Python binding of the paged-cache
    calls is left to binding(): a library that is up to date needs no compiler."""
    global _lib
    if _lib is None:
        path = build_library()
        L = ctypes.CDLL(str(path))
        _bind(L)
        _lib = L
    return _lib


def binding():
    """The native binding of the paged-cache entry points, built if needed (once per process)."""
    global _binding_module
    if _binding_module is None:
        L = load()
        build_binding()
        spec = importlib.util.spec_from_file_location("_paged_binding", BINDING_PATH)
        m = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(m)
        m.bind(*(ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in (
            "rib_status_string", "rib_last_error_string", "rib_rotary_apply", "rib_paged_append",
            "rib_paged_decode_workspace_bytes", "rib_paged_decode_attention", "rib_paged_evict")))
        _binding_module = m
    return _binding_module


def check(status: int, what: str) -> None:
    """Raises like the reference: ValueError for shape/capacity/alignment
    problems (agent-test/v2/engine.py:45-46, 69-70), RuntimeError otherwise."""
    if status == RIB_OK:
        return
    msg = load().rib_status_string(status).decode()
    if status in (RIB_EINVAL, RIB_ECAPACITY, RIB_EALIGN):
        raise ValueError(f"{what}: {msg}")
    detail = load().rib_last_error_string().decode()
    raise RuntimeError(f"{what}: {msg} (status {status}): {detail}")


def take_device_status() -> int:
    """Reads and clears the device status word (synchronises the device)."""
    v = ctypes.c_int(0)
    check(load().rib_take_device_status(ctypes.byref(v)), "rib_take_device_status")
    return v.value


DEFAULT_WAIT_LIMIT_NS = 2_000_000_000


def set_wait_limit_ns(ns: int) -> None:
    """Sets the wall-clock limit of every device-side wait on the current
    device (1 ms .. 60 s; the default is 2 s).  Takes effect for kernels
    launched afterwards; call it while none of this library's kernels runs."""
    check(load().rib_set_wait_limit_ns(int(ns)), "rib_set_wait_limit_ns")


def wait_limit_ns() -> int:
    v = ctypes.c_ulonglong(0)
    check(load().rib_get_wait_limit_ns(ctypes.byref(v)), "rib_get_wait_limit_ns")
    return v.value
