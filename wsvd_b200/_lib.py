"""Build and load the CUDA library (libwsvd_b200.so) and describe its C ABI to ctypes.

The library is compiled in-tree with nvcc for sm_100a only.  There is no fallback: if
the shared object cannot be built or loaded, importing an op raises.
"""
from __future__ import annotations

import ctypes
import os
import shutil
import struct
import subprocess
import sys
import threading
import warnings

_PKG = os.path.dirname(os.path.abspath(__file__))
_ROOT = os.path.dirname(_PKG)
_CSRC = os.path.join(_PKG, "csrc")
_INCLUDE = os.path.join(_ROOT, "include")
LIB_PATH = os.path.join(_PKG, "libwsvd_b200.so")
NO_BIND = (ImportError, OSError, RuntimeError)  # what building or loading csrc/bind.cpp's module fails with

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared", "--threads", "0",
]

_lock = threading.Lock()
_lib = None


def sources():
    return sorted(os.path.join(_CSRC, f) for f in os.listdir(_CSRC) if f.endswith(".cu"))


def _deps():
    hdr = [os.path.join(_CSRC, f) for f in os.listdir(_CSRC) if f.endswith((".cuh", ".h"))]
    return sources() + hdr + [os.path.join(_INCLUDE, "wsvd_b200.h")]


def _bind_deps():
    return [os.path.join(_CSRC, "bind.cpp"), os.path.join(_INCLUDE, "wsvd_b200.h")]


def _older(path, deps) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(f) > t for f in deps)


def bind_path() -> str:
    """csrc/bind.cpp's module: calls of the dense block's operators straight from torch tensors.  It is made for one Python and one
    torch, which its name says."""
    import importlib.metadata

    try:
        torch = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError as e:
        raise ImportError("csrc/bind.cpp needs torch") from e
    return os.path.join(_PKG, f"_bind.{sys.implementation.cache_tag}-torch{torch}.so")


def _bind_command(out):
    """The compiler call for csrc/bind.cpp: a Python module on torch's headers and libraries."""
    import importlib.util
    import sysconfig

    spec = importlib.util.find_spec("torch")
    if spec is None:
        raise ImportError("csrc/bind.cpp needs torch")
    torch = spec.submodule_search_locations[0]
    cuda = os.environ.get("CUDA_HOME") or "/usr/local/cuda"
    include = [_INCLUDE, os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    libs = os.path.join(torch, "lib")
    return [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", *(f"-I{d}" for d in include),
            os.path.join(_CSRC, "bind.cpp"), "-o", out, f"-L{libs}", f"-Wl,-rpath,{libs}", "-ltorch_python", "-ltorch_cpu", "-lc10",
            "-lc10_cuda"]


def _made(path, deps, force, make) -> str:
    """`path`, made by make(temporary name) where it is missing, older than one of `deps` or `force`d.

    Safe when several processes start at once (one rank per GPU under torchrun): the
    staleness check, the compile and the rename happen under an inter-process file lock, the
    compiler writes to a per-process temporary name, and a process that gets the lock after
    another one has built finds the file fresh and returns."""
    import fcntl

    with _lock:
        if not force and not _older(path, deps()):
            return path
        with open(path + ".lock", "w") as lockfile:
            fcntl.flock(lockfile, fcntl.LOCK_EX)
            tmp = f"{path}.{os.getpid()}.tmp"
            try:
                if force or _older(path, deps()):
                    make(tmp)
                    os.replace(tmp, path)
            finally:
                if os.path.exists(tmp):
                    os.remove(tmp)
                fcntl.flock(lockfile, fcntl.LOCK_UN)
        return path


def _compile_lib(verbose):
    def make(tmp):
        nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
        if not os.path.exists(nvcc):
            raise RuntimeError("nvcc not found: cannot build libwsvd_b200.so")
        cmd = [nvcc, *NVCC_FLAGS, "-I", _INCLUDE, "-I", _CSRC, *sources(), "-o", tmp, "-lcuda"]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
        if verbose:
            print(res.stderr)

    return make


def _compile_bind(tmp):
    res = subprocess.run(_bind_command(tmp), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if res.returncode != 0:
        raise RuntimeError("the C++ compiler failed on csrc/bind.cpp:\n" + res.stdout)


def _build_bind(force: bool = False) -> str:
    return _made(bind_path(), _bind_deps, force, _compile_bind)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every .cu under csrc/ into one shared object for sm_100a, and csrc/bind.cpp into a Python module.

    The module needs a C++ compiler and torch's headers; without them the library is all there is, and calls go through
    ctypes (a warning says so)."""
    path = _made(LIB_PATH, _deps, force, _compile_lib(verbose))
    try:
        _build_bind(force)
    except NO_BIND as e:
        warnings.warn(f"csrc/bind.cpp was not built, calls go through ctypes: {e}", RuntimeWarning, stacklevel=2)
    return path


class LatentDecodeParams(ctypes.Structure):
    """ctypes mirror of WsvdLatentDecodeParams (include/wsvd_b200.h)."""

    _fields_ = [
        ("q", ctypes.c_void_p), ("q_stride_b", ctypes.c_int64), ("q_stride_h", ctypes.c_int64),
        ("latent_k", ctypes.c_void_p), ("k_stride_t", ctypes.c_int64), ("k_stride_h", ctypes.c_int64),
        ("k_scale", ctypes.c_void_p), ("ks_stride_t", ctypes.c_int64), ("ks_stride_h", ctypes.c_int64),
        ("latent_v", ctypes.c_void_p), ("v_stride_t", ctypes.c_int64), ("v_stride_h", ctypes.c_int64),
        ("v_scale", ctypes.c_void_p), ("vs_stride_t", ctypes.c_int64), ("vs_stride_h", ctypes.c_int64),
        ("wk", ctypes.c_void_p), ("wk_stride_r", ctypes.c_int64),
        ("wk_scale", ctypes.c_void_p),
        ("wv", ctypes.c_void_p), ("wv_stride_r", ctypes.c_int64),
        ("req_to_token", ctypes.c_void_p), ("rtt_stride", ctypes.c_int64),
        ("b_req_idx", ctypes.c_void_p),
        ("b_seq_len", ctypes.c_void_p),
        ("pos_offset", ctypes.c_void_p),
        ("out", ctypes.c_void_p), ("out_stride_b", ctypes.c_int64), ("out_stride_h", ctypes.c_int64),
        ("batch", ctypes.c_int32), ("n_q_heads", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32), ("rank_k", ctypes.c_int32), ("rank_v", ctypes.c_int32),
        ("max_len", ctypes.c_int32),
        ("latent_dtype", ctypes.c_int32), ("wk_dtype", ctypes.c_int32), ("rope_layout", ctypes.c_int32),
        ("split_len", ctypes.c_int32), ("kernel", ctypes.c_int32),
        ("theta", ctypes.c_float), ("sm_scale", ctypes.c_float),
        ("rope_table", ctypes.c_void_p), ("rope_table_rows", ctypes.c_int32),
        ("n_token_slots", ctypes.c_int64),
    ]


class DenseDecodeParams(ctypes.Structure):
    """ctypes mirror of WsvdDenseDecodeParams."""

    _fields_ = [
        ("q", ctypes.c_void_p), ("q_stride_b", ctypes.c_int64), ("q_stride_h", ctypes.c_int64),
        ("k", ctypes.c_void_p), ("k_stride_t", ctypes.c_int64), ("k_stride_h", ctypes.c_int64),
        ("v", ctypes.c_void_p), ("v_stride_t", ctypes.c_int64), ("v_stride_h", ctypes.c_int64),
        ("req_to_token", ctypes.c_void_p), ("rtt_stride", ctypes.c_int64),
        ("b_req_idx", ctypes.c_void_p), ("b_seq_len", ctypes.c_void_p),
        ("out", ctypes.c_void_p), ("out_stride_b", ctypes.c_int64), ("out_stride_h", ctypes.c_int64),
        ("batch", ctypes.c_int32), ("n_q_heads", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32), ("max_len", ctypes.c_int32), ("split_len", ctypes.c_int32),
        ("sm_scale", ctypes.c_float),
    ]


class QuantAppendParams(ctypes.Structure):
    """ctypes mirror of WsvdQuantAppendParams."""

    _fields_ = [
        ("x_k", ctypes.c_void_p), ("xk_stride_b", ctypes.c_int64), ("xk_stride_h", ctypes.c_int64),
        ("x_v", ctypes.c_void_p), ("xv_stride_b", ctypes.c_int64), ("xv_stride_h", ctypes.c_int64),
        ("latent_k", ctypes.c_void_p), ("k_stride_t", ctypes.c_int64), ("k_stride_h", ctypes.c_int64),
        ("k_scale", ctypes.c_void_p), ("ks_stride_t", ctypes.c_int64), ("ks_stride_h", ctypes.c_int64),
        ("latent_v", ctypes.c_void_p), ("v_stride_t", ctypes.c_int64), ("v_stride_h", ctypes.c_int64),
        ("v_scale", ctypes.c_void_p), ("vs_stride_t", ctypes.c_int64), ("vs_stride_h", ctypes.c_int64),
        ("req_to_token", ctypes.c_void_p), ("rtt_stride", ctypes.c_int64),
        ("b_req_idx", ctypes.c_void_p), ("b_seq_len", ctypes.c_void_p),
        ("batch", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32), ("rank_k", ctypes.c_int32),
        ("rank_v", ctypes.c_int32), ("max_len", ctypes.c_int32), ("x_dtype", ctypes.c_int32),
    ]


class KvRopeAppendParams(ctypes.Structure):
    """ctypes mirror of WsvdKvRopeAppendParams."""

    _fields_ = [
        ("k", ctypes.c_void_p), ("k_stride_n", ctypes.c_int64), ("k_stride_h", ctypes.c_int64),
        ("v", ctypes.c_void_p), ("v_stride_n", ctypes.c_int64), ("v_stride_h", ctypes.c_int64),
        ("q", ctypes.c_void_p), ("q_stride_n", ctypes.c_int64), ("q_stride_h", ctypes.c_int64),
        ("q_out", ctypes.c_void_p), ("qo_stride_n", ctypes.c_int64), ("qo_stride_h", ctypes.c_int64),
        ("cache_k", ctypes.c_void_p), ("ck_stride_t", ctypes.c_int64), ("ck_stride_h", ctypes.c_int64),
        ("cache_v", ctypes.c_void_p), ("cv_stride_t", ctypes.c_int64), ("cv_stride_h", ctypes.c_int64),
        ("k_scale", ctypes.c_void_p), ("ks_stride_t", ctypes.c_int64), ("ks_stride_h", ctypes.c_int64),
        ("v_scale", ctypes.c_void_p), ("vs_stride_t", ctypes.c_int64), ("vs_stride_h", ctypes.c_int64),
        ("inv_freq", ctypes.c_void_p),
        ("req_to_token", ctypes.c_void_p), ("rtt_stride", ctypes.c_int64),
        ("b_req_idx", ctypes.c_void_p), ("b_seq_len", ctypes.c_void_p),
        ("cu_new", ctypes.c_void_p), ("pos_offset", ctypes.c_void_p),
        ("n_token_slots", ctypes.c_int64),
        ("rows", ctypes.c_int32), ("batch", ctypes.c_int32), ("n_q_heads", ctypes.c_int32),
        ("n_kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("rot_dim", ctypes.c_int32),
        ("max_len", ctypes.c_int32), ("n_req", ctypes.c_int32),
        ("dtype", ctypes.c_int32), ("cache_dtype", ctypes.c_int32), ("rope_layout", ctypes.c_int32),
        ("clear_tail", ctypes.c_int32),
    ]


class PagedDecodeParams(ctypes.Structure):
    """ctypes mirror of WsvdPagedDecodeParams."""

    _fields_ = [
        ("q", ctypes.c_void_p), ("q_stride_b", ctypes.c_int64), ("q_stride_h", ctypes.c_int64),
        ("k", ctypes.c_void_p), ("k_stride_t", ctypes.c_int64), ("k_stride_h", ctypes.c_int64),
        ("v", ctypes.c_void_p), ("v_stride_t", ctypes.c_int64), ("v_stride_h", ctypes.c_int64),
        ("k_scale", ctypes.c_void_p), ("ks_stride_t", ctypes.c_int64), ("ks_stride_h", ctypes.c_int64),
        ("v_scale", ctypes.c_void_p), ("vs_stride_t", ctypes.c_int64), ("vs_stride_h", ctypes.c_int64),
        ("req_to_token", ctypes.c_void_p), ("rtt_stride", ctypes.c_int64),
        ("b_req_idx", ctypes.c_void_p), ("b_seq_len", ctypes.c_void_p),
        ("out", ctypes.c_void_p), ("out_stride_b", ctypes.c_int64), ("out_stride_h", ctypes.c_int64),
        ("lse", ctypes.c_void_p),
        ("n_token_slots", ctypes.c_int64),
        ("batch", ctypes.c_int32), ("n_q_heads", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32), ("max_len", ctypes.c_int32), ("n_req", ctypes.c_int32),
        ("dtype", ctypes.c_int32), ("cache_dtype", ctypes.c_int32), ("window", ctypes.c_int32),
        ("sm_scale", ctypes.c_float),
    ]


class AdapterAddParams(ctypes.Structure):
    """ctypes mirror of WsvdAdapterAddParams."""

    _fields_ = [
        ("y", ctypes.c_void_p), ("y_stride", ctypes.c_int64),
        ("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64),
        ("a", ctypes.c_void_p), ("a_stride_i", ctypes.c_int64), ("a_stride_k", ctypes.c_int64),
        ("b", ctypes.c_void_p), ("b_stride_i", ctypes.c_int64), ("b_stride_r", ctypes.c_int64),
        ("out", ctypes.c_void_p), ("out_stride", ctypes.c_int64),
        ("adapter", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("cu_new", ctypes.c_void_p),
        ("rows", ctypes.c_int32), ("batch", ctypes.c_int32), ("n_in", ctypes.c_int32), ("n_out", ctypes.c_int32),
        ("rank", ctypes.c_int32), ("n_adapters", ctypes.c_int32), ("dtype", ctypes.c_int32),
        ("copy_tail", ctypes.c_int32),
    ]


def packer(cls):
    """A function of a structure's fields, in order, that gives the structure's bytes (pointers as whole numbers, 0 for
    none): a tenth of the time that filling the ctypes structure takes, which is most of a small call's."""
    code = {ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_float: "f"}
    s = struct.Struct("@" + "".join(code[t] for _, t in cls._fields_))
    assert s.size <= ctypes.sizeof(cls) < s.size + 8  # C pads the end to the widest field, struct does not
    s = struct.Struct(s.format + f"{ctypes.sizeof(cls) - s.size}x")
    return s.pack


MAX_PEERS = 8
PEER_HANDLE_BYTES = 64


class PeerSet(ctypes.Structure):
    """ctypes mirror of WsvdPeerSet."""

    _fields_ = [
        ("out", ctypes.c_void_p * MAX_PEERS), ("flags", ctypes.c_void_p * MAX_PEERS), ("counter", ctypes.c_void_p),
        ("n_peers", ctypes.c_int32), ("rank", ctypes.c_int32), ("head_offset", ctypes.c_int32),
        ("epoch", ctypes.c_uint32), ("out_stride_b", ctypes.c_int64), ("out_stride_h", ctypes.c_int64),
        ("timeout_ms", ctypes.c_int32), ("epoch_counter", ctypes.c_void_p),
    ]


# name -> (restype, argtypes); every symbol include/wsvd_b200.h declares
_P = ctypes.POINTER(LatentDecodeParams)
SYMBOLS = {
    "wsvd_abi_version": (ctypes.c_int, []),
    "wsvd_status_string": (ctypes.c_char_p, [ctypes.c_int]),
    "wsvd_last_cuda_error": (ctypes.c_int, []),
    "wsvd_rope_table_bytes": (ctypes.c_size_t, [ctypes.c_int32, ctypes.c_int32]),
    "wsvd_rope_table_init": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int32, ctypes.c_int32,
                                            ctypes.c_float, ctypes.c_void_p]),
    "wsvd_kernel_status": (ctypes.c_int, [ctypes.POINTER(ctypes.c_uint32)]),
    "wsvd_kernel_status_reset": (ctypes.c_int, []),
    "wsvd_latent_decode_plan": (ctypes.c_int, [_P, ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(ctypes.c_int32)]),
    "wsvd_latent_decode_workspace_bytes": (ctypes.c_size_t, [_P]),
    "wsvd_latent_decode": (ctypes.c_int, [_P, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "wsvd_share_begin": (ctypes.c_int64, [ctypes.c_int32, ctypes.c_int64, ctypes.c_int32]),
    "wsvd_share_owner": (ctypes.c_int32, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32]),
    "wsvd_latent_decode_partials": (ctypes.c_int, [_P, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "wsvd_dense_decode_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(DenseDecodeParams)]),
    "wsvd_dense_decode_f16": (ctypes.c_int, [ctypes.POINTER(DenseDecodeParams), ctypes.c_void_p, ctypes.c_size_t,
                                             ctypes.c_void_p]),
    "wsvd_latent_decode_static": (ctypes.c_int, [_P, ctypes.c_void_p]),
    "wsvd_latent_decode_gather": (ctypes.c_int, [_P, ctypes.POINTER(PeerSet), ctypes.c_void_p, ctypes.c_size_t,
                                                 ctypes.c_void_p]),
    "wsvd_peer_alloc": (ctypes.c_int, [ctypes.c_size_t, ctypes.POINTER(ctypes.c_void_p)]),
    "wsvd_peer_free": (ctypes.c_int, [ctypes.c_void_p]),
    "wsvd_peer_export": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_char_p]),
    "wsvd_peer_import": (ctypes.c_int, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_void_p)]),
    "wsvd_peer_release": (ctypes.c_int, [ctypes.c_void_p]),
    "wsvd_latent_quant_append_i8": (ctypes.c_int, [ctypes.POINTER(QuantAppendParams), ctypes.c_void_p]),
    # (c_void_p: the bytes of a packed structure, or byref of one)
    "wsvd_kv_rope_append": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "wsvd_paged_decode_workspace_bytes": (ctypes.c_size_t, [ctypes.c_void_p]),
    "wsvd_paged_decode": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "wsvd_adapter_add_workspace_bytes": (ctypes.c_size_t, [ctypes.c_void_p]),
    "wsvd_adapter_add": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "wsvd_rms_norm_f16": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32,
                                         ctypes.c_float, ctypes.c_void_p]),
    "wsvd_add_rms_norm_f16": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                             ctypes.c_int32, ctypes.c_int32, ctypes.c_float, ctypes.c_void_p]),
    "wsvd_rope_half_f16": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p,
                                          ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
    "wsvd_silu_mul_f16": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64,
                                         ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
    "wsvd_latent_decode_stage1": (ctypes.c_int, [_P, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p]),
    "wsvd_decode_stage2": (ctypes.c_int, [
        ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64,
        ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
        ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
}


def lib() -> ctypes.CDLL:
    """The loaded library; builds it first if the shared object is missing or stale."""
    global _lib
    if _lib is None:
        _made(LIB_PATH, _deps, False, _compile_lib(False))
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SYMBOLS.items():
            fn = getattr(handle, name)  # AttributeError if the symbol is missing
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


_bind = None


def bind():
    """The module of csrc/bind.cpp, connected to the library's entries; builds both first where they are missing or stale.
    Raises one of NO_BIND where there is no such module to be had."""
    global _bind
    if _bind is None:
        import importlib.util

        import torch  # noqa: F401  (the module's libraries)

        handle = lib()
        spec = importlib.util.spec_from_file_location("wsvd_b200._bind", _build_bind())
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.connect(*(ctypes.cast(getattr(handle, f"wsvd_{n}"), ctypes.c_void_p).value for n in
                         ("kv_rope_append", "paged_decode_workspace_bytes", "paged_decode", "adapter_add_workspace_bytes",
                          "adapter_add")))
        _bind = module
    return _bind


class WsvdError(RuntimeError):
    """A C entry point returned a nonzero status."""

    def __init__(self, status: int, where: str):
        self.status = status
        msg = lib().wsvd_status_string(status).decode()
        if status == 6:
            msg += f" [cudaError {lib().wsvd_last_cuda_error()}]"
        super().__init__(f"{where}: {msg} (status {status})")


def check(status: int, where: str) -> None:
    if status != 0:
        raise WsvdError(status, where)
