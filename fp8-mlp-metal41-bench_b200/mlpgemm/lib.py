"""ctypes binding of libgemm.so (the C ABI declared in include/mlpgemm.h).

The library is the product: there is no fallback.  If libgemm.so is missing
or cannot be loaded, every entry point here raises GemmError.
"""
from __future__ import annotations

import ctypes
import operator
import os
import struct
import subprocess
import threading

PKG_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.environ.get("GEMM_LIB", os.path.join(PKG_ROOT, "libgemm.so"))

GEMM_OK, GEMM_ERR_ARGS, GEMM_ERR_INIT, GEMM_ERR_MISMATCH, GEMM_ERR_CUDA, GEMM_ERR_TIMEOUT = range(6)

# Every symbol the header declares (tests check the library exports them all).
EXPORTS = [
    "gemm_init", "gemm_device_count", "gemm_device_info", "gemm_last_error", "gemm_version",
    "gemm_dtype_name", "gemm_kernel_name", "gemm_num_tiles", "gemm_tile_name",
    "gemm_tile_index", "gemm_tile_supported", "gemm_default_tile", "gemm_check_layout",
    "gemm_workspace_size", "gemm_alloc", "gemm_free", "gemm_memset", "gemm_h2d", "gemm_d2h",
    "gemm_host_alloc", "gemm_host_free", "gemm_run", "gemm_sync", "gemm_time",
    "gemm_time_e2e", "gemm_time_e2e_pipelined", "gemm_launches_per_run", "gemm_peak_probe",
    "gemm_read_probe",
    "gemm_run_noalloc",
    "gemm_quantize",
    "gemm_linear", "gemm_linear_dx", "gemm_linear_dw", "gemm_linear_workspace", "gemm_act_grad", "gemm_dropout",
    "gemm_run_gather", "gemm_gather_supported", "gemm_peer_alloc", "gemm_peer_open", "gemm_peer_close",
]

MAX_PEERS = 7            # GEMM_MAX_PEERS
PEER_HANDLE_BYTES = 64   # GEMM_PEER_HANDLE_BYTES

# quantiser formats (GEMM_Q_* in include/mlpgemm.h)
Q_E4M3_REF, Q_E4M3, Q_E2M1, Q_MXFP4, Q_MXFP8 = 0, 1, 2, 3, 4

# the MLP layer's operand types (GEMM_TYPE_*), activations (GEMM_ACT_*) and products (GEMM_OP_*)
TYPES = {"f16": 0, "bf16": 1, "f32": 2}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
OP_LINEAR, OP_DX, OP_DW = 0, 1, 2


# gemm_dropout_args and gemm_epilogue, packed for one call (a few times cheaper than ctypes structures)
DROPOUT_ARGS = struct.Struct("=dQQQ")                 # p, seed, offset, offset_ptr
EPILOGUE = struct.Struct("=QQqQqi4xdQQQ")             # bias, residual, ldr, preact, ldz, act, dropout
_U64 = (1 << 64) - 1


class GemmError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"[{code}] {msg}")
        self.code = code


_lib = None
_lock = threading.Lock()


def build() -> str:
    """Compile libgemm.so in-tree with the package Makefile (nvcc, sm_100a)."""
    subprocess.run(["make", "-s", "-C", PKG_ROOT], check=True)
    return LIB_PATH


def _declare(L):
    c_int, c_size, vp, c_char_p = ctypes.c_int, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_char_p
    c_long = ctypes.c_long
    vpp = ctypes.POINTER(ctypes.c_void_p)
    sig = {
        "gemm_init": (c_int, [c_int]),
        "gemm_device_count": (c_int, []),
        "gemm_device_info": (c_int, [c_int, c_char_p, c_int, c_char_p, c_int, ctypes.POINTER(c_int)]),
        "gemm_last_error": (c_char_p, []),
        "gemm_version": (c_char_p, []),
        "gemm_dtype_name": (c_char_p, [c_int]),
        "gemm_kernel_name": (c_char_p, [c_int]),
        "gemm_num_tiles": (c_int, []),
        "gemm_tile_name": (c_char_p, [c_int]),
        "gemm_tile_index": (c_int, [c_char_p]),
        "gemm_tile_supported": (c_int, [c_int, c_int, c_int, c_int, c_int]),
        "gemm_default_tile": (c_int, [c_int, c_int, c_int, c_int]),
        "gemm_check_layout": (c_int, [c_int, c_int, c_int, c_int]),
        "gemm_workspace_size": (c_size, [c_int, c_int, c_int, c_int, c_int]),
        "gemm_alloc": (vp, [c_int, c_size]),
        "gemm_free": (c_int, [c_int, vp]),
        "gemm_memset": (c_int, [c_int, vp, c_int, c_size]),
        "gemm_h2d": (c_int, [c_int, vp, vp, c_size]),
        "gemm_d2h": (c_int, [c_int, vp, vp, c_size]),
        "gemm_host_alloc": (vp, [c_size]),
        "gemm_host_free": (c_int, [vp]),
        "gemm_run": (c_int, [c_int, c_int, c_int, vp, vp, vp, c_int, c_int, c_int, vp, vp, vp,
                             c_size, vp]),
        "gemm_sync": (c_int, [c_int, vp]),
        "gemm_time": (c_int, [c_int, c_int, c_int, vp, vpp, vp, c_int, c_int, c_int, vp, vpp,
                              c_int, vp, c_size, c_int, c_int, vp, c_size,
                              ctypes.POINTER(ctypes.c_float)]),
        "gemm_time_e2e": (c_int, [c_int, c_int, c_int, vp, vp, vp, vp, vp, c_int, c_int, c_int,
                                  vp, vp, vp, vp, c_size, c_int, c_int,
                                  ctypes.POINTER(ctypes.c_float)]),
        "gemm_time_e2e_pipelined": (c_int, [c_int, c_int, c_int, vp, vp, vp, vp, vp, vp, vp, c_int, c_int,
                                            c_int, vp, vp, vp, vp, vp, c_size, c_int, c_int,
                                            ctypes.POINTER(ctypes.c_float)]),
        "gemm_launches_per_run": (c_int, [c_int, c_int, c_int, c_int, c_int]),
        "gemm_peak_probe": (c_int, [c_int, c_int, c_int, c_int, ctypes.POINTER(ctypes.c_double)]),
        "gemm_read_probe": (c_int, [c_int, vp, c_size, c_int, c_int, vp, c_size,
                                    ctypes.POINTER(ctypes.c_float)]),
        "gemm_run_noalloc": (c_int, [c_int, c_int, c_int, vp, vp, vp, c_int, c_int, c_int, vp, vp,
                                     vp]),
        "gemm_quantize": (c_int, [c_int, c_int, vp, vp, vp, ctypes.c_long, ctypes.c_long, vp]),
        "gemm_linear": (c_int, [c_int, c_int, vp, c_long, vp, c_long, vp, c_long, c_int, c_int, c_int, vp, vp,
                                c_size, vp]),
        "gemm_linear_dx": (c_int, [c_int, c_int, vp, c_long, vp, c_long, vp, c_long, c_int, c_int, c_int, vp,
                                   c_long, vp, c_size, vp]),
        "gemm_linear_dw": (c_int, [c_int, c_int, vp, c_long, vp, c_long, vp, c_int, c_long, c_int, c_int, c_int,
                                   vp, c_long, vp, c_size, vp]),
        "gemm_linear_workspace": (c_size, [c_int, vp, c_long, vp, c_long, c_int, c_int, c_int]),
        "gemm_act_grad": (c_int, [c_int, c_int, vp, c_long, vp, c_long, vp, c_long, vp, c_int, c_int, c_int, vp,
                                  vp]),
        "gemm_dropout": (c_int, [c_int, c_int, vp, c_long, vp, c_long, vp, c_long, c_int, c_int, vp, vp]),
        "gemm_run_gather": (c_int, [c_int, c_int, c_int, vp, vp, vp, c_int, c_int, c_int, vp, vp, vp,
                                    c_size, vpp, c_int, vp]),
        "gemm_gather_supported": (c_int, [c_int, c_int]),
        "gemm_peer_alloc": (c_int, [c_int, c_size, vpp, vp]),
        "gemm_peer_open": (c_int, [c_int, vp, vpp]),
        "gemm_peer_close": (c_int, [c_int, vp]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args


def lib() -> ctypes.CDLL:
    """Load libgemm.so (once).  Raises GemmError(GEMM_ERR_INIT) if it is absent."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise GemmError(GEMM_ERR_INIT,
                                f"{LIB_PATH} not found: build it with `make -C {PKG_ROOT}`")
            try:
                L = ctypes.CDLL(LIB_PATH)
            except OSError as e:
                raise GemmError(GEMM_ERR_INIT, f"cannot load {LIB_PATH}: {e}") from e
            _declare(L)
            _lib = L
    return _lib


def last_error() -> str:
    return lib().gemm_last_error().decode(errors="replace")


def check(rc: int, what: str = "") -> None:
    if rc != GEMM_OK:
        raise GemmError(rc, f"{what}: {last_error()}" if what else last_error())


def _s(b: bytes) -> str:
    return b.decode() if b is not None else ""


# ---- thin wrappers -------------------------------------------------------------
def init(device: int = 0) -> None:
    check(lib().gemm_init(device), f"gemm_init({device})")


def device_count() -> int:
    return lib().gemm_device_count()


def device_info(device: int = 0):
    name = ctypes.create_string_buffer(256)
    arch = ctypes.create_string_buffer(64)
    sms = ctypes.c_int(0)
    check(lib().gemm_device_info(device, name, 256, arch, 64, ctypes.byref(sms)), "device info")
    return name.value.decode(), arch.value.decode(), sms.value


def version() -> str:
    return _s(lib().gemm_version())


def tile_names() -> list[str]:
    L = lib()
    return [_s(L.gemm_tile_name(i)) for i in range(L.gemm_num_tiles())]


def tile_index(name: str) -> int:
    return lib().gemm_tile_index(name.encode())


def tile_supported(dtype: int, tile: int, N: int, K: int, M: int) -> bool:
    return bool(lib().gemm_tile_supported(dtype, tile, N, K, M))


def default_tile(dtype: int, N: int, K: int, M: int) -> int:
    return lib().gemm_default_tile(dtype, N, K, M)


def workspace_size(dtype: int, tile: int, N: int, K: int, M: int) -> int:
    return lib().gemm_workspace_size(dtype, tile, N, K, M)


def launches_per_run(dtype: int, tile: int, N: int, K: int, M: int) -> int:
    return lib().gemm_launches_per_run(dtype, tile, N, K, M)


class DeviceBuffer:
    """Device memory from gemm_alloc (freed on close / garbage collection)."""

    def __init__(self, device: int, nbytes: int):
        self.device = device
        self.nbytes = int(nbytes)
        p = lib().gemm_alloc(device, max(self.nbytes, 1))
        if not p:
            raise GemmError(GEMM_ERR_CUDA, f"gemm_alloc({nbytes}): {last_error()}")
        self.ptr = p

    def upload(self, arr) -> "DeviceBuffer":
        import numpy as np
        a = np.ascontiguousarray(arr)
        assert a.nbytes <= self.nbytes, (a.nbytes, self.nbytes)
        check(lib().gemm_h2d(self.device, self.ptr, a.ctypes.data_as(ctypes.c_void_p), a.nbytes), "h2d")
        return self

    def download(self, arr):
        import numpy as np
        assert arr.flags["C_CONTIGUOUS"] and arr.nbytes <= self.nbytes
        check(lib().gemm_d2h(self.device, arr.ctypes.data_as(ctypes.c_void_p), self.ptr, arr.nbytes),
              "d2h")
        return arr

    def zero(self) -> "DeviceBuffer":
        check(lib().gemm_memset(self.device, self.ptr, 0, self.nbytes), "memset")
        return self

    def close(self):
        if getattr(self, "ptr", None):
            try:
                lib().gemm_free(self.device, self.ptr)
            finally:
                self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def as_ptr(x):
    """Device pointer of a DeviceBuffer, a torch tensor, an int or None."""
    if x is None or type(x) is int:
        return x
    if isinstance(x, DeviceBuffer):
        return x.ptr
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    return int(x)


def run(device, dtype, tile, X, W, Y, N, K, M, xscale=None, wscale=None, workspace=None,
        workspace_bytes=0, stream=None) -> None:
    check(lib().gemm_run(device, dtype, tile, as_ptr(X), as_ptr(W), as_ptr(Y), N, K, M,
                         as_ptr(xscale), as_ptr(wscale), as_ptr(workspace), int(workspace_bytes),
                         as_ptr(stream)), "gemm_run")


def run_noalloc(device, dtype, ksplit, X, W, Y, N, K, M, xscale=None, wscale=None,
                stream=None) -> None:
    """Thin-row GEMM whose split-K scratch is the library's fixed device array
    (no allocation by the library or the caller; see gemm_run_noalloc)."""
    check(lib().gemm_run_noalloc(device, dtype, ksplit, as_ptr(X), as_ptr(W), as_ptr(Y), N, K, M,
                                 as_ptr(xscale), as_ptr(wscale), as_ptr(stream)),
          "gemm_run_noalloc")


def run_gather(device, dtype, tile, X, W, Y, N, K, M, xscale=None, wscale=None, workspace=None,
               workspace_bytes=0, peers=(), stream=None) -> None:
    """gemm_run whose epilogue also stores Y at the same offset from every
    pointer of `peers` (other GPUs' Y buffers mapped with peer_open)."""
    arr = (ctypes.c_void_p * max(1, len(peers)))(*[as_ptr(q) for q in peers])
    check(lib().gemm_run_gather(device, dtype, tile, as_ptr(X), as_ptr(W), as_ptr(Y), N, K, M,
                                as_ptr(xscale), as_ptr(wscale), as_ptr(workspace), int(workspace_bytes),
                                arr, len(peers), as_ptr(stream)), "gemm_run_gather")


def gather_supported(dtype: int, tile: int) -> bool:
    return bool(lib().gemm_gather_supported(dtype, tile))


def peer_alloc(device: int, nbytes: int):
    """(device pointer, IPC handle bytes) of a buffer other processes can map."""
    ptr = ctypes.c_void_p()
    h = ctypes.create_string_buffer(PEER_HANDLE_BYTES)
    check(lib().gemm_peer_alloc(device, int(nbytes), ctypes.byref(ptr), h), "gemm_peer_alloc")
    return int(ptr.value), bytes(h.raw)


def peer_open(device: int, handle: bytes) -> int:
    assert len(handle) == PEER_HANDLE_BYTES
    ptr = ctypes.c_void_p()
    h = ctypes.create_string_buffer(bytes(handle), PEER_HANDLE_BYTES)
    check(lib().gemm_peer_open(device, h, ctypes.byref(ptr)), "gemm_peer_open")
    return int(ptr.value)


def peer_close(device: int, ptr: int) -> None:
    check(lib().gemm_peer_close(device, ctypes.c_void_p(ptr)), "gemm_peer_close")


def free(device: int, ptr: int) -> None:
    check(lib().gemm_free(device, ctypes.c_void_p(ptr)), "gemm_free")


def sync(device: int = 0, stream=None) -> None:
    check(lib().gemm_sync(device, as_ptr(stream)), "gemm_sync")


def time(device, dtype, tile, X, Ws, Y, N, K, M, xscale=None, wscales=None, workspace=None,
         workspace_bytes=0, warmup=5, iters=100, flush=None, flush_bytes=0):
    """Per-iteration CUDA-event times (ms) of `iters` back-to-back GEMMs."""
    Ws = list(Ws) if isinstance(Ws, (list, tuple)) else [Ws]
    nrot = len(Ws)
    warr = (ctypes.c_void_p * nrot)(*[as_ptr(w) for w in Ws])
    if wscales is None:
        sarr = None
    else:
        wscales = list(wscales) if isinstance(wscales, (list, tuple)) else [wscales]
        assert len(wscales) == nrot
        sarr = (ctypes.c_void_p * nrot)(*[as_ptr(s) for s in wscales])
    out = (ctypes.c_float * iters)()
    check(lib().gemm_time(device, dtype, tile, as_ptr(X), warr, as_ptr(Y), N, K, M, as_ptr(xscale),
                          sarr, nrot, as_ptr(workspace), int(workspace_bytes), warmup, iters,
                          as_ptr(flush), int(flush_bytes), out), "gemm_time")
    return list(out)


def time_e2e(device, dtype, tile, hX, dX, dW, dY, hY, N, K, M, hxscale=None, dxscale=None,
             dwscale=None, workspace=None, workspace_bytes=0, warmup=3, iters=10):
    out = (ctypes.c_float * iters)()
    check(lib().gemm_time_e2e(device, dtype, tile, as_ptr(hX), as_ptr(dX), as_ptr(dW), as_ptr(dY),
                              as_ptr(hY), N, K, M, as_ptr(hxscale), as_ptr(dxscale),
                              as_ptr(dwscale), as_ptr(workspace), int(workspace_bytes), warmup,
                              iters, out), "gemm_time_e2e")
    return list(out)


def time_e2e_pipelined(device, dtype, tile, hX, dX, dW, dY, hY, N, K, M, hxscale=None, dxscale=(None, None),
                       dwscale=None, workspace=None, workspace_bytes=0, warmup=3, iters=10) -> float:
    """Total ms of `iters` end-to-end steps overlapped two deep; dX, dY (and
    dxscale) are pairs of device buffers used in turn."""
    out = ctypes.c_float(0.0)
    check(lib().gemm_time_e2e_pipelined(device, dtype, tile, as_ptr(hX), as_ptr(dX[0]), as_ptr(dX[1]),
                                        as_ptr(dW), as_ptr(dY[0]), as_ptr(dY[1]), as_ptr(hY), N, K, M,
                                        as_ptr(hxscale), as_ptr(dxscale[0]), as_ptr(dxscale[1]),
                                        as_ptr(dwscale), as_ptr(workspace), int(workspace_bytes), warmup,
                                        iters, ctypes.byref(out)), "gemm_time_e2e_pipelined")
    return out.value


def peak_probe(device: int, kind: int, reps: int = 4096, iters: int = 10) -> float:
    v = ctypes.c_double(0.0)
    check(lib().gemm_peak_probe(device, kind, reps, iters, ctypes.byref(v)), "gemm_peak_probe")
    return v.value


def read_probe(device: int, buf, nbytes: int, warmup: int = 3, iters: int = 20, flush=None,
               flush_bytes: int = 0) -> list:
    """CUDA-event times (ms) of a plain streaming read of `nbytes` of `buf`."""
    out = (ctypes.c_float * iters)()
    check(lib().gemm_read_probe(device, as_ptr(buf), int(nbytes), warmup, iters, as_ptr(flush),
                                int(flush_bytes), out), "gemm_read_probe")
    return list(out)


def quantize(device, fmt, src, dst, scales=None, rows=1, cols=1, stream=None) -> None:
    """f32 [rows, cols] on the device -> a GEMM_Q_* format in `dst` (+ UE8M0 `scales`)."""
    check(lib().gemm_quantize(device, fmt, as_ptr(src), as_ptr(dst), as_ptr(scales), int(rows), int(cols),
                              as_ptr(stream)), "gemm_quantize")


# ---- the MLP layer (f16 / bf16 operands; see the header for the formulas) -----------------
# What the C side can't see of a torch tensor or DeviceBuffer is checked here: a host tensor, another
# GPU's, or one that is smaller or laid out otherwise than the call takes it for would have the kernels
# read or write where they must not.
_dtypes = {}    # GEMM_TYPE_* -> torch dtype, once a torch tensor has been seen
_layer = {}     # the entry points without argtypes, whose conversion takes 0.1 us per argument:
                # pointers, longs and sizes go in as ctypes objects, the rest are ints of 32 bits

_VP, _LONG, _SIZE = ctypes.c_void_p, ctypes.c_long, ctypes.c_size_t
_LONG0, _SIZE0 = _LONG(0), _SIZE(0)


def _refuse(name: str, why: str):
    raise GemmError(GEMM_ERR_ARGS, f"{name} {why}")


def _bind(name):
    fn = _layer[name] = lib()[name]
    return fn


def _ints(*values):
    """The same as Python's own ints, which ctypes would cut to 32 bits without a word."""
    values = [operator.index(v) for v in values]
    for v in values:
        if not -(1 << 31) <= v < 1 << 31:
            _refuse(f"size {v}", "does not fit an int")
    return values


def _on(device, name, x):
    """Address of a buffer on `device`."""
    if x is None or x.__class__ is int:
        return x
    if hasattr(x, "get_device"):
        if x.get_device() != device:
            _refuse(name, f"is on {x.device}, not on device {device}")
        return x.data_ptr()
    if isinstance(x, DeviceBuffer) and x.device != device:
        _refuse(name, f"is on device {x.device}, not on device {device}")
    return as_ptr(x)


def _matrix(x, dtype, device, type, rows, cols, ld, name):
    """Address of rows x cols elements of `type` (torch's `dtype`), `ld` from row to row (0: dense)."""
    if x is None or x.__class__ is int:
        return x
    try:   # the usual case
        if (x.dtype is dtype and x.get_device() == device and x.is_contiguous()
                and x.numel() >= (rows - 1) * (ld or cols) + cols):
            return x.data_ptr()
    except AttributeError:
        pass
    need = (rows - 1) * (ld or cols) + cols
    if hasattr(x, "get_device"):
        if not _dtypes:
            import torch
            _dtypes.update({TYPES["f16"]: torch.float16, TYPES["bf16"]: torch.bfloat16, TYPES["f32"]: torch.float32})
        if x.dtype is not _dtypes.get(type):
            _refuse(name, f"has elements of {x.dtype}, not of type {type}")
        if x.is_contiguous():
            if x.numel() < need:
                _refuse(name, f"has {x.numel()} elements, {need} needed")
        elif x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1) or x.stride(0) != (ld or cols):
            _refuse(name, f"of strides {tuple(x.stride())} does not have rows {ld or cols} elements apart")
        elif x.shape[0] < rows or x.shape[1] < cols:
            _refuse(name, f"is {tuple(x.shape)}, {rows} x {cols} needed")
    elif isinstance(x, DeviceBuffer) and x.nbytes < need * (4 if type == TYPES["f32"] else 2):
        _refuse(name, f"has {x.nbytes} bytes, {need} elements needed")
    return _on(device, name, x)


def _scratch(device, x, nbytes):
    """Workspace address and bytes as the C side takes them."""
    if x is None and not nbytes:
        return None, _SIZE0
    if hasattr(x, "get_device"):
        have = x.numel() * x.element_size()
    else:
        have = x.nbytes if isinstance(x, DeviceBuffer) else nbytes
    if have < nbytes:
        _refuse("workspace", f"has {have} bytes, {nbytes} given")
    return _VP(_on(device, "workspace", x)), _SIZE(int(nbytes))


def _dropout(device, p, seed, offset, offset_ptr) -> bytes:
    return DROPOUT_ARGS.pack(p, seed & _U64, offset & _U64, _on(device, "offset_ptr", offset_ptr) or 0)


def linear_workspace(op: int, A, B, N: int, K: int, M: int, lda: int = 0, ldb: int = 0) -> int:
    """Workspace bytes of a product: A, B are X, W (OP_LINEAR), dZ, W (OP_DX) or X, dZ (OP_DW)."""
    N, K, M = _ints(N, K, M)
    return lib().gemm_linear_workspace(op, as_ptr(A), lda, as_ptr(B), ldb, N, K, M)


def linear(device, type, X, W, Y, N, K, M, bias=None, act=0, residual=None, preact=None, dropout_p=0.0, seed=0,
           offset=0, offset_ptr=None, ldx=0, ldw=0, ldy=0, ldr=0, ldz=0, workspace=None, workspace_bytes=0,
           stream=None) -> None:
    """Y = residual + dropout(act(X @ W + bias)); preact receives X @ W + bias.  Row lengths 0: dense."""
    all_ = N | K | M | device | type
    if all_.__class__ is not int or all_ >> 31:
        device, type, N, K, M = _ints(device, type, N, K, M)
    dt = _dtypes.get(type)
    ws, wsb = _scratch(device, workspace, workspace_bytes)
    epi = EPILOGUE.pack(_matrix(bias, dt, device, type, 1, M, 0, "bias") or 0,
                        _matrix(residual, dt, device, type, N, M, ldr, "residual") or 0, ldr,
                        _matrix(preact, dt, device, type, N, M, ldz, "preact") or 0, ldz, act, dropout_p,
                        seed & _U64, offset & _U64, _on(device, "offset_ptr", offset_ptr) or 0)
    rc = (_layer.get("gemm_linear") or _bind("gemm_linear"))(
        device, type, _VP(_matrix(X, dt, device, type, N, K, ldx, "X")), _LONG(ldx) if ldx else _LONG0,
        _VP(_matrix(W, dt, device, type, K, M, ldw, "W")), _LONG(ldw) if ldw else _LONG0,
        _VP(_matrix(Y, dt, device, type, N, M, ldy, "Y")), _LONG(ldy) if ldy else _LONG0, N, K, M, epi, ws, wsb,
        _VP(as_ptr(stream)))
    if rc:
        check(rc, "gemm_linear")


def linear_dx(device, type, dZ, W, dX, N, K, M, residual=None, lddz=0, ldw=0, lddx=0, ldr=0, workspace=None,
              workspace_bytes=0, stream=None) -> None:
    """dX = residual + dZ @ W^T."""
    all_ = N | K | M | device | type
    if all_.__class__ is not int or all_ >> 31:
        device, type, N, K, M = _ints(device, type, N, K, M)
    dt = _dtypes.get(type)
    ws, wsb = _scratch(device, workspace, workspace_bytes)
    rc = (_layer.get("gemm_linear_dx") or _bind("gemm_linear_dx"))(
        device, type, _VP(_matrix(dZ, dt, device, type, N, M, lddz, "dZ")), _LONG(lddz) if lddz else _LONG0,
        _VP(_matrix(W, dt, device, type, K, M, ldw, "W")), _LONG(ldw) if ldw else _LONG0,
        _VP(_matrix(dX, dt, device, type, N, K, lddx, "dX")), _LONG(lddx) if lddx else _LONG0, N, K, M,
        _VP(_matrix(residual, dt, device, type, N, K, ldr, "residual")), _LONG(ldr) if ldr else _LONG0, ws, wsb,
        _VP(as_ptr(stream)))
    if rc:
        check(rc, "gemm_linear_dx")


def linear_dw(device, type, X, dZ, dW, N, K, M, out_type=None, residual=None, ldx=0, lddz=0, lddw=0, ldr=0,
              workspace=None, workspace_bytes=0, stream=None) -> None:
    """dW = residual + X^T @ dZ, of `out_type` (default: the operands' type)."""
    out = type if out_type is None else out_type
    all_ = N | K | M | device | type | out
    if all_.__class__ is not int or all_ >> 31:
        device, type, out, N, K, M = _ints(device, type, out, N, K, M)
    dt, dto = _dtypes.get(type), _dtypes.get(out)
    ws, wsb = _scratch(device, workspace, workspace_bytes)
    rc = (_layer.get("gemm_linear_dw") or _bind("gemm_linear_dw"))(
        device, type, _VP(_matrix(X, dt, device, type, N, K, ldx, "X")), _LONG(ldx) if ldx else _LONG0,
        _VP(_matrix(dZ, dt, device, type, N, M, lddz, "dZ")), _LONG(lddz) if lddz else _LONG0,
        _VP(_matrix(dW, dto, device, out, K, M, lddw, "dW")), out, _LONG(lddw) if lddw else _LONG0, N, K, M,
        _VP(_matrix(residual, dto, device, out, K, M, ldr, "residual")), _LONG(ldr) if ldr else _LONG0, ws, wsb,
        _VP(as_ptr(stream)))
    if rc:
        check(rc, "gemm_linear_dw")


def act_grad(device, type, dY, Z, dZ, dbias, N, M, act=0, dropout_p=0.0, seed=0, offset=0, offset_ptr=None,
             lddy=0, ldz=0, lddz=0, stream=None) -> None:
    """dZ = dropout(dY) * act'(Z); dbias (f32) = its column sums."""
    all_ = N | M | device | type | act
    if all_.__class__ is not int or all_ >> 31:
        device, type, act, N, M = _ints(device, type, act, N, M)
    dt = _dtypes.get(type)
    drop = _dropout(device, dropout_p, seed, offset, offset_ptr)
    rc = (_layer.get("gemm_act_grad") or _bind("gemm_act_grad"))(
        device, type, _VP(_matrix(dY, dt, device, type, N, M, lddy, "dY")), _LONG(lddy) if lddy else _LONG0,
        _VP(_matrix(Z, dt, device, type, N, M, ldz, "Z")), _LONG(ldz) if ldz else _LONG0,
        _VP(_matrix(dZ, dt, device, type, N, M, lddz, "dZ")), _LONG(lddz) if lddz else _LONG0,
        _VP(_matrix(dbias, _dtypes.get(2), device, 2, 1, M, 0, "dbias")), N, M, act, drop, _VP(as_ptr(stream)))
    if rc:
        check(rc, "gemm_act_grad")


def dropout(device, type, X, Y, N, M, p, seed, offset, offset_ptr=None, residual=None, ldx=0, ldr=0, ldy=0,
            stream=None) -> None:
    """Y = residual + dropout(X); on dY the same call is its gradient."""
    all_ = N | M | device | type
    if all_.__class__ is not int or all_ >> 31:
        device, type, N, M = _ints(device, type, N, M)
    dt = _dtypes.get(type)
    drop = _dropout(device, p, seed, offset, offset_ptr)
    rc = (_layer.get("gemm_dropout") or _bind("gemm_dropout"))(
        device, type, _VP(_matrix(X, dt, device, type, N, M, ldx, "X")), _LONG(ldx) if ldx else _LONG0,
        _VP(_matrix(residual, dt, device, type, N, M, ldr, "residual")), _LONG(ldr) if ldr else _LONG0,
        _VP(_matrix(Y, dt, device, type, N, M, ldy, "Y")), _LONG(ldy) if ldy else _LONG0, N, M, drop,
        _VP(as_ptr(stream)))
    if rc:
        check(rc, "gemm_dropout")
