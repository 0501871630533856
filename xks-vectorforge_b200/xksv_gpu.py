"""ctypes binding of libxksv_cuda.so (include/xksv_cuda.h).

``load()`` returns the CDLL with the argument types the reference's own
callers declare for the five GPU entry points (python/runtime.py:40-44 and
251-255, python/tune.py:16-19, tests/test_cuda.py:11-12, 24-25, 35-36, 48-49,
66-67), plus the batched plan interface.  ``Plan`` wraps a plan for torch
callers.  There is no fallback: a missing library raises.
"""
import ctypes
import os
import struct
from pathlib import Path

HERE = Path(__file__).resolve().parent
DEFAULT_LIB = HERE / "libxksv_cuda.so"

CODEC_RAW, CODEC_TILE16, CODEC_PARALLEL32 = 0, 1, 2
CODEC_BY_NAME = {"raw": CODEC_RAW, "bf16-huffman-tile16": CODEC_TILE16,
                 "bf16-huffman-parallel32": CODEC_PARALLEL32}


class Slab(ctypes.Structure):
    _fields_ = [("src_offset", ctypes.c_uint64), ("src_size", ctypes.c_uint64),
                ("rows", ctypes.c_uint64), ("cols", ctypes.c_uint64),
                ("dst_offset", ctypes.c_uint64), ("x_offset", ctypes.c_uint64),
                ("codec", ctypes.c_uint32), ("flags", ctypes.c_uint32)]


class KvDesc(ctypes.Structure):
    """xksv_kv_desc."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_bytes", ctypes.c_uint64),
                ("v_bytes", ctypes.c_uint64), ("pages", ctypes.c_uint64), ("page_size", ctypes.c_uint64),
                ("k_stride", ctypes.c_uint64 * 3), ("v_stride", ctypes.c_uint64 * 3), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("kv_heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32),
                ("type", ctypes.c_uint32), ("flags", ctypes.c_uint32)]


# Argument blocks of the calls made once a token, packed as the C structs of
# the same name lie in memory (a ctypes.Structure takes 3 us to fill).
LINEAR_ARGS = struct.Struct("@3Q3QQQ2Q2Q6I")     # xksv_linear_args
KV_APPEND_ARGS = struct.Struct("@4Q8QQ4Q4Qf4I4x")  # xksv_kv_append_args
KV_ATTEND_ARGS = struct.Struct("@3Q4QQ3QQ2fQ2I")  # xksv_kv_attend_args


_SIGS = {
    "xksv_cuda_decode": ([ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t,
                          ctypes.c_void_p], ctypes.c_int),
    "xksv_cuda_gemv": ([ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t,
                        ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int),
    "xksv_cuda_gemm": ([ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t,
                        ctypes.c_size_t, ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int),
    "xksv_cuda_decode_parallel": ([ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "xksv_cuda_gemv_parallel": ([ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
                                 ctypes.c_void_p], ctypes.c_int),
    "xksv_plan_create": ([ctypes.POINTER(Slab), ctypes.c_size_t, ctypes.POINTER(ctypes.c_void_p)],
                         ctypes.c_int),
    "xksv_plan_destroy": ([ctypes.c_void_p], None),
    "xksv_plan_decode": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
                          ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "xksv_plan_decode_host": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
                               ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "xksv_plan_gemm": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
                        ctypes.c_size_t, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t,
                        ctypes.c_void_p], ctypes.c_int),
    "xksv_plan_status": ([ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int),
    "xksv_plan_scratch_bytes": ([ctypes.c_void_p], ctypes.c_size_t),
    "xksv_plan_set_scratch": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t], ctypes.c_int),
    "xksv_plan_launches": ([ctypes.c_void_p], ctypes.c_int),
    "xksv_plan_set_gemm_route": ([ctypes.c_void_p, ctypes.c_int], ctypes.c_int),
    "xksv_plan_fused_ready": ([ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int),
    "xksv_plan_set_parts": ([ctypes.c_void_p, ctypes.c_int], ctypes.c_int),
    "xksv_plan_index": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "xksv_cuda_sha256": ([ctypes.POINTER(ctypes.c_uint64), ctypes.c_size_t, ctypes.c_void_p,
                          ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int),
    "xksv_plan_sha256": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
                          ctypes.c_void_p], ctypes.c_int),
    "xksv_cuda_pack_tensor": ([ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int,
                               ctypes.c_uint64, ctypes.POINTER(ctypes.c_void_p),
                               ctypes.POINTER(ctypes.c_size_t), ctypes.POINTER(ctypes.c_void_p),
                               ctypes.POINTER(ctypes.c_size_t), ctypes.c_void_p], ctypes.c_int),
    "xksv_cuda_free": ([ctypes.c_void_p], None),
    "xksv_tp_fused_create": ([ctypes.c_int, ctypes.c_int, ctypes.c_size_t, ctypes.c_size_t,
                              ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p], ctypes.c_int),
    "xksv_tp_fused_open": ([ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int),
    "xksv_tp_fused_gemm": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t,
                            ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t,
                            ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p],
                           ctypes.c_int),
    "xksv_tp_fused_destroy": ([ctypes.c_void_p], None),
    "xksv_tp_unique_id": ([ctypes.c_void_p], ctypes.c_int),
    "xksv_tp_comm_create": ([ctypes.c_void_p, ctypes.c_int, ctypes.c_int,
                             ctypes.POINTER(ctypes.c_void_p)], ctypes.c_int),
    "xksv_tp_comm_destroy": ([ctypes.c_void_p], None),
    "xksv_tp_gemm": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
                      ctypes.c_size_t, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
                      ctypes.c_size_t, ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int),
    "xksv_host_pack": ([ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t,
                        ctypes.c_int, ctypes.POINTER(ctypes.c_void_p),
                        ctypes.POINTER(ctypes.c_size_t)], ctypes.c_int),
    "xksv_host_free": ([ctypes.c_void_p], None),
    "xksv_host_pack_tensor": ([ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t,
                               ctypes.c_int, ctypes.c_int, ctypes.c_uint64,
                               ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_size_t),
                               ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_size_t)],
                              ctypes.c_int),
    "xksv_cuda_decode_noalloc": ([ctypes.POINTER(Slab), ctypes.c_size_t, ctypes.c_void_p,
                                  ctypes.c_size_t, ctypes.c_void_p, ctypes.c_size_t,
                                  ctypes.c_void_p], ctypes.c_int),
    "xksv_plan_device": ([ctypes.c_void_p], ctypes.c_int),
    "xksv_plan_linear_workspace": ([ctypes.c_void_p, ctypes.c_size_t], ctypes.c_size_t),
    "xksv_plan_linear_workspace_for": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_uint32],
                                       ctypes.c_size_t),
    "xksv_plan_linear": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
                          ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "xksv_kv_create": ([ctypes.POINTER(KvDesc), ctypes.POINTER(ctypes.c_void_p)], ctypes.c_int),
    "xksv_kv_destroy": ([ctypes.c_void_p], None),
    "xksv_kv_status": ([ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int),
    "xksv_kv_append": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int),
    "xksv_kv_attend_workspace": ([ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t],
                                 ctypes.c_size_t),
    "xksv_kv_attend": ([ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t,
                        ctypes.c_void_p], ctypes.c_int),
}

# element types and activations of the linear layer and the key/value cache
BF16, FP16, FP32, E4M3 = 1, 2, 3, 4
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
KV_INTERLEAVED = 1

NOALLOC_MAX_SLABS = 4096
# xksv_plan_set_gemm_route
GEMM_AUTO, GEMM_SCRATCH, GEMM_FUSED = 0, 1, 2
# the fused decode -> tensor-core GEMM takes batches up to this size
FUSED_MAX_BATCH = 128
# xksv_plan_gemm: batches from this size run on the tensor cores (X rounded
# to BF16) when the plan has a tensor-core path (xksv_plan_scratch_bytes > 0)
TC_MIN_BATCH = 4

EXPORTS = tuple(_SIGS)
_lib = None


def library_path():
    return Path(os.environ.get("XKSV_CUDA_LIBRARY", DEFAULT_LIB))


def load(path=None):
    """Loads (once) and returns the CDLL with argtypes/restype set."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path else library_path()
    if not p.exists():
        raise FileNotFoundError(f"{p} is missing: build it with xks-vectorforge_b200/build.py")
    lib = ctypes.CDLL(str(p))
    for name, (args, res) in _SIGS.items():
        f = getattr(lib, name)
        f.argtypes = args
        f.restype = res
    if path is None:
        _lib = lib
    return lib


def slab_dtype():
    """numpy structured dtype with the memory layout of xksv_slab."""
    import numpy as np
    return np.dtype({"names": [f for f, _ in Slab._fields_],
                     "formats": ["<u8"] * 6 + ["<u4"] * 2,
                     "offsets": [getattr(Slab, f).offset for f, _ in Slab._fields_],
                     "itemsize": ctypes.sizeof(Slab)})


def slab_table(entries):
    """entries: iterable of dicts/tuples with the xksv_slab fields, or a
    numpy array of slab_dtype() (used in place, no per-row Python work)."""
    if hasattr(entries, "dtype") and entries.dtype == slab_dtype():
        import numpy as np
        arr = np.ascontiguousarray(entries)
        # the pointer keeps a reference to the array
        return arr.ctypes.data_as(ctypes.POINTER(Slab)), len(arr)
    entries = list(entries)
    arr = (Slab * max(1, len(entries)))()
    for i, e in enumerate(entries):
        if isinstance(e, dict):
            arr[i] = Slab(e["src_offset"], e["src_size"], e.get("rows", 0), e.get("cols", 0),
                          e.get("dst_offset", 0), e.get("x_offset", 0), e["codec"], 0)
        else:
            arr[i] = Slab(*e)
    return arr, len(entries)


def host_pack(raw, rows, cols, codec, lib=None):
    """Encodes one slab on the host (xksv_host_pack); returns bytes."""
    lib = lib or load()
    buf = ctypes.create_string_buffer(bytes(raw), max(1, len(raw)))
    out, size = ctypes.c_void_p(), ctypes.c_size_t()
    if lib.xksv_host_pack(buf, len(raw), rows, cols, codec, ctypes.byref(out), ctypes.byref(size)):
        raise ValueError("xksv_host_pack failed")
    try:
        return ctypes.string_at(out, size.value)
    finally:
        lib.xksv_host_free(out)


def host_pack_tensor(ptr, nbytes, rows, cols, codec, threads=0, dst_base=0, lib=None):
    """Encodes a row-major BF16 tensor at host address `ptr` into compiler
    slabs.  Returns (payload bytes as a numpy uint8 array, list of slab dicts)."""
    import numpy as np
    lib = lib or load()
    pay, psize = ctypes.c_void_p(), ctypes.c_size_t()
    tab, ns = ctypes.c_void_p(), ctypes.c_size_t()
    if lib.xksv_host_pack_tensor(ptr, nbytes, rows, cols, codec, threads, dst_base,
                                 ctypes.byref(pay), ctypes.byref(psize), ctypes.byref(tab),
                                 ctypes.byref(ns)):
        raise ValueError("xksv_host_pack_tensor failed")
    try:
        payload = np.ctypeslib.as_array((ctypes.c_uint8 * max(1, psize.value)).from_address(pay.value))[:psize.value].copy()
        arr = (Slab * max(1, ns.value)).from_address(tab.value)
        slabs = [dict(src_offset=s.src_offset, src_size=s.src_size, rows=s.rows, cols=s.cols,
                      dst_offset=s.dst_offset, x_offset=s.x_offset, codec=s.codec)
                 for s in arr[:ns.value]]
    finally:
        lib.xksv_host_free(pay)
        lib.xksv_host_free(tab)
    return payload, slabs


def cuda_pack_tensor(d_ptr, rows, cols, codec, dst_base=0, stream=0, lib=None):
    """GPU encoder (xksv_cuda_pack_tensor) of a row-major BF16 tensor at device
    address `d_ptr`.  Returns (device payload address, payload bytes, slab
    dicts); release the payload with free_device()."""
    lib = lib or load()
    pay, psize = ctypes.c_void_p(), ctypes.c_size_t()
    tab, ns = ctypes.c_void_p(), ctypes.c_size_t()
    if lib.xksv_cuda_pack_tensor(d_ptr, rows, cols, codec, dst_base, ctypes.byref(pay), ctypes.byref(psize),
                                 ctypes.byref(tab), ctypes.byref(ns), stream):
        raise ValueError("xksv_cuda_pack_tensor failed")
    try:
        arr = (Slab * max(1, ns.value)).from_address(tab.value)
        slabs = [dict(src_offset=s.src_offset, src_size=s.src_size, rows=s.rows, cols=s.cols,
                      dst_offset=s.dst_offset, x_offset=s.x_offset, codec=s.codec)
                 for s in arr[:ns.value]]
    finally:
        lib.xksv_host_free(tab)
    return pay.value, psize.value, slabs


def free_device(d_ptr, lib=None):
    (lib or load()).xksv_cuda_free(d_ptr)


def dev_buffer(buf, nbytes=None, what="buffer"):
    """(address, byte size) of a device buffer given to a plan call: a torch
    tensor (its own size, or `nbytes` when that is smaller) or an integer
    device address with its byte size.  The library refuses a call whose
    slabs fall outside the sizes it is given."""
    if hasattr(buf, "data_ptr"):
        n = buf.numel() * buf.element_size()
        return buf.data_ptr(), n if nbytes is None else min(int(nbytes), n)
    if nbytes is None:
        raise TypeError(f"{what}: an integer device address needs its byte size")
    return int(buf), int(nbytes)


def _rows(buf, nrows, batch, what):
    """(address, rows) of an FP32 [rows, batch] matrix (tensor or address)."""
    if hasattr(buf, "data_ptr"):
        n = buf.numel() * buf.element_size() // (4 * max(1, batch))
        return buf.data_ptr(), n if nrows is None else min(int(nrows), n)
    if nrows is None:
        raise TypeError(f"{what}: an integer device address needs its row count")
    return int(buf), int(nrows)


_types = {}
_i32 = None


def _type(t, allowed, what):
    """The element type code of tensor t, one of `allowed`."""
    if not _types:
        _torch_types()
    code = _types.get(t.dtype)
    if code not in allowed:
        raise ValueError(f"{what}: dtype {t.dtype} is not supported")
    return code


def _torch_types():
    global _i32
    import torch
    _i32 = torch.int32
    _types.update({torch.bfloat16: BF16, torch.float16: FP16, torch.float32: FP32, torch.float8_e4m3fn: E4M3})


def _matrix(t, rows, cols, what, device):
    """(address, row stride) of a [rows, cols] tensor whose rows are contiguous."""
    if t.shape != (rows, cols):
        raise ValueError(f"{what}: shape {tuple(t.shape)} is not [{rows}, {cols}]")
    row, one = t.stride()
    if one != 1 and cols > 1:
        raise ValueError(f"{what}: rows must be contiguous")
    if t.get_device() != device:
        raise ValueError(f"{what}: on {t.device}, expected CUDA device {device}")
    return t.data_ptr(), row


def _heads(t, rows, heads, dim, what, device):
    """(address, row stride, head stride) of a [rows, heads, dim] tensor whose
    last dimension is contiguous."""
    if t.shape != (rows, heads, dim):
        raise ValueError(f"{what}: shape {tuple(t.shape)} is not [{rows}, {heads}, {dim}]")
    row, head, one = t.stride()
    if one != 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")
    if t.get_device() != device:
        raise ValueError(f"{what}: on {t.device}, expected CUDA device {device}")
    return t.data_ptr(), row, head


def _ints(t, n, what, device):
    """Address of a contiguous int32 [n] tensor."""
    if t.dtype != _i32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous int32 [{n}] tensor is needed")
    if t.get_device() != device:
        raise ValueError(f"{what}: on {t.device}, expected CUDA device {device}")
    return t.data_ptr()


def _table(t, device):
    """(address, rows, columns, row stride) of an int32 page table."""
    if t.dtype != _i32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError("table: an int32 [sequences, pages] tensor with contiguous rows is needed")
    if t.get_device() != device:
        raise ValueError(f"table: on {t.device}, expected CUDA device {device}")
    rows, cols = t.shape
    return t.data_ptr(), rows, cols, t.stride(0)


def _workspace(given, nbytes, device, stream):
    """(tensor, address, bytes) of a call's workspace: the caller's uint8 tensor, or a
    new one from torch's allocator of the call's stream, so that neither two
    calls nor two captured graphs share one."""
    import torch
    if given is not None:
        if given.device != device or not given.is_contiguous():
            raise ValueError("workspace: a contiguous tensor on the call's device is needed")
        return given, given.data_ptr(), given.numel() * given.element_size()
    if not nbytes:
        return None, None, 0
    # (the raw handle: building a torch Stream object takes 3.5 us of a 20 us call)
    if stream == torch._C._cuda_getCurrentRawStream(device.index):
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
    else:
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device)):
            buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return buf, buf.data_ptr(), nbytes


class Plan:
    """A device-resident plan over one payload buffer (see include/xksv_cuda.h).
    Device buffers are torch tensors (their sizes bound the call) or integer
    addresses with explicit sizes (payload_bytes, out_bytes, x_rows, y_rows)."""

    def __init__(self, entries, lib=None):
        self.lib = lib or load()
        arr, n = slab_table(entries)
        h = ctypes.c_void_p()
        if self.lib.xksv_plan_create(arr, n, ctypes.byref(h)):
            raise ValueError("xksv_plan_create rejected the slab table")
        self.handle = h
        self.n = n
        self.device = self.lib.xksv_plan_device(h)  # its calls' tensors live there

    def decode(self, d_payload, d_out, stream=0, payload_bytes=None, out_bytes=None):
        pay, npay = dev_buffer(d_payload, payload_bytes, "payload")
        out, nout = dev_buffer(d_out, out_bytes, "output")
        if self.lib.xksv_plan_decode(self.handle, pay, npay, out, nout, stream):
            raise RuntimeError("xksv_plan_decode refused the call or failed to launch")

    def decode_host(self, h_payload, size, d_payload, d_out, stream=0, out_bytes=None):
        """Host payload (`size` bytes at host address h_payload) -> d_payload
        -> decode, copy and decode overlapped (xksv_plan_decode_host)."""
        pay, npay = dev_buffer(d_payload, None if hasattr(d_payload, "data_ptr") else size, "payload")
        out, nout = dev_buffer(d_out, out_bytes, "output")
        if npay < size:
            raise ValueError("device payload buffer smaller than the host payload")
        if self.lib.xksv_plan_decode_host(self.handle, h_payload, size, pay, out, nout, stream):
            raise RuntimeError("xksv_plan_decode_host refused the call or failed")

    def gemm(self, d_payload, d_x, d_y, batch, stream=0, payload_bytes=None, x_rows=None, y_rows=None):
        pay, npay = dev_buffer(d_payload, payload_bytes, "payload")
        x, nx = _rows(d_x, x_rows, batch, "x")
        y, ny = _rows(d_y, y_rows, batch, "y")
        if self.lib.xksv_plan_gemm(self.handle, pay, npay, x, nx, y, ny, batch, stream):
            raise RuntimeError("xksv_plan_gemm refused the call or failed to launch")

    def linear(self, d_payload, x, y, bias=None, act="none", mul=None, residual=None, stream=0, payload_bytes=None,
               workspace=None):
        """y = act(x W^T + bias) * mul + residual (xksv_plan_linear): x BF16
        [batch, x columns], y BF16 or FP32 [batch, Y rows]; bias [Y rows], mul and
        residual [batch, Y rows] are BF16 or FP32; act is a key of ACTS.  Rows may
        be strided; residual or mul may be y.  `workspace` (uint8, at least
        linear_workspace(batch) bytes) defaults to a new buffer per call, of
        the bytes this call takes."""
        if act not in ACTS:
            raise ValueError(f"unknown activation {act}")
        device = self.device
        pay, npay = dev_buffer(d_payload, payload_bytes, "payload")
        if x.dim() != 2 or y.dim() != 2:
            raise ValueError("x and y are [batch, columns]")
        (batch, cols), rows = x.shape, y.shape[1]
        _type(x, (BF16,), "x")
        xp, xs = _matrix(x, batch, cols, "x", device)
        yp, ys = _matrix(y, batch, rows, "y", device)
        y_type = _type(y, (BF16, FP32), "y")
        bp = mp = ms = rp = rs = b_type = m_type = r_type = 0
        if bias is not None:
            b_type = _type(bias, (BF16, FP32), "bias")
            if bias.shape != (rows,) or not bias.is_contiguous() or bias.get_device() != device:
                raise ValueError(f"bias: a contiguous [{rows}] tensor on CUDA device {device} is needed")
            bp = bias.data_ptr()
        if mul is not None:
            m_type = _type(mul, (BF16, FP32), "mul")
            mp, ms = _matrix(mul, batch, rows, "mul", device)
        if residual is not None:
            r_type = _type(residual, (BF16, FP32), "residual")
            rp, rs = _matrix(residual, batch, rows, "residual", device)
        a = LINEAR_ARGS.pack(xp, cols, xs, yp, rows, ys, batch, bp, mp, ms, rp, rs, y_type, b_type, m_type, r_type,
                             ACTS[act], 0)
        need = self.lib.xksv_plan_linear_workspace_for(self.handle, pay, batch, y_type)
        ws, wp, wn = _workspace(workspace, need, x.device, stream)
        if self.lib.xksv_plan_linear(self.handle, pay, npay, a, wp, wn, stream):
            raise RuntimeError("xksv_plan_linear refused the call or failed to launch")

    def linear_workspace(self, batch):
        """Bytes of workspace that serve any linear call of `batch` tokens, before
        and after an index or another route."""
        return self.lib.xksv_plan_linear_workspace(self.handle, batch)

    def index(self, d_payload, stream=0, payload_bytes=None, parts=True):
        """Builds the tile index (xksv_plan_index); returns 0, or 1 on a bad slab.
        `parts` False leaves the parts of parallel-codec slabs off, which take
        10 KB a slab (29 % of a compressed 2048 x 2048 weight, 4 % of a 4096 x
        14336 one) and make decodes of few slabs faster."""
        self.lib.xksv_plan_set_parts(self.handle, int(parts))
        pay, npay = dev_buffer(d_payload, payload_bytes, "payload")
        return self.lib.xksv_plan_index(self.handle, pay, npay, stream)

    def sha256(self, d_out, d_digests, stream=0, out_bytes=None):
        """Enqueues the SHA-256 of every slab's decoded bytes (xksv_plan_sha256)."""
        out, nout = dev_buffer(d_out, out_bytes, "output")
        dig = d_digests.data_ptr() if hasattr(d_digests, "data_ptr") else d_digests
        if self.lib.xksv_plan_sha256(self.handle, out, nout, dig, stream):
            raise RuntimeError("xksv_plan_sha256 failed")

    def scratch_bytes(self):
        """Bytes of BF16 scratch the tensor-core path needs (0: none)."""
        return self.lib.xksv_plan_scratch_bytes(self.handle)

    def set_scratch(self, d_scratch, nbytes):
        """Lends the plan a caller-owned scratch (xksv_plan_set_scratch)."""
        if self.lib.xksv_plan_set_scratch(self.handle, d_scratch, nbytes):
            raise ValueError("scratch too small or misaligned")

    def set_gemm_route(self, route):
        """GEMM_AUTO, GEMM_SCRATCH or GEMM_FUSED (xksv_plan_set_gemm_route)."""
        if self.lib.xksv_plan_set_gemm_route(self.handle, int(route)):
            raise ValueError(f"unknown GEMM route {route}")

    def fused_ready(self, d_payload):
        """True when the fused decode -> tensor-core GEMM applies to this
        plan on d_payload (indexed, all 16-row serial slabs)."""
        pay = d_payload.data_ptr() if hasattr(d_payload, "data_ptr") else d_payload
        return bool(self.lib.xksv_plan_fused_ready(self.handle, pay))

    def status(self, stream=0):
        """0 when no slab reported an error since the last call, else 1."""
        return self.lib.xksv_plan_status(self.handle, stream)

    def launches(self):
        return self.lib.xksv_plan_launches(self.handle)

    def close(self):
        if self.handle:
            self.lib.xksv_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KVCache:
    """A paged key/value cache over two torch tensors (xksv_kv_*): k and v are
    [pages, page_size, heads, dim] (layout "nhd") or [pages, heads, page_size,
    dim] ("hnd") of BF16, FP16 or float8_e4m3fn, any strides that are
    multiples of 16 bytes; k_scale and v_scale are FP32 [heads] for float8.
    A page table is an int32 [sequences, pages] tensor of page numbers."""

    def __init__(self, k, v, k_scale=None, v_scale=None, layout="nhd", lib=None):
        import torch
        if layout not in ("nhd", "hnd"):
            raise ValueError(f"unknown layout {layout}")
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.device.type != "cuda":
            raise ValueError("k and v are CUDA tensors of one shape [pages, page_size, heads, dim] and dtype")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("the last dimension of k and v must be contiguous")
        self.lib = lib or load()
        self.handle = None
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.index, self.type = k.device, k.get_device(), _type(k, (BF16, FP16, E4M3), "k")
        order = (0, 1, 2) if layout == "nhd" else (0, 2, 1)  # page, token, head
        self.pages, self.page_size, self.kv_heads = (k.shape[i] for i in order)
        self.head_dim = k.shape[3]
        for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
            if s is not None and (s.dtype != torch.float32 or tuple(s.shape) != (self.kv_heads,)
                                  or not s.is_contiguous() or s.device != self.device):
                raise ValueError(f"{name}: a contiguous FP32 [{self.kv_heads}] tensor on {self.device} is needed")
        nbytes = [(t.untyped_storage().nbytes() - t.storage_offset() * t.element_size()) for t in (k, v)]
        d = KvDesc(k.data_ptr(), v.data_ptr(), nbytes[0], nbytes[1], self.pages, self.page_size)
        d.k_stride[:] = [k.stride(i) for i in order]
        d.v_stride[:] = [v.stride(i) for i in order]
        d.k_scale = k_scale.data_ptr() if k_scale is not None else None
        d.v_scale = v_scale.data_ptr() if v_scale is not None else None
        d.kv_heads, d.head_dim, d.type = self.kv_heads, self.head_dim, self.type
        h = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            if self.lib.xksv_kv_create(ctypes.byref(d), ctypes.byref(h)):
                raise ValueError("xksv_kv_create rejected the cache")
        self.handle = h

    def append(self, k, v, table, index, seq=None, positions=None, inv_freq=None, rot_scale=1.0, interleaved=False,
               q=None, q_out=None, stream=0):
        """Rotates new keys (and queries) and writes keys and values to their
        places (xksv_kv_append): k, v [tokens, heads, dim] and q, q_out [tokens,
        query heads, dim] of one dtype; token t is token index[t] of sequence
        seq[t] (default t; negative: padding, skipped), rotated by positions[t]
        (default index[t]) and inv_freq FP32 [rotated dims / 2] (None: no
        rotation).  q_out defaults to q, in place."""
        n, dev, dim = k.shape[0], self.index, self.head_dim
        code = _type(k, (BF16, FP16, FP32), "k")
        kp, k0, k1 = _heads(k, n, self.kv_heads, dim, "k", dev)
        vp, v0, v1 = _heads(v, n, self.kv_heads, dim, "v", dev)
        if v.dtype != k.dtype:
            raise ValueError("k and v are of one dtype")
        qp = q0 = q1 = op = o0 = o1 = heads = 0
        if q is not None:
            q_out = q if q_out is None else q_out
            if q.dtype != k.dtype or q_out.dtype != k.dtype or q.dim() != 3:
                raise ValueError("q and q_out are [tokens, heads, dim] of k's dtype")
            heads = q.shape[1]
            qp, q0, q1 = _heads(q, n, heads, dim, "q", dev)
            op, o0, o1 = _heads(q_out, n, heads, dim, "q_out", dev)
        elif q_out is not None:
            raise ValueError("q_out without q")
        tp, rows, cols, stride = _table(table, dev)
        ip = _ints(index, n, "index", dev)
        sp = 0 if seq is None else _ints(seq, n, "seq", dev)
        pp = 0 if positions is None else _ints(positions, n, "positions", dev)
        fp = rot = 0
        if inv_freq is not None:
            _type(inv_freq, (FP32,), "inv_freq")
            if inv_freq.dim() != 1 or not inv_freq.is_contiguous() or inv_freq.get_device() != dev:
                raise ValueError(f"inv_freq: a contiguous FP32 vector on CUDA device {dev} is needed")
            fp, rot = inv_freq.data_ptr(), 2 * inv_freq.shape[0]
        a = KV_APPEND_ARGS.pack(qp, kp, vp, op, q0, q1, k0, k1, v0, v1, o0, o1, n, tp, rows, cols, stride, sp, ip, pp, fp,
                                rot_scale, rot, heads, code, KV_INTERLEAVED if interleaved else 0)
        if self.lib.xksv_kv_append(self.handle, a, stream):
            raise RuntimeError("xksv_kv_append refused the call or failed to launch")

    def attend(self, q, table, lens, out, lse=None, scale=None, window=0, softcap=0.0, stream=0, workspace=None):
        """Attention of one new token per sequence over its lens[s] cached
        tokens (xksv_kv_attend): q and out [sequences, query heads, dim] of the
        cache's dtype (BF16 or FP16 over float8), lse FP32 [sequences, query
        heads] or None; scale defaults to dim ** -0.5; window 0 sees the whole
        sequence; softcap 0 is off.  `workspace` (uint8, at least
        attend_workspace(...) bytes) defaults to a new buffer per call."""
        dev, n, dim = self.index, lens.shape[0], self.head_dim
        if q.dim() != 3 or out.dtype != q.dtype:
            raise ValueError("q and out are [sequences, heads, dim] of one dtype")
        heads = q.shape[1]
        code = _type(q, (BF16, FP16), "q")
        qp, q0, q1 = _heads(q, n, heads, dim, "q", dev)
        op, o0, o1 = _heads(out, n, heads, dim, "out", dev)
        lp = 0
        if lse is not None:
            _type(lse, (FP32,), "lse")
            if lse.shape != (n, heads) or not lse.is_contiguous() or lse.get_device() != dev:
                raise ValueError(f"lse: a contiguous FP32 [{n}, {heads}] tensor on CUDA device {dev} is needed")
            lp = lse.data_ptr()
        tp, rows, cols, stride = _table(table, dev)
        if rows < n:
            raise ValueError(f"table: {rows} rows for {n} sequences")
        if window < 0:
            raise ValueError("window is not negative")
        a = KV_ATTEND_ARGS.pack(qp, op, lp, q0, q1, o0, o1, n, tp, cols, stride, _ints(lens, n, "lens", dev),
                                dim ** -0.5 if scale is None else scale, softcap, window, heads, code)
        ws, wp, wn = workspace, None, 0
        if n:
            need = self.lib.xksv_kv_attend_workspace(self.handle, n, heads, cols)
            ws, wp, wn = _workspace(workspace, need, self.device, stream)
        if self.lib.xksv_kv_attend(self.handle, a, wp, wn, stream):
            raise RuntimeError("xksv_kv_attend refused the call or failed to launch")

    def attend_workspace(self, seqs, q_heads, table_cols):
        """Bytes of workspace an attend call needs."""
        return self.lib.xksv_kv_attend_workspace(self.handle, seqs, q_heads, table_cols)

    def status(self, stream=0):
        """0 when no call met a page, place or length outside the cache since
        the last call, else 1."""
        return self.lib.xksv_kv_status(self.handle, stream)

    def close(self):
        if self.handle:
            self.lib.xksv_kv_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---------------------------------------------------------- tensor parallel
TP_ID_BYTES = 128


def shard_rows(rows, world, rank, align=16):
    """Row range [r0, r1) of `rank` when `rows` rows are split over `world`
    ranks in whole 16-row slabs (the first ranks take one slab more when the
    slab count does not divide)."""
    nslab = (rows + align - 1) // align
    base, extra = divmod(nslab, world)
    s0 = rank * base + min(rank, extra)
    s1 = s0 + base + (1 if rank < extra else 0)
    return min(rows, s0 * align), min(rows, s1 * align)


def shard_entries(entries, world, rank, rows_of):
    """The slab entries of this rank's rows, for TP GEMV/GEMM.

    `entries` are GEMV slab entries whose dst_offset is the slab's first row
    in the full Y (a plan may cover several tensors); `rows_of(e)` gives the
    (first row, row count) of the tensor the slab belongs to.  Each tensor is
    split separately with shard_rows; returns (local entries with dst_offset
    rebased to the rank's shard of Y, rows in the shard, and the list of
    (full_row0, local_row0, nrows) runs that map the shard back)."""
    out, runs, local = [], [], 0
    seen = {}
    for e in entries:
        t0, trows = rows_of(e)
        if t0 not in seen:
            r0, r1 = shard_rows(trows, world, rank)
            seen[t0] = (r0, r1, local)
            runs.append((t0 + r0, local, r1 - r0))
            local += r1 - r0
        r0, r1, l0 = seen[t0]
        row = e["dst_offset"] - t0
        if r0 <= row < r1:
            d = dict(e)
            d["dst_offset"] = l0 + row - r0
            out.append(d)
    return out, local, runs


def gathered_to_full(gathered, world, runs_per_rank, rows_shard):
    """Row indices: full_row -> row of the all-gathered buffer
    ([world * rows_shard] rows in rank order), from each rank's runs."""
    import numpy as np
    total = sum(n for runs in runs_per_rank for _, _, n in runs)
    idx = np.empty(total, dtype=np.int64)
    for g, runs in enumerate(runs_per_rank):
        for full0, local0, n in runs:
            idx[full0:full0 + n] = g * rows_shard + local0 + np.arange(n)
    return idx


class TPComm:
    """NCCL communicator for xksv_tp_gemm over the ranks of a torch.distributed
    group (which only carries the unique id)."""

    def __init__(self, rank, world, lib=None):
        import torch.distributed as dist
        self.lib = lib or load()
        uid = ctypes.create_string_buffer(TP_ID_BYTES)
        if rank == 0 and self.lib.xksv_tp_unique_id(uid):
            raise RuntimeError("xksv_tp_unique_id failed (NCCL not available?)")
        obj = [bytes(uid.raw) if rank == 0 else None]
        dist.broadcast_object_list(obj, src=0)
        uid = ctypes.create_string_buffer(obj[0], TP_ID_BYTES)
        h = ctypes.c_void_p()
        if self.lib.xksv_tp_comm_create(uid, world, rank, ctypes.byref(h)):
            raise RuntimeError("xksv_tp_comm_create failed")
        self.handle = h
        self.rank, self.world = rank, world

    def gemm(self, plan, d_payload, d_x, d_y_shard, rows_shard, d_y_full, batch, stream=0,
             payload_bytes=None, x_rows=None):
        pay, npay = dev_buffer(d_payload, payload_bytes, "payload")
        x, nx = _rows(d_x, x_rows, batch, "x")
        ys = d_y_shard.data_ptr() if hasattr(d_y_shard, "data_ptr") else d_y_shard
        yf = d_y_full.data_ptr() if hasattr(d_y_full, "data_ptr") else d_y_full
        if self.lib.xksv_tp_gemm(plan.handle, pay, npay, x, nx, ys, rows_shard, yf, batch, self.handle, stream):
            raise RuntimeError("xksv_tp_gemm failed")

    def close(self):
        if self.handle:
            self.lib.xksv_tp_comm_destroy(self.handle)
            self.handle = None


def sha256_ranges(ranges, d_base, d_digests, stream=0, lib=None):
    """SHA-256 of device byte ranges [(offset, length), ...] (or an n x 2
    integer array) at d_base into d_digests (n * 32 bytes, device);
    xksv_cuda_sha256."""
    import numpy as np
    lib = lib or load()
    flat = np.ascontiguousarray(np.asarray(ranges, dtype=np.uint64).reshape(-1))
    n = flat.size // 2
    ptr = flat.ctypes.data_as(ctypes.POINTER(ctypes.c_uint64))
    if lib.xksv_cuda_sha256(ptr, n, d_base, d_digests, stream):
        raise RuntimeError("xksv_cuda_sha256 failed")


class TPFused:
    """Fused tensor-parallel GEMV/GEMM (xksv_tp_fused_*): the GEMV epilogue
    stores each output row into every rank's gathered buffer over NVLink; the
    IPC handles travel over a torch.distributed group."""

    IPC_BYTES = 64

    def __init__(self, rank, world, max_rows_shard, max_batch=1, lib=None):
        import torch.distributed as dist
        self.lib = lib or load()
        h = ctypes.create_string_buffer(self.IPC_BYTES)
        ctx = ctypes.c_void_p()
        if self.lib.xksv_tp_fused_create(world, rank, max_rows_shard, max_batch, ctypes.byref(ctx), h):
            raise RuntimeError("xksv_tp_fused_create failed")
        self.handle = ctx
        handles = [None] * world
        dist.all_gather_object(handles, bytes(h.raw))
        joined = ctypes.create_string_buffer(b"".join(handles), self.IPC_BYTES * world)
        if self.lib.xksv_tp_fused_open(ctx, joined):
            self.close()
            raise RuntimeError("xksv_tp_fused_open failed")
        dist.barrier()

    def gemm(self, plan, d_payload, d_x, rows_shard, batch, stream=0, d_y_full=None, payload_bytes=None,
             x_rows=None):
        """Enqueues the fused call (and a copy of the gathered Y to d_y_full
        when given); returns the device address of the gathered Y."""
        pay, npay = dev_buffer(d_payload, payload_bytes, "payload")
        x, nx = _rows(d_x, x_rows, batch, "x")
        yf = d_y_full.data_ptr() if hasattr(d_y_full, "data_ptr") else d_y_full
        y = ctypes.c_void_p()
        if self.lib.xksv_tp_fused_gemm(self.handle, plan.handle, pay, npay, x, nx, rows_shard, batch,
                                       yf, ctypes.byref(y), stream):
            raise RuntimeError("xksv_tp_fused_gemm failed")
        return y.value

    def close(self):
        if self.handle:
            self.lib.xksv_tp_fused_destroy(self.handle)
            self.handle = None
