"""ctypes binding of libkernelsmith (B200).

The product is the C library (ulir-kernels_b200/lib/libkernelsmith.so) and
its headers (include/kernelsmith/*.h, include/ks_b200.h).  This module binds
every exported symbol with its C signature so Python callers -- the tests,
bench.py and the multi-GPU host logic -- go through exactly the entry points
a C caller of the reference libkernelsmith would use.

Buffers are passed as raw addresses: `addr(t)` accepts a torch tensor (device
or host), a numpy array, an int or None.

There is no Python or CPU implementation of any kernel here; if the library
is missing, `lib()` raises.
"""

from __future__ import annotations

import ctypes
import os
from ctypes import POINTER, c_char_p, c_float, c_int, c_int32, c_size_t, c_uint16, c_uint32, c_void_p
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent.parent
# the in-tree build; KS_B200_LIBRARY names another build of the same library
LIB_PATH = Path(os.environ.get("KS_B200_LIBRARY") or (PKG_DIR / "lib" / "libkernelsmith.so"))

KS_OK = 0
KS_ERR_INVALID_ARG = -1
KS_ERR_WORKSPACE = -2
KS_ERR_UNSUPPORTED = -3
KS_ERR_DEVICE = -4

SCALE_F32 = 0
SCALE_F16 = 1
STATUS_WORDS = 2
STATUS_BAD_SCALE = 0
STATUS_TIMEOUT = 1
IPC_HANDLE_BYTES = 64
DTYPE_F32 = 0
DTYPE_F16 = 1
DTYPE_BF16 = 2
KS_QUANT_LAYOUT_VERSION = 1  # include/ks_b200.h; lib().ks_b200_quant_layout_version() returns the built value

_vp = c_void_p
_sz = c_size_t
_i32 = c_int32
_f = c_float

# name -> (restype, argtypes); the C declarations are in include/.
SIGNATURES: dict[str, tuple[object, list[object]]] = {
    # ks_common.h
    "ks_target_name": (c_char_p, []),
    "ks_simd_width_f32": (_sz, []),
    # ks_quantized.h
    "ks_dot_i8": (c_int, [_vp, _vp, _sz, _i32, _i32, _vp, _vp, _sz]),
    "ks_matvec_i8": (c_int, [_vp, _vp, _sz, _vp, _sz, _sz, _i32, _i32, _vp, _sz]),
    "ks_dot_w4a8": (c_int, [_vp, _vp, _vp, _sz, _sz, _f, _i32, _i32, _vp, _vp, _sz]),
    "ks_matvec_w4a8": (
        c_int,
        [_vp, _vp, _sz, _vp, _sz, _vp, _sz, _sz, _sz, _f, _i32, _i32, _vp, _sz],
    ),
    "ks_dot_i8_workspace": (_sz, [_sz]),
    "ks_matvec_i8_workspace": (_sz, [_sz, _sz]),
    "ks_dot_w4a8_workspace": (_sz, [_sz, _sz]),
    "ks_matvec_w4a8_workspace": (_sz, [_sz, _sz, _sz]),
    "ks_quantized_alignment": (_sz, []),
    "ks_w4a8_packed_row_bytes": (_sz, [_sz]),
    "ks_w4a8_scale_groups": (_sz, [_sz, _sz]),
    # ks_b200.h
    "ks_b200_version": (c_char_p, []),
    "ks_b200_last_error": (c_char_p, []),
    "ks_b200_device_count": (c_int, []),
    "ks_b200_matvec_w4a8_f16": (
        c_int,
        [_vp, _vp, _sz, _vp, _sz, _vp, _sz, _sz, _sz, _f, _i32, _i32],
    ),
    "ks_b200_matvec_w4a8_f16_noalloc": (
        c_int,
        [_vp, _vp, _sz, _vp, _sz, _vp, _sz, _sz, _sz, _f, _i32, _i32],
    ),
    "ks_b200_matvec_i8_dequant": (c_int, [_vp, _vp, _sz, _vp, _f, _vp, _sz, _sz, _i32, _i32]),
    "ks_b200_matvec_w4a8_async": (
        c_int,
        [_vp, _vp, _sz, _vp, c_int, _sz, _vp, _sz, _sz, _sz, _f, _i32, _i32, _vp, _vp],
    ),
    "ks_b200_matvec_i8_async": (c_int, [_vp, _vp, _sz, _vp, _sz, _sz, _i32, _i32, _vp]),
    "ks_b200_matvec_i8_dequant_async": (
        c_int,
        [_vp, _vp, _sz, _vp, _f, _vp, _sz, _sz, _i32, _i32, _vp],
    ),
    "ks_b200_matvec_w4a8_batch_async": (
        c_int,
        [c_int, _vp, _vp, _vp, _vp, _sz, c_int, _sz, _sz, _sz, _sz, _f, _i32, _i32, _vp, _vp],
    ),
    "ks_b200_matvec_i8_batch_async": (c_int, [c_int, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _i32, _i32, _f, _vp]),
    "ks_b200_ipc_get_handle": (c_int, [_vp, _vp, _vp]),
    "ks_b200_ipc_open_handle": (c_int, [_vp, _sz, _vp]),
    "ks_b200_ipc_close_handle": (c_int, [_vp, _sz]),
    "ks_b200_matvec_w4a8_batch_gather_async": (
        c_int,
        [c_int, _vp, _vp, _vp, c_int, _vp, _vp, _sz, _sz, _sz, c_int, _sz, _sz, _sz, _sz, _f, _i32, _i32, _vp,
         _vp, _vp],
    ),
    "ks_b200_peer_arrival_wait_async": (c_int, [_vp, _vp, c_uint32, _vp, _vp]),
    "ks_b200_peer_arrival_wait_ranks_async": (c_int, [_vp, c_int, _vp, c_uint32, ctypes.c_uint64, _vp, _vp]),
    "ks_b200_status_check": (c_int, [_vp, _vp]),
    "ks_b200_decode_layer_workspace": (_sz, [_sz, _sz]),
    "ks_b200_decode_layers_workspace": (_sz, [_sz, _sz]),
    "ks_b200_decode_layers_w4a8_async": (
        c_int,
        [_sz, _vp, _vp, _vp, _vp, _f, _vp, _vp, _sz, _sz, _sz, _vp, _sz, _vp, _vp],
    ),
    "ks_b200_decode_layer_offsets": (c_int, [_sz, _sz, _vp]),
    "ks_b200_decode_layer_w4a8_async": (
        c_int,
        [_vp, _vp, _vp, _vp, _f, _vp, _vp, _sz, _sz, _sz, _vp, _sz, _vp, _vp],
    ),
    "ks_b200_gemm_i8_requant": (c_int, [_vp, _sz, _vp, _vp, _sz, _vp, _f, _vp, _sz, _sz, _sz, _sz]),
    "ks_b200_gemm_i8_requant_async": (
        c_int,
        [_vp, _sz, _vp, _vp, _sz, _vp, _f, _vp, _sz, _sz, _sz, _sz, _vp, _vp, _vp],
    ),
    "ks_b200_gemm_i8_kernel_path": (c_int, [_vp, _sz, _vp, _sz, _sz, _sz, _sz]),
    "ks_b200_gemm_i8_requant_batch_async": (
        c_int,
        [c_int, _vp, _sz, _vp, _vp, _sz, _vp, _f, _vp, _sz, _sz, _sz, _sz, _vp, _vp],
    ),
    "ks_b200_quant_layout_version": (c_int, []),
    "ks_b200_w4a8_register": (c_int, [_vp, _sz, _vp, c_int, _sz, _sz, _sz, _sz, _sz, _sz, c_int, _vp]),
    "ks_b200_w4a8_weights_info": (c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "ks_b200_w4a8_matvec_registered_async": (c_int, [_vp, _vp, _f, _i32, _i32, _vp, _vp, _vp]),
    "ks_b200_w4a8_release": (c_int, [_vp]),
    "ks_b200_gemm_w4a8_async": (
        c_int,
        [_vp, _sz, _vp, _vp, _sz, _vp, c_int, _sz, _vp, _sz, _sz, _sz, _sz, _sz, _vp, _vp],
    ),
    "ks_b200_import_ggml_q4_0_async": (c_int, [_vp, _sz, _sz, _sz, _sz, _vp, _sz, _vp, c_int, _sz, _vp]),
    "ks_b200_w4a8_kernel_path": (c_int, [_vp, _vp, _sz, _vp, c_int, _sz, _sz, _sz, _sz]),
    "ks_b200_i8_kernel_path": (c_int, [_vp, _vp, _sz, _sz, _sz]),
    "ks_b200_matvec_w4a8_f32in_async": (
        c_int,
        [_vp, _vp, _sz, _vp, c_int, _sz, _vp, _sz, _sz, _sz, _vp, _vp, _vp, _vp],
    ),
    "ks_b200_quantize_per_token_async": (c_int, [_vp, _sz, _sz, _sz, _vp, _sz, _vp, _vp]),
    "ks_b200_decode_layer_launches": (c_int, [_sz, _sz, _sz]),
    "ks_b200_kv4_page_bytes": (_sz, [_sz, _sz, _sz, _sz]),
    "ks_b200_kv4_append_async": (
        c_int,
        [_vp, _vp, _sz, _vp, _vp, _sz, _sz, _vp, _sz, _sz, _vp, _sz, _sz, c_int, _vp, _vp],
    ),
    "ks_b200_kv4_read_async": (
        c_int,
        [_vp, _vp, _sz, _vp, _vp, _sz, _sz, _vp, _sz, _sz, _vp, _sz, _sz, c_int, _vp, _vp],
    ),
    "ks_b200_kv4_append_bounded_async": (
        c_int,
        [_vp, _vp, _sz, _vp, _vp, _sz, _sz, _sz, _vp, _sz, _sz, _vp, _sz, _sz, c_int, _vp, _vp],
    ),
    "ks_b200_kv4_read_bounded_async": (
        c_int,
        [_vp, _vp, _sz, _vp, _vp, _sz, _sz, _sz, _vp, _sz, _sz, _vp, _sz, _sz, c_int, _vp, _vp],
    ),
    "ks_b200_kv4_attention_workspace": (_sz, [_vp, _sz, _sz, _sz, _sz, _sz]),
    "ks_b200_kv4_attention_async": (
        c_int,
        [_vp, _vp, _sz, _vp, _vp, _sz, _sz, _sz, _sz, _vp, _sz, _sz, _sz, _f, _vp, _sz, _sz, c_int, _vp, c_int,
         _vp, _sz, _vp, _vp],
    ),
    "ks_b200_kv4_evict_workspace": (_sz, [_vp, _sz, _sz, _sz]),
    "ks_b200_kv4_evict_async": (
        c_int,
        [_vp, _vp, _sz, _vp, _sz, _sz, _vp, _sz, _vp, _sz, _sz, _vp, _vp, _sz, _vp, _vp],
    ),
    # include/ks_b200_ggml.h: the GGML MUL_MAT(Q4_0, f32) adapter
    "ks_b200_ggml_q4_0_create": (c_int, [_vp, _sz, _sz, _sz, _vp, _vp]),
    "ks_b200_ggml_q4_0_destroy": (c_int, [_vp]),
    "ks_b200_ggml_q4_0_native": (c_int, [_vp, _vp, _vp, _vp, _vp]),
    "ks_b200_ggml_mul_mat_q4_0_async": (c_int, [_vp, _vp, _sz, _vp, _sz, _sz, _vp, _vp]),
    "ks_b200_ggml_report_get": (None, [_vp]),
    "ks_b200_ggml_report_reset": (None, []),
}

_lib: ctypes.CDLL | None = None


class KernelSmithError(RuntimeError):
    def __init__(self, rc: int, msg: str):
        super().__init__(f"libkernelsmith returned {rc}: {msg}")
        self.rc = rc


def lib() -> ctypes.CDLL:
    """Load libkernelsmith (B200) once and bind every signature."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise ImportError(
                f"libkernelsmith (B200) is not built at {LIB_PATH}; run "
                "`python ulir-kernels_b200/build.py` (or __graft_entry__.build())"
            )
        handle = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def addr(obj) -> int | None:
    """Raw address of a torch tensor, numpy array, int or None."""
    if obj is None:
        return None
    if isinstance(obj, int):
        return obj
    if hasattr(obj, "data_ptr"):
        return obj.data_ptr()
    if hasattr(obj, "ctypes"):
        return obj.ctypes.data
    raise TypeError(f"cannot take the address of {type(obj)!r}")


def last_error() -> str:
    return lib().ks_b200_last_error().decode()


def check(rc: int) -> None:
    if rc != KS_OK:
        raise KernelSmithError(rc, last_error())


def stream_handle(stream) -> int | None:
    """cudaStream_t of a torch.cuda.Stream (None -> legacy default stream)."""
    if stream is None:
        return None
    return int(stream.cuda_stream)


def matvec_w4a8_async(x, w, w_stride, s, s_stride, y, rows, cols, group, sx, zx=0, zw=0,
                      scale_type=SCALE_F16, status=None, stream=None) -> None:
    """Queue one W4A8 GEMV on `stream` (device buffers); raises on a bad argument."""
    check(
        lib().ks_b200_matvec_w4a8_async(
            addr(x), addr(w), w_stride, addr(s), scale_type, s_stride, addr(y), rows, cols,
            group, sx, zx, zw, addr(status), stream_handle(stream),
        )
    )


def matvec_i8_dequant_async(x, w, w_stride, ws, sa, y, rows, cols, zx=0, zw=0, stream=None) -> None:
    check(
        lib().ks_b200_matvec_i8_dequant_async(
            addr(x), addr(w), w_stride, addr(ws), sa, addr(y), rows, cols, zx, zw,
            stream_handle(stream),
        )
    )


def matvec_i8_async(x, w, w_stride, y, rows, cols, zx=0, zw=0, stream=None) -> None:
    check(
        lib().ks_b200_matvec_i8_async(
            addr(x), addr(w), w_stride, addr(y), rows, cols, zx, zw, stream_handle(stream)
        )
    )


def gemm_i8_requant_async(a, sa, w, ws, out_scale, out, m, n, k, lda=None, ldw=None, ldo=None,
                          acc_out=None, status=None, stream=None) -> None:
    check(
        lib().ks_b200_gemm_i8_requant_async(
            addr(a), lda or k, addr(sa), addr(w), ldw or k, addr(ws), out_scale, addr(out), ldo or n, m, n, k,
            addr(acc_out), addr(status), stream_handle(stream),
        )
    )


def gemm_i8_requant_batch_async(a, sa, w, ws, out_scale, out, m, n, k, lda=None, ldw=None, ldo=None,
                                status=None, stream=None) -> None:
    """count independent INT8 GEMMs with requantisation (lists of device tensors)."""
    count = len(w)
    if not (len(a) == len(sa) == len(ws) == len(out) == count):
        raise ValueError("batch lists differ in length")
    check(
        lib().ks_b200_gemm_i8_requant_batch_async(
            count, _ptr_array(a), lda or k, _ptr_array(sa), _ptr_array(w), ldw or k, _ptr_array(ws), out_scale,
            _ptr_array(out), ldo or n, m, n, k,
            addr(status), stream_handle(stream),
        )
    )


def gemm_w4a8_async(a, sx, w, s, out, m, n, k, group, lda=None, w_stride=None, s_stride=None, ldo=None,
                    scale_type=SCALE_F16, status=None, stream=None) -> None:
    """Batched W4A8 GEMM: out[m, n] = sx[m] * sum_g acc_g * s[n, g] (device buffers)."""
    check(
        lib().ks_b200_gemm_w4a8_async(
            addr(a), lda or k, addr(sx), addr(w), w_stride or (k + 1) // 2, addr(s), scale_type,
            s_stride or -(-k // group), addr(out), ldo or n, m, n, k, group, addr(status), stream_handle(stream),
        )
    )


def import_ggml_q4_0_async(blocks, block_row_stride, rows, cols, group, packed, packed_stride, scales,
                           scale_type=SCALE_F16, scale_stride=None, stream=None) -> None:
    """GGML Q4_0 blocks (device) -> packed int4 + positive group scales (device)."""
    check(
        lib().ks_b200_import_ggml_q4_0_async(
            addr(blocks), block_row_stride, rows, cols, group, addr(packed), packed_stride, addr(scales),
            scale_type, scale_stride or cols // group, stream_handle(stream),
        )
    )


def matvec_w4a8_f32in_async(x, w, w_stride, s, s_stride, y, rows, cols, group, scale_type=SCALE_F16, xq=None,
                            xs=None, status=None, stream=None) -> None:
    """W4A8 GEMV on f32 activations, quantised per token on the device."""
    check(
        lib().ks_b200_matvec_w4a8_f32in_async(
            addr(x), addr(w), w_stride, addr(s), scale_type, s_stride, addr(y), rows, cols, group, addr(xq),
            addr(xs), addr(status), stream_handle(stream),
        )
    )


def quantize_per_token_async(x, ldx, n_tokens, cols, q, ldq, scales, stream=None) -> None:
    """int8 per-token quantisation (s = max|x| / 127, round half to even)."""
    check(lib().ks_b200_quantize_per_token_async(addr(x), ldx, n_tokens, cols, addr(q), ldq, addr(scales),
                                                 stream_handle(stream)))


class GgmlReport(ctypes.Structure):
    """ks_b200_ggml_report (include/ks_b200_ggml.h)."""

    _fields_ = [("conversions", ctypes.c_uint64), ("mul_mat_calls", ctypes.c_uint64), ("tokens", ctypes.c_uint64),
                ("gemv_launches", ctypes.c_uint64), ("gemm_launches", ctypes.c_uint64)]


def ggml_report() -> dict:
    r = GgmlReport()
    lib().ks_b200_ggml_report_get(ctypes.byref(r))
    return {name: int(getattr(r, name)) for name, _ in GgmlReport._fields_}


class GgmlQ4_0:
    """A GGML Q4_0 weight converted once to the native W4A8 layout (device-resident),
    multiplied through ks_b200_ggml_mul_mat_q4_0_async."""

    def __init__(self, blocks, block_row_stride, rows, cols, stream=None):
        h = c_void_p()
        check(lib().ks_b200_ggml_q4_0_create(addr(blocks), block_row_stride, rows, cols, stream_handle(stream),
                                             ctypes.byref(h)))
        self.handle, self.rows, self.cols = h, rows, cols

    def mul_mat_async(self, src1, src1_stride, dst, dst_stride, n_tokens, status=None, stream=None) -> None:
        check(lib().ks_b200_ggml_mul_mat_q4_0_async(self.handle, addr(src1), src1_stride, addr(dst), dst_stride,
                                                    n_tokens, addr(status), stream_handle(stream)))

    def native(self):
        p, s = c_void_p(), c_void_p()
        check(lib().ks_b200_ggml_q4_0_native(self.handle, ctypes.byref(p), ctypes.byref(s), None, None))
        return p.value, s.value

    def close(self) -> None:
        if self.handle:
            check(lib().ks_b200_ggml_q4_0_destroy(self.handle))
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _ptr_array(objs):
    arr = (c_void_p * len(objs))(*[addr(o) for o in objs])
    return arr


def matvec_w4a8_batch_async(xs, ws, ss, ys, w_stride, s_stride, rows, cols, group, sx, zx=0, zw=0,
                            scale_type=SCALE_F16, status=None, stream=None) -> None:
    """Queue len(xs) independent W4A8 GEMVs of one shape as one launch."""
    n = len(xs)
    assert len(ws) == len(ss) == len(ys) == n
    check(
        lib().ks_b200_matvec_w4a8_batch_async(
            n, _ptr_array(xs), _ptr_array(ws), _ptr_array(ss), _ptr_array(ys), w_stride, scale_type, s_stride,
            rows, cols, group, sx, zx, zw, addr(status), stream_handle(stream),
        )
    )


def matvec_i8_batch_async(xs, ws, ys, w_stride, rows, cols, zx=0, zw=0, w_scales=None, sa=1.0,
                          stream=None) -> None:
    n = len(xs)
    check(
        lib().ks_b200_matvec_i8_batch_async(
            n, _ptr_array(xs), _ptr_array(ws), _ptr_array(w_scales) if w_scales is not None else None,
            _ptr_array(ys), w_stride, rows, cols, zx, zw, sa, stream_handle(stream),
        )
    )


class _Dtypes(dict):
    """KS_B200_DTYPE_* by torch dtype, looked up by name once (torch itself is not imported here)."""

    def __missing__(self, dtype):
        names = {"torch.float32": DTYPE_F32, "torch.float16": DTYPE_F16, "torch.bfloat16": DTYPE_BF16}
        if str(dtype) not in names:
            raise ValueError(f"{dtype} is not float32, float16 or bfloat16")
        return self.setdefault(dtype, names[str(dtype)])


_DTYPES = _Dtypes()


class _IsDtype(dict):
    """Whether a torch dtype is the one of this name, looked up by name once."""

    def __init__(self, name):
        super().__init__()
        self._name = name

    def __missing__(self, dtype):
        return self.setdefault(dtype, str(dtype) == self._name)


_INT32, _FLOAT32 = _IsDtype("torch.int32"), _IsDtype("torch.float32")


# The kv4 calls stand in a decode loop, so they take what they need from their tensors once and directly.
def _at(t):
    return None if t is None else t.data_ptr()


def _sequences(page_table, seq_lens, token_offsets=None):
    """The table's row stride and columns and the number of sequences, which table, lengths and offsets are for.  The
    columns are what a row holds: of a table that is part of a wider one the stride is more."""
    n_seqs = seq_lens.numel()
    stride, one = page_table.stride()
    rows, columns = page_table.shape
    if not _INT32[page_table.dtype] or rows < n_seqs or (one != 1 and columns > 1):
        raise ValueError("a page table must be int32 [n_seqs, pages], its rows contiguous")
    if stride < columns:
        if n_seqs > 1:
            raise ValueError("the rows of a page table may not lie over each other")
        stride = columns  # of a single row
    if not _INT32[seq_lens.dtype] or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be contiguous int32 [n_seqs]")
    if token_offsets is not None and (not _INT32[token_offsets.dtype] or token_offsets.numel() <= n_seqs or
                                      not token_offsets.is_contiguous()):
        raise ValueError("token_offsets must be contiguous int32 [n_seqs + 1]")
    return stride, n_seqs, columns


def _workspace(t):
    if not t.is_contiguous():
        raise ValueError("a workspace must be contiguous")
    return t.data_ptr()


def _bound(max_len, holds):
    """max_len, or what a row of the page table holds and it may not exceed."""
    if max_len is None:
        return holds
    if max_len > holds:
        raise KernelSmithError(KS_ERR_INVALID_ARG, "max_len is more than a row of the page table holds")
    return max_len


class Kv4Cache(ctypes.Structure):
    """ks_b200_kv4_cache (include/ks_b200.h): a pool of pages of 4-bit keys and values on the device,
    n_pages * kv4_page_bytes(...) bytes, and (or None) the tokens' accumulated attention weights, f32
    [n_pages, kv_heads, page_size].  The tensors are kept alive with it."""

    _fields_ = [("pool", _vp), ("weights", _vp), ("n_pages", _sz), ("page_size", _sz), ("kv_heads", _sz),
                ("head_dim", _sz), ("group_size", _sz)]

    def __init__(self, pool, n_pages, page_size, kv_heads, head_dim, group_size, weights=None):
        super().__init__(addr(pool), addr(weights), n_pages, page_size, kv_heads, head_dim, group_size)
        need = n_pages * kv4_page_bytes(page_size, kv_heads, head_dim, group_size)
        if hasattr(pool, "numel") and (pool.numel() * pool.element_size() < need or not pool.is_contiguous()):
            raise ValueError(f"a pool of {n_pages} such pages is {need} contiguous bytes")
        if hasattr(weights, "numel") and (weights.numel() < n_pages * kv_heads * page_size or
                                          not _FLOAT32[weights.dtype] or not weights.is_contiguous()):
            raise ValueError("weights must be contiguous f32 [n_pages, kv_heads, page_size]")
        self._tensors = (pool, weights)
        self._row, self._page = (kv_heads, head_dim), page_size
        self._address = ctypes.addressof(self)


def kv4_page_bytes(page_size, kv_heads, head_dim, group_size) -> int:
    return lib().ks_b200_kv4_page_bytes(page_size, kv_heads, head_dim, group_size)


def _kv4_rows(call, cache, page_table, seq_lens, k, v, token_offsets, status, stream) -> None:
    kt, kh, k1 = k.stride()
    vt, vh, v1 = v.stride()
    shape = k.shape
    if k.dtype != v.dtype or shape != v.shape or shape[1:] != cache._row or k1 != 1 or v1 != 1:
        raise ValueError("k and v must be [n_tokens, kv_heads, head_dim] of one type, the last dimension contiguous")
    stride, n_seqs, columns = _sequences(page_table, seq_lens, token_offsets)
    rc = call(cache._address, page_table.data_ptr(), stride, seq_lens.data_ptr(), _at(token_offsets), n_seqs,
              shape[0], columns * cache._page, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, _DTYPES[k.dtype],
              _at(status), stream_handle(stream))
    if rc:
        check(rc)


def kv4_append_async(cache, page_table, seq_lens, k, v, token_offsets=None, status=None, stream=None) -> None:
    """Quantise the newest tokens of each sequence, k and v [n_tokens, kv_heads, head_dim], into the cache."""
    _kv4_rows(lib().ks_b200_kv4_append_bounded_async, cache, page_table, seq_lens, k, v, token_offsets, status, stream)


def kv4_read_async(cache, page_table, seq_lens, k, v, token_offsets=None, status=None, stream=None) -> None:
    """Dequantise the newest tokens of each sequence into k and v [n_tokens, kv_heads, head_dim]."""
    _kv4_rows(lib().ks_b200_kv4_read_bounded_async, cache, page_table, seq_lens, k, v, token_offsets, status, stream)


def kv4_attention_workspace(cache, q_heads, n_seqs, n_tokens, max_new, max_len) -> int:
    return lib().ks_b200_kv4_attention_workspace(cache._address, q_heads, n_seqs, n_tokens, max_new, max_len)


def kv4_attention_async(cache, page_table, seq_lens, q, out, scale, workspace, token_offsets=None, max_new=None,
                        max_len=None, lse=None, accumulate=False, status=None, stream=None) -> None:
    """Attention of the newest tokens, q and out [n_tokens, q_heads, head_dim], over the cache.  max_new: no sequence
    has more new tokens (needed with token_offsets, else 1); max_len: no sequence is longer (default: what a row of the
    page table holds); workspace: a device byte tensor, zero-filled before its first use."""
    qt, qh, q1 = q.stride()
    ot, oh, o1 = out.stride()
    n_tokens, q_heads, head_dim = shape = q.shape
    if q.dtype != out.dtype or shape != out.shape or head_dim != cache._row[1] or q1 != 1 or o1 != 1:
        raise ValueError("q and out must be [n_tokens, q_heads, head_dim] of one type, the last dimension contiguous")
    if lse is not None and (lse.shape != shape[:2] or not _FLOAT32[lse.dtype] or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous f32 [n_tokens, q_heads]")
    stride, n_seqs, columns = _sequences(page_table, seq_lens, token_offsets)
    if max_new is None:
        if token_offsets is not None:
            raise ValueError("token_offsets needs max_new, the most new tokens of a sequence")
        max_new = 1
    max_len = _bound(max_len, columns * cache._page)
    rc = lib().ks_b200_kv4_attention_async(
        cache._address, page_table.data_ptr(), stride, seq_lens.data_ptr(), _at(token_offsets), n_seqs, n_tokens,
        max_new, max_len, q.data_ptr(), qt, qh, q_heads, scale, out.data_ptr(), ot, oh, _DTYPES[q.dtype], _at(lse),
        1 if accumulate else 0, _workspace(workspace), workspace.numel(), _at(status), stream_handle(stream))
    if rc:
        check(rc)


def kv4_evict_workspace(cache, n_seqs, max_len, budget) -> int:
    return lib().ks_b200_kv4_evict_workspace(cache._address, n_seqs, max_len, budget)


def kv4_evict_async(cache, page_table, seq_lens, to_table, to_lens, max_len, budget, recent, workspace, kept=None,
                    status=None, stream=None) -> None:
    """Keep the newest `recent` tokens of each sequence and head and the heaviest others, `budget` in all, in the
    pages of to_table; kept: None or int32 [n_seqs, kv_heads, budget] for their old positions; workspace: a device
    byte tensor, which may be the attention's."""
    stride, n_seqs, columns = _sequences(page_table, seq_lens)
    to_stride, to_seqs, to_columns = _sequences(to_table, to_lens)
    if to_seqs != n_seqs:
        raise ValueError("seq_lens and to_lens must be of one length")
    max_len = _bound(max_len, columns * cache._page)
    if to_columns * cache._page < min(budget, max_len):
        raise KernelSmithError(KS_ERR_INVALID_ARG, "a row of to_table holds fewer tokens than may be kept")
    if kept is not None and (kept.shape != (n_seqs, cache._row[0], budget) or not _INT32[kept.dtype] or
                             not kept.is_contiguous()):
        raise ValueError("kept must be a contiguous int32 [n_seqs, kv_heads, budget]")
    rc = lib().ks_b200_kv4_evict_async(
        cache._address, page_table.data_ptr(), stride, seq_lens.data_ptr(), n_seqs, max_len,
        to_table.data_ptr(), to_stride, to_lens.data_ptr(), budget, recent, _at(kept), _workspace(workspace),
        workspace.numel(), _at(status), stream_handle(stream))
    if rc:
        check(rc)


__all__ = [name for name in dir() if not name.startswith("_")]
