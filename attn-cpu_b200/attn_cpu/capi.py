"""capi -- ctypes access to the C ABI of libattnb.so (include/attnb.h).

The device-pointer entry points (``*_dev``) take raw device addresses and a
CUDA stream; the helpers below accept torch CUDA tensors (torch is used only
for device memory and streams) and enqueue on the current torch stream.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libattnb.so")

OK = 0
ERR_INVALID_ARGUMENT = 1
ERR_RUNTIME = 2
ERR_CUDA = 3
ERR_DEVICE_TIMEOUT = 4
ERR_OUT_OF_MEMORY = 5
ERR_INDEX = 6

PREC = {None: -1, "default": -1, "3xtf32": 0, "tf32": 1}

# Every symbol include/attnb.h declares.
EXPORTED = [
    "attnb_last_error", "attnb_version", "attnb_stream_status", "attnb_selftest_wait_timeout",
    "attnb_profile_enable", "attnb_profile_read", "attnb_host_alloc", "attnb_host_free",
    "attnb_sgemm", "attnb_gemm_jit", "attnb_sgemm_dev", "attnb_gemm_ex_dev",
    "attnb_gemm_ex_bcast_dev", "attnb_ipc_alloc", "attnb_ipc_free", "attnb_ipc_export", "attnb_ipc_import", "attnb_ipc_close",
    "attnb_linear_dev", "attnb_weight_pack_dev", "attnb_weight_free", "attnb_linear_packed_dev",
    "attnb_attn_step_dense", "attnb_attn_step_dense_dev", "attnb_attn_step_dense_noalloc",
    "attnb_attn_step_dense_bcast_dev", "attnb_peer_barrier_dev",
    "attnb_attn_block_dense", "attnb_attn_block_dense_dev",
    "attnb_attn_block_dense_batched_dev",
    "attnb_mha_block_dense", "attnb_mha_block_dense_dev",
    "attnb_kv_cache_create", "attnb_kv_cache_destroy", "attnb_kv_cache_length",
    "attnb_kv_cache_truncate", "attnb_kv_cache_append", "attnb_kv_cache_step",
    "attnb_kv_cache_step_dev",
    "attnb_seq_workspace", "attnb_attn_packed_dev", "attnb_attn_paged_dev",
    "attnb_kv_pages_append_dev", "attnb_kv_pages_read_dev", "attnb_kv_pages_append_rope_dev",
    "attnb_kv_blocks_bounds_dev", "attnb_blocks_workspace", "attnb_kv_blocks_select_dev",
    "attnb_attn_blocks_dev",
]


class Tensor(ctypes.Structure):
    """attnb_tensor / attnb_mtensor: data, H, T, Dh, strideH, strideT, strideDh."""
    _fields_ = [("data", ctypes.c_void_p), ("H", ctypes.c_int), ("T", ctypes.c_int),
                ("Dh", ctypes.c_int), ("strideH", ctypes.c_int64), ("strideT", ctypes.c_int64),
                ("strideDh", ctypes.c_int64)]


class Rows(ctypes.Structure):
    """attnb_rows: data, type, tokens, heads, Dh, strideT, strideH."""
    _fields_ = [("data", ctypes.c_void_p), ("type", ctypes.c_int), ("tokens", ctypes.c_int),
                ("heads", ctypes.c_int), ("Dh", ctypes.c_int), ("strideT", ctypes.c_int64),
                ("strideH", ctypes.c_int64)]


class KvPages(ctypes.Structure):
    """attnb_kv_pages: k, v, k_scale, v_scale, type, num_pages, H, page_size, Dh, k_group, v_group."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("type", ctypes.c_int), ("num_pages", ctypes.c_int),
                ("H", ctypes.c_int), ("page_size", ctypes.c_int), ("Dh", ctypes.c_int),
                ("k_group", ctypes.c_void_p), ("v_group", ctypes.c_void_p)]


class Rope(ctypes.Structure):
    """attnb_rope: inv_freq, pairs, interleaved."""
    _fields_ = [("inv_freq", ctypes.c_void_p), ("pairs", ctypes.c_int),
                ("interleaved", ctypes.c_int)]


class Bounds(ctypes.Structure):
    """attnb_bounds: data, type."""
    _fields_ = [("data", ctypes.c_void_p), ("type", ctypes.c_int)]


class Seqs(ctypes.Structure):
    """attnb_seqs: cu, batch, table, table_stride, max_pages, lens."""
    _fields_ = [("cu", ctypes.c_void_p), ("batch", ctypes.c_int), ("table", ctypes.c_void_p),
                ("table_stride", ctypes.c_int64), ("max_pages", ctypes.c_int),
                ("lens", ctypes.c_void_p)]


class AttnbError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"attnb error {code}: {msg}")
        self.code = code


class AttnbOutOfMemory(AttnbError, MemoryError):
    """ATTNB_ERR_OUT_OF_MEMORY: the device scratch the call needs could not be had."""


_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: run attn-cpu_b200/build.py")
        L = ctypes.CDLL(LIB_PATH)
        vp, i, f, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_int64
        T = ctypes.POINTER(Tensor)
        L.attnb_last_error.restype = ctypes.c_char_p
        L.attnb_version.restype = ctypes.c_char_p
        L.attnb_stream_status.argtypes = [vp]
        L.attnb_selftest_wait_timeout.argtypes = [i, vp]
        L.attnb_profile_enable.argtypes = [i]
        L.attnb_profile_read.argtypes = [ctypes.c_char_p, ctypes.POINTER(ctypes.c_double),
                                         ctypes.POINTER(ctypes.c_int)]
        L.attnb_host_alloc.argtypes = [ctypes.c_size_t, ctypes.POINTER(vp)]
        L.attnb_host_free.argtypes = [vp]
        L.attnb_sgemm.argtypes = [vp, i, i, vp, i, vp, f, f, i]
        L.attnb_gemm_jit.argtypes = [vp, i, i, vp, i, vp, f, f, i]
        L.attnb_sgemm_dev.argtypes = [vp, i, vp, i, vp, i, i, i, i, f, f, i, vp]
        L.attnb_linear_dev.argtypes = [vp, i, vp, i, vp, vp, i, i, i, i, i, vp]
        L.attnb_gemm_ex_dev.argtypes = [i, i, vp, i, vp, i, vp, vp, i, i, i, i, f, f, i, vp]
        L.attnb_gemm_ex_bcast_dev.argtypes = [i, i, vp, i, vp, i, vp, vp, i,
                                              ctypes.POINTER(vp), i, i, i, i, f, f, i, vp]
        L.attnb_weight_pack_dev.argtypes = [vp, i, i, i, i, ctypes.POINTER(vp), vp]
        L.attnb_weight_free.argtypes = [vp]
        L.attnb_linear_packed_dev.argtypes = [i, vp, i, vp, vp, vp, i, i, ctypes.POINTER(vp), i,
                                              vp]
        L.attnb_ipc_alloc.argtypes = [ctypes.c_size_t, ctypes.POINTER(vp)]
        L.attnb_ipc_free.argtypes = [vp]
        L.attnb_ipc_export.argtypes = [vp, vp, ctypes.POINTER(ctypes.c_uint64)]
        L.attnb_ipc_import.argtypes = [vp, ctypes.c_uint64, ctypes.POINTER(vp)]
        L.attnb_ipc_close.argtypes = [vp]
        L.attnb_attn_step_dense.argtypes = [T, T, T, T]
        L.attnb_attn_step_dense_dev.argtypes = [T, T, T, T, vp]
        L.attnb_attn_step_dense_noalloc.argtypes = [T, T, T, T, vp]
        L.attnb_attn_step_dense_bcast_dev.argtypes = [T, T, T, T, ctypes.POINTER(vp), i, vp]
        L.attnb_peer_barrier_dev.argtypes = [vp, ctypes.POINTER(vp), i, i, i, vp]
        L.attnb_attn_block_dense.argtypes = [T, T, T, T, i, i]
        L.attnb_attn_block_dense_dev.argtypes = [T, T, T, T, i, i, vp]
        L.attnb_attn_block_dense_batched_dev.argtypes = [T, T, T, T, i, i64, i64, i64, i64, i, i,
                                                         vp]
        L.attnb_mha_block_dense.argtypes = [vp, i, i, vp, vp, vp, vp, i, i, vp, i]
        L.attnb_mha_block_dense_dev.argtypes = [vp, i, i, i, vp, vp, vp, vp, i, i, vp, i, vp]
        L.attnb_kv_cache_create.argtypes = [i, i, i, ctypes.POINTER(vp)]
        L.attnb_kv_cache_destroy.argtypes = [vp]
        L.attnb_kv_cache_length.argtypes = [vp, ctypes.POINTER(i)]
        L.attnb_kv_cache_truncate.argtypes = [vp, i]
        L.attnb_kv_cache_append.argtypes = [vp, vp, vp, i, vp]
        L.attnb_kv_cache_step.argtypes = [vp, vp, vp, vp, vp]
        L.attnb_kv_cache_step_dev.argtypes = [vp, vp, vp, vp, vp, vp]
        R, P, S = (ctypes.POINTER(x) for x in (Rows, KvPages, Seqs))
        L.attnb_seq_workspace.argtypes = [i, i, i, ctypes.POINTER(ctypes.c_size_t)]
        L.attnb_attn_packed_dev.argtypes = [R, R, R, R, vp, vp, i, i, f, vp, ctypes.c_size_t, vp]
        L.attnb_attn_paged_dev.argtypes = [R, P, R, S, i, i, f, vp, ctypes.c_size_t, vp]
        L.attnb_kv_pages_append_dev.argtypes = [R, R, P, S, vp]
        L.attnb_kv_pages_read_dev.argtypes = [P, R, R, S, vp]
        B = ctypes.POINTER(Bounds)
        L.attnb_kv_pages_append_rope_dev.argtypes = [R, R, R, R, P, S, ctypes.POINTER(Rope), vp]
        L.attnb_kv_blocks_bounds_dev.argtypes = [P, B, S, vp]
        L.attnb_blocks_workspace.argtypes = [i, i, i, i, i, i, ctypes.POINTER(ctypes.c_size_t)]
        L.attnb_kv_blocks_select_dev.argtypes = [R, B, i, i, i, S, i, i, vp, i, vp, ctypes.c_size_t,
                                                 vp]
        L.attnb_attn_blocks_dev.argtypes = [R, P, R, S, vp, i, f, vp, ctypes.c_size_t, vp]
        for name in EXPORTED:
            if name not in ("attnb_last_error", "attnb_version"):
                getattr(L, name).restype = ctypes.c_int
        _lib = L
    return _lib


def check(rc: int) -> None:
    if rc != OK:
        cls = AttnbOutOfMemory if rc == ERR_OUT_OF_MEMORY else AttnbError
        raise cls(rc, lib().attnb_last_error().decode())


def _stream(stream=None) -> int:
    import torch

    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def tensor3(t, as_2d: bool = False) -> Tensor:
    """attnb_tensor view of a float32 CUDA tensor [H,T,Dh] (or [H,Dh] with as_2d)."""
    if as_2d:
        H, Dh = t.shape
        return Tensor(t.data_ptr(), H, 1, Dh, t.stride(0), 0, t.stride(1))
    H, T_, Dh = t.shape
    return Tensor(t.data_ptr(), H, T_, Dh, t.stride(0), t.stride(1), t.stride(2))


def sgemm_dev(A, B, C, alpha=1.0, beta=0.0, precision=None, stream=None) -> None:
    """C = alpha * A @ B + beta * C on 2-D float32 CUDA tensors with unit column stride."""
    M, K = A.shape
    N = B.shape[1]
    check(lib().attnb_sgemm_dev(A.data_ptr(), A.stride(0), B.data_ptr(), B.stride(0),
                                C.data_ptr(), C.stride(0), M, N, K, alpha, beta,
                                PREC[precision], _stream(stream)))


def gemm_ex_dev(A, B, C, trans_a=False, trans_b=False, bias=None, alpha=1.0, beta=0.0,
                precision=None, stream=None) -> None:
    """C = alpha * op(A) @ op(B) + beta * C + bias, op(X) = X.T when trans_x.
    A, B, C: 2-D float32 CUDA tensors with unit column stride (A and B may be
    column slices: their row pitch is passed as the leading dimension)."""
    M = A.shape[1] if trans_a else A.shape[0]
    K = A.shape[0] if trans_a else A.shape[1]
    N = B.shape[0] if trans_b else B.shape[1]
    if (B.shape[1] if trans_b else B.shape[0]) != K or tuple(C.shape) != (M, N):
        raise ValueError("gemm_ex_dev: shapes do not match")
    if A.stride(1) != 1 or B.stride(1) != 1 or C.stride(1) != 1:
        raise ValueError("gemm_ex_dev: operands need a unit column stride")
    check(lib().attnb_gemm_ex_dev(int(trans_a), int(trans_b), A.data_ptr(), A.stride(0),
                                  B.data_ptr(), B.stride(0),
                                  bias.data_ptr() if bias is not None else None, C.data_ptr(),
                                  C.stride(0), M, N, K, alpha, beta, PREC[precision],
                                  _stream(stream)))


def gemm_ex_bcast_dev(A, B, C, replicas, trans_a=False, trans_b=False, bias=None, alpha=1.0,
                      beta=0.0, precision=None, stream=None) -> None:
    """gemm_ex_dev that also writes C, element for element, into each address
    in `replicas` (device addresses as ints, same layout and leading dimension
    as C -- e.g. C's rows in the other GPUs' replicas, from ipc_import)."""
    M = A.shape[1] if trans_a else A.shape[0]
    K = A.shape[0] if trans_a else A.shape[1]
    N = B.shape[0] if trans_b else B.shape[1]
    if (B.shape[1] if trans_b else B.shape[0]) != K or tuple(C.shape) != (M, N):
        raise ValueError("gemm_ex_bcast_dev: shapes do not match")
    if A.stride(1) != 1 or B.stride(1) != 1 or C.stride(1) != 1:
        raise ValueError("gemm_ex_bcast_dev: operands need a unit column stride")
    arr = (ctypes.c_void_p * max(1, len(replicas)))(*[int(r) for r in replicas])
    check(lib().attnb_gemm_ex_bcast_dev(int(trans_a), int(trans_b), A.data_ptr(), A.stride(0),
                                        B.data_ptr(), B.stride(0),
                                        bias.data_ptr() if bias is not None else None,
                                        C.data_ptr(), C.stride(0), arr, len(replicas), M, N, K,
                                        alpha, beta, PREC[precision], _stream(stream)))


IPC_HANDLE_BYTES = 64


class _SharedBlock:
    """A device allocation of its own (attnb_ipc_alloc), exposed through the
    CUDA array interface so torch can view it; freed when the last view dies."""

    def __init__(self, shape: tuple):
        n = 1
        for d in shape:
            n *= int(d)
        p = ctypes.c_void_p()
        check(lib().attnb_ipc_alloc(max(4, 4 * n), ctypes.byref(p)))
        self.ptr = p.value
        self.__cuda_array_interface__ = {"shape": tuple(int(d) for d in shape), "typestr": "<f4",
                                         "data": (self.ptr, False), "version": 3,
                                         "strides": None}

    def __del__(self):
        try:
            lib().attnb_ipc_free(self.ptr)
        except Exception:  # interpreter shutdown: the library may be gone
            pass


def shared_empty(shape: tuple):
    """An uninitialised float32 CUDA tensor on the current device in an
    allocation of its own, exportable with ipc_export."""
    import torch

    return torch.as_tensor(_SharedBlock(tuple(shape)), device="cuda")


def ipc_export(t) -> tuple[bytes, int]:
    """(handle, byte offset) of the device allocation holding CUDA tensor `t`,
    for ipc_import in another process of the node."""
    h = ctypes.create_string_buffer(IPC_HANDLE_BYTES)
    off = ctypes.c_uint64()
    check(lib().attnb_ipc_export(t.data_ptr(), h, ctypes.byref(off)))
    return h.raw, off.value


def ipc_import(handle: bytes, offset: int) -> int:
    """Device address, in the current device's context, of another process's
    allocation (see ipc_export); release with ipc_close."""
    if len(handle) != IPC_HANDLE_BYTES:
        raise ValueError("ipc handle must be 64 bytes")
    p = ctypes.c_void_p()
    check(lib().attnb_ipc_import(handle, offset, ctypes.byref(p)))
    return p.value


def ipc_close(ptr: int) -> None:
    check(lib().attnb_ipc_close(ptr))


class PackedWeight:
    """A projection weight W [N, K] (float32 CUDA tensor, unit column stride)
    packed once on the current device for repeated y = x W^T
    (attnb_weight_pack_dev); the packing is enqueued on `stream`."""

    def __init__(self, W, precision=None, stream=None):
        import torch

        if W.dim() != 2 or W.stride(1) != 1 or W.dtype != torch.float32:
            raise ValueError("PackedWeight: W must be 2-D float32 with a unit column stride")
        self.N, self.K = W.shape
        self._h = ctypes.c_void_p()
        check(lib().attnb_weight_pack_dev(W.data_ptr(), W.stride(0), self.N, self.K,
                                          PREC[precision], ctypes.byref(self._h),
                                          _stream(stream)))

    def close(self) -> None:
        if self._h:
            check(lib().attnb_weight_free(self._h))
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter shutdown: the library may be gone
            pass


def linear_packed_dev(x, W: PackedWeight, b, y, trans_x=False, replicas=(), stream=None) -> None:
    """y = op(x) @ W^T + b (b may be None), op(x) = x.T when trans_x; y is also
    stored into each address in `replicas` (see gemm_ex_bcast_dev)."""
    M = x.shape[1] if trans_x else x.shape[0]
    K = x.shape[0] if trans_x else x.shape[1]
    if K != W.K or tuple(y.shape) != (M, W.N):
        raise ValueError("linear_packed_dev: shapes do not match")
    if x.stride(1) != 1 or y.stride(1) != 1:
        raise ValueError("linear_packed_dev: operands need a unit column stride")
    if x.dtype != y.dtype or str(x.dtype) != "torch.float32":
        raise ValueError("linear_packed_dev: x and y must be float32")
    arr = (ctypes.c_void_p * max(1, len(replicas)))(*[int(r) for r in replicas])
    check(lib().attnb_linear_packed_dev(int(trans_x), x.data_ptr(), x.stride(0), W._h,
                                        b.data_ptr() if b is not None else None, y.data_ptr(),
                                        y.stride(0), M, arr, len(replicas), _stream(stream)))


def linear_dev(x, W, b, y, precision=None, stream=None) -> None:
    """y = x @ W^T + b (b may be None)."""
    T_, K = x.shape
    N = W.shape[0]
    check(lib().attnb_linear_dev(x.data_ptr(), x.stride(0), W.data_ptr(), W.stride(0),
                                 b.data_ptr() if b is not None else None, y.data_ptr(),
                                 y.stride(0), T_, N, K, PREC[precision], _stream(stream)))


def attn_step_dense_dev(Q, K, V, O, stream=None) -> None:
    q, k, v, o = tensor3(Q, True), tensor3(K), tensor3(V), tensor3(O, True)
    check(lib().attnb_attn_step_dense_dev(ctypes.byref(q), ctypes.byref(k), ctypes.byref(v),
                                          ctypes.byref(o), _stream(stream)))


def attn_step_dense_bcast_dev(Q, K, V, O, replicas, stream=None) -> None:
    """attn_step_dense_dev that also stores O into each address in `replicas`
    (device addresses as ints: O's heads in other GPUs' copies)."""
    q, k, v, o = tensor3(Q, True), tensor3(K), tensor3(V), tensor3(O, True)
    arr = (ctypes.c_void_p * max(1, len(replicas)))(*[int(r) for r in replicas])
    check(lib().attnb_attn_step_dense_bcast_dev(ctypes.byref(q), ctypes.byref(k),
                                                ctypes.byref(v), ctypes.byref(o), arr,
                                                len(replicas), _stream(stream)))


def peer_barrier_dev(flags: int, peer_flags: list, rank: int, limit_us: int = 0,
                     stream=None) -> None:
    """Enqueue the next peer-memory barrier (attnb_peer_barrier_dev): `flags`
    is this rank's array (one epoch per rank, then its barrier count),
    peer_flags[r] rank r's array as mapped here (any value at index `rank`)."""
    n = len(peer_flags)
    arr = (ctypes.c_void_p * n)(*[int(p) if p else None for p in peer_flags])
    check(lib().attnb_peer_barrier_dev(flags, arr, n, rank, limit_us, _stream(stream)))


def attn_step_dense_noalloc(Q, K, V, O, stream=None) -> None:
    """Decode step without any device allocation (fixed 2 MiB scratch shared by
    all calls; see attnb_attn_step_dense_noalloc in include/attnb.h)."""
    q, k, v, o = tensor3(Q, True), tensor3(K), tensor3(V), tensor3(O, True)
    check(lib().attnb_attn_step_dense_noalloc(ctypes.byref(q), ctypes.byref(k), ctypes.byref(v),
                                              ctypes.byref(o), _stream(stream)))


def attn_block_dense_dev(Q, K, V, O, causal=False, precision=None, stream=None) -> None:
    q, k, v, o = tensor3(Q), tensor3(K), tensor3(V), tensor3(O)
    check(lib().attnb_attn_block_dense_dev(ctypes.byref(q), ctypes.byref(k), ctypes.byref(v),
                                           ctypes.byref(o), int(causal), PREC[precision],
                                           _stream(stream)))


def attn_block_dense_batched_dev(Q, K, V, O, causal=False, precision=None, stream=None) -> None:
    """Prefill for independent sequences: Q, O [B, H, L, Dh] and K, V [B, H, T, Dh]
    float32 CUDA views (any strides); the sequences run side by side."""
    if not (Q.dim() == K.dim() == V.dim() == O.dim() == 4):
        raise ValueError("attn_block_dense_batched_dev: 4-D views [B, H, T, Dh] expected")
    B = Q.shape[0]
    if K.shape[0] != B or V.shape[0] != B or O.shape[0] != B:
        raise ValueError("attn_block_dense_batched_dev: batch sizes differ")
    if B == 0:
        return
    q, k, v, o = tensor3(Q[0]), tensor3(K[0]), tensor3(V[0]), tensor3(O[0])
    check(lib().attnb_attn_block_dense_batched_dev(
        ctypes.byref(q), ctypes.byref(k), ctypes.byref(v), ctypes.byref(o), B, Q.stride(0),
        K.stride(0), V.stride(0), O.stride(0), int(causal), PREC[precision], _stream(stream)))


def mha_block_dense_dev(x, W_in, b_in, W_out, b_out, num_heads, y, causal=False,
                        precision=None, stream=None) -> None:
    """x, y: [batch, T, D] (or [T, D]) contiguous float32 CUDA tensors."""
    if x.dim() == 2:
        batch, (T_, D) = 1, x.shape
    else:
        batch, T_, D = x.shape
    check(lib().attnb_mha_block_dense_dev(x.data_ptr(), batch, T_, D, W_in.data_ptr(),
                                          b_in.data_ptr(), W_out.data_ptr(), b_out.data_ptr(),
                                          num_heads, int(causal), y.data_ptr(), PREC[precision],
                                          _stream(stream)))


def profile_enable(on: bool = True) -> None:
    check(lib().attnb_profile_enable(int(on)))


def profile_read(kernel: str) -> tuple[float, int]:
    """(summed milliseconds, launches) of `kernel` since the last read."""
    ms, n = ctypes.c_double(), ctypes.c_int()
    check(lib().attnb_profile_read(kernel.encode(), ctypes.byref(ms), ctypes.byref(n)))
    return ms.value, n.value


def stream_status(stream=None) -> None:
    check(lib().attnb_stream_status(_stream(stream)))


class KVCacheDev:
    """The resident K/V cache (attnb_kv_cache_*) driven with CUDA tensors.

    K and V stay on the device current at construction, [H, capacity, Dh];
    ``append`` and ``step`` enqueue on ``stream`` (default: torch's current
    stream) and return without synchronising."""

    def __init__(self, H: int, Dh: int, capacity: int):
        self._h = ctypes.c_void_p()
        check(lib().attnb_kv_cache_create(H, Dh, capacity, ctypes.byref(self._h)))
        self.H, self.Dh = H, Dh

    def __len__(self) -> int:
        n = ctypes.c_int()
        check(lib().attnb_kv_cache_length(self._h, ctypes.byref(n)))
        return n.value

    def truncate(self, length: int) -> None:
        check(lib().attnb_kv_cache_truncate(self._h, length))

    def append(self, k, v, stream=None) -> None:
        """k, v: [H, n, Dh] contiguous float32 tensors (CUDA or CPU)."""
        check(lib().attnb_kv_cache_append(self._h, k.data_ptr(), v.data_ptr(), k.shape[1],
                                          _stream(stream)))

    def step(self, q, o, k_new=None, v_new=None, stream=None) -> None:
        """o[H, Dh] = attention of q[H, Dh] over the cache, after appending k_new, v_new."""
        kp = k_new.data_ptr() if k_new is not None else None
        vp_ = v_new.data_ptr() if v_new is not None else None
        check(lib().attnb_kv_cache_step_dev(self._h, q.data_ptr(), kp, vp_, o.data_ptr(),
                                            _stream(stream)))

    def close(self) -> None:
        if self._h:
            check(lib().attnb_kv_cache_destroy(self._h))
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter shutdown: the library may be gone
            pass


# ------------------------------------------------- ragged sequences, paged KV cache
# These calls are made once per layer and step, where a few microseconds of the
# host count: the checks below read each property of a tensor once.
_torch = _raw_stream = None
_I4 = 6  # torch.uint8 pages: two 4-bit codes a byte
_TYPES: dict = {}  # torch dtype -> ATTNB_TYPE_*
_workspace_bytes: dict = {}


def _setup() -> None:
    global _torch, _TYPES, _raw_stream
    import torch

    _torch = torch
    # torch's current stream as an address, without an object around it.
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
        lambda index: torch.cuda.current_stream(index).cuda_stream)
    _TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3,
              torch.int8: 4, torch.uint8: _I4}
    lib()


def _on(device, stream):
    """None when `device` is current and no stream is given (the usual case),
    else a context that makes both current: what is allocated inside belongs to
    that stream."""
    if _torch is None:
        _setup()
    if device.type != "cuda":
        raise ValueError("CUDA tensors expected")
    if stream is not None:
        if stream.device != device:
            raise ValueError(f"stream is on {stream.device}, not on {device}")
        return _torch.cuda.stream(stream)
    if device.index != _torch.cuda.current_device():
        return _torch.cuda.device(device)
    return None


def _rows(t, name: str, device) -> Rows:
    """attnb_rows view of a CUDA tensor [tokens, heads, Dh]."""
    try:
        n, h, d = t.shape
    except ValueError:
        raise ValueError(f"{name} must be [tokens, heads, Dh]") from None
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    sT, sH, sD = t.stride()
    if sD != 1 and d > 1:
        raise ValueError(f"{name} needs a unit stride of the head size")
    ty = _TYPES.get(t.dtype)
    if ty is None:
        raise ValueError(f"{name}: {t.dtype} is not supported")
    return Rows(t.data_ptr(), ty, n, h, d, sT, sH)


def _offsets(t, name: str, device, n=None) -> int:
    """Device address of a contiguous int32 vector (of n entries)."""
    shape = t.shape
    if t.dtype != _torch.int32 or len(shape) != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector")
    if n is not None and shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, one more than sequences for offsets")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    return t.data_ptr()


def _pages(k_pages, v_pages, k_scale, v_scale, device, k_group=None, v_group=None) -> KvPages:
    shape, dtype = k_pages.shape, k_pages.dtype
    if len(shape) != 4 or shape != v_pages.shape or dtype != v_pages.dtype:
        raise ValueError("k_pages and v_pages must be [pages, H, page_size, Dh] of one type")
    n, H, page, Dh = shape
    ty = _TYPES.get(dtype)
    if ty is None:
        raise ValueError(f"k_pages: {dtype} is not supported")
    ks = vs = None
    if k_pages.device != device or v_pages.device != device:
        raise ValueError(f"pages and scales must be on {device}, not on {k_pages.device} "
                         f"and {v_pages.device}")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("pages and scales must be contiguous")
    if k_scale is not None:
        ks = _scales(k_scale, (n, H, page), device)
    if v_scale is not None:
        vs = ks if v_scale is k_scale else _scales(v_scale, (n, H, page), device)
    if ty != _I4:
        if k_group is not None or v_group is not None:
            raise ValueError("only uint8 pages have k_group and v_group")
        return KvPages(k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, ty, n, H, page, Dh)
    Dh *= 2
    want = (n, H, page, 4 * -(-Dh // 128))
    for t in (k_group, v_group):
        if t is None or t.dtype != _torch.uint8 or t.shape != want or not t.is_contiguous():
            raise ValueError(f"uint8 pages need k_group and v_group, contiguous uint8 {want}")
        if t.device != device:
            raise ValueError(f"pages and factors must be on {device}, not on {t.device}")
    return KvPages(k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, ty, n, H, page, Dh,
                   k_group.data_ptr(), v_group.data_ptr())


def _scales(t, shape, device) -> int:
    if t.device != device:
        raise ValueError(f"pages and scales must be on {device}, not on {t.device}")
    if not t.is_contiguous():
        raise ValueError("pages and scales must be contiguous")
    if t.dtype != _torch.float32 or t.shape != shape:
        raise ValueError("k_scale and v_scale must be float32 [pages, H, page_size]")
    return t.data_ptr()


def i4_group_bytes(Dh: int) -> int:
    """Length of the last dimension of a 4-bit cache's k_group and v_group."""
    return 4 * -(-Dh // 128)


def _seqs(cu, table, lens, device) -> Seqs:
    shape = table.shape
    if len(shape) != 2 or table.dtype != _torch.int32 or table.device != device:
        raise ValueError(f"table must be int32 [sequences, pages] on {device}, rows contiguous")
    batch, width = shape
    stride, step = table.stride()
    if width > 1 and step != 1:
        raise ValueError(f"table must be int32 [sequences, pages] on {device}, rows contiguous")
    return Seqs(_offsets(cu, "cu", device, batch + 1), batch, table.data_ptr(), stride, width,
                _offsets(lens, "lens", device, batch))


def _workspace(device, q_heads: int, kv_heads: int, Dh: int):
    """A fresh workspace from torch's allocator: calls in flight at the same
    time, and captured graphs, each have their own."""
    if kv_heads == 0 or q_heads % kv_heads:
        raise ValueError("Q heads must be a multiple of the KV heads")
    key = (device.index, q_heads, kv_heads, Dh)
    n = _workspace_bytes.get(key)
    if n is None:
        size = ctypes.c_size_t()
        check(lib().attnb_seq_workspace(q_heads, kv_heads, Dh, ctypes.byref(size)))
        n = _workspace_bytes[key] = size.value
    return _torch.empty(n, dtype=_torch.uint8, device=device), n


def _scale(scale) -> float:
    if scale is None:
        return 0.0  # the library's 1 / sqrt(Dh)
    if not ctypes.c_float(float(scale)).value > 0:  # as the library sees it: 0 is the default there
        raise ValueError("scale must be positive")
    return float(scale)


def attn_packed_dev(Q, K, V, O, cu_q, cu_k=None, causal=False, scale=None, stream=None) -> None:
    """O = attention of packed sequences (attnb_attn_packed_dev): Q, O [tokens,
    heads, Dh], K, V [tokens, kv_heads, Dh], float32, bfloat16 or float16 CUDA
    tensors; sequence b is rows cu_q[b]:cu_q[b+1] of Q and O and cu_k[b]:cu_k[b+1]
    of K and V (int32; cu_k defaults to cu_q).  causal: the last row of a
    sequence sees all its keys, each row before it one less.  heads is a
    multiple of kv_heads.  Rows of O behind cu_q[-1] stay as they are."""
    dev = Q.device
    on = _on(dev, stream)
    if on is not None:
        with on:
            return attn_packed_dev(Q, K, V, O, cu_q, cu_k, causal, scale)
    q, k, v, o = _rows(Q, "Q", dev), _rows(K, "K", dev), _rows(V, "V", dev), _rows(O, "O", dev)
    cq = _offsets(cu_q, "cu_q", dev)
    batch = len(cu_q) - 1
    if batch < 0:
        raise ValueError("cu_q must have one entry more than there are sequences")
    ck = cq if cu_k is None else _offsets(cu_k, "cu_k", dev, batch + 1)
    ws, n = _workspace(dev, q.heads, k.heads, q.Dh)
    check(_lib.attnb_attn_packed_dev(q, k, v, o, cq, ck, batch, int(causal), _scale(scale),
                                     ws.data_ptr(), n, _raw_stream(dev.index)))


def attn_paged_dev(Q, k_pages, v_pages, O, cu, table, lens, max_new=0, causal=True, scale=None,
                   k_scale=None, v_scale=None, stream=None, k_group=None, v_group=None) -> None:
    """O = attention of new tokens over a paged cache (attnb_attn_paged_dev): Q,
    O [tokens, heads, Dh]; k_pages, v_pages [pages, kv_heads, page_size, Dh] of
    Q's type, or float8_e4m3fn or int8 codes with k_scale, v_scale [pages,
    kv_heads, page_size], or uint8 [pages, kv_heads, page_size, Dh / 2], two 4-bit
    codes a byte, with scales and k_group, v_group, uint8 [pages, kv_heads,
    page_size, i4_group_bytes(Dh)]; sequence b is rows cu[b]:cu[b+1] of Q, the last of the
    lens[b] tokens in pages table[b] (all int32).  max_new: the most rows of one
    sequence, where the caller knows it; it only steers the choice of kernel."""
    dev = Q.device
    on = _on(dev, stream)
    if on is not None:
        with on:
            return attn_paged_dev(Q, k_pages, v_pages, O, cu, table, lens, max_new, causal, scale,
                                  k_scale, v_scale, None, k_group, v_group)
    q, o = _rows(Q, "Q", dev), _rows(O, "O", dev)
    pg = _pages(k_pages, v_pages, k_scale, v_scale, dev, k_group, v_group)
    sq = _seqs(cu, table, lens, dev)
    ws, n = _workspace(dev, q.heads, pg.H, q.Dh)
    check(_lib.attnb_attn_paged_dev(q, pg, o, sq, max_new, int(causal), _scale(scale),
                                    ws.data_ptr(), n, _raw_stream(dev.index)))


def kv_pages_append_dev(K, V, k_pages, v_pages, cu, table, lens, k_scale=None, v_scale=None,
                        stream=None, k_group=None, v_group=None) -> None:
    """Write new tokens K, V [tokens, kv_heads, Dh] into the pages, quantising
    them for float8_e4m3fn, int8 and uint8 pages (attnb_kv_pages_append_dev); lens
    counts them already.  Other arguments as in attn_paged_dev."""
    dev = K.device
    on = _on(dev, stream)
    if on is not None:
        with on:
            return kv_pages_append_dev(K, V, k_pages, v_pages, cu, table, lens, k_scale, v_scale,
                                       None, k_group, v_group)
    check(_lib.attnb_kv_pages_append_dev(
        _rows(K, "K", dev), _rows(V, "V", dev),
        _pages(k_pages, v_pages, k_scale, v_scale, dev, k_group, v_group),
        _seqs(cu, table, lens, dev), _raw_stream(dev.index)))


def kv_pages_append_rope_dev(K, V, k_pages, v_pages, cu, table, lens, inv_freq, interleaved=False,
                             Q=None, Q_out=None, k_scale=None, v_scale=None, stream=None,
                             k_group=None, v_group=None) -> None:
    """kv_pages_append_dev with K rotated by its tokens' positions on the way, and
    the queries Q [tokens, heads, Dh] rotated into Q_out, which may be Q
    (attnb_kv_pages_append_rope_dev).  inv_freq: float32 [pairs], the angle of
    each pair of dimensions from one position to the next; the pairs are (i, i + pairs)
    or, interleaved, (2i, 2i + 1), and dimensions from 2 * pairs on stay."""
    dev = K.device
    on = _on(dev, stream)
    if on is not None:
        with on:
            return kv_pages_append_rope_dev(K, V, k_pages, v_pages, cu, table, lens, inv_freq,
                                            interleaved, Q, Q_out, k_scale, v_scale, None, k_group,
                                            v_group)
    if inv_freq.dtype != _torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() or \
            inv_freq.device != dev:
        raise ValueError(f"inv_freq must be a contiguous float32 vector on {dev}")
    if (Q is None) != (Q_out is None):
        raise ValueError("Q and Q_out belong together")
    check(_lib.attnb_kv_pages_append_rope_dev(
        None if Q is None else _rows(Q, "Q", dev),
        None if Q is None else _rows(Q_out, "Q_out", dev), _rows(K, "K", dev), _rows(V, "V", dev),
        _pages(k_pages, v_pages, k_scale, v_scale, dev, k_group, v_group),
        _seqs(cu, table, lens, dev), Rope(inv_freq.data_ptr(), len(inv_freq), int(interleaved)),
        _raw_stream(dev.index)))


def kv_pages_read_dev(k_pages, v_pages, K, V, cu, table, lens, k_scale=None, v_scale=None,
                      stream=None, k_group=None, v_group=None) -> None:
    """Read the last cu[b+1] - cu[b] tokens of each sequence out of the pages
    into K, V [tokens, kv_heads, Dh] (attnb_kv_pages_read_dev)."""
    dev = K.device
    on = _on(dev, stream)
    if on is not None:
        with on:
            return kv_pages_read_dev(k_pages, v_pages, K, V, cu, table, lens, k_scale, v_scale,
                                     None, k_group, v_group)
    check(_lib.attnb_kv_pages_read_dev(
        _pages(k_pages, v_pages, k_scale, v_scale, dev, k_group, v_group), _rows(K, "K", dev),
        _rows(V, "V", dev), _seqs(cu, table, lens, dev), _raw_stream(dev.index)))


def _bounds(bounds, pages: int, heads: int, Dh: int, device) -> Bounds:
    if bounds.shape != (pages, heads, 2, Dh) or not bounds.is_contiguous() or \
            bounds.device != device:
        raise ValueError(f"bounds must be [pages, H, 2, Dh] = {(pages, heads, 2, Dh)}, contiguous, "
                         f"on {device}")
    ty = _TYPES.get(bounds.dtype)
    if ty is None:
        raise ValueError(f"bounds: {bounds.dtype} is not supported")
    return Bounds(bounds.data_ptr(), ty)


def _lists(blocks, tokens: int, heads: int, device) -> int:
    if blocks.dtype != _torch.int32 or blocks.dim() != 3 or \
            tuple(blocks.shape[:2]) != (tokens, heads) or not blocks.is_contiguous():
        raise ValueError(f"blocks must be contiguous int32 [{tokens}, {heads}, take]")
    if blocks.device != device:
        raise ValueError(f"blocks is on {blocks.device}, not on {device}")
    return blocks.data_ptr()


@functools.lru_cache(maxsize=4096)
def _blocks_bytes(index, tokens, q_heads, kv_heads, Dh, take, max_pages) -> int:
    size = ctypes.c_size_t()
    check(_lib.attnb_blocks_workspace(tokens, q_heads, kv_heads, Dh, take, max_pages,
                                      ctypes.byref(size)))
    return size.value


def _blocks_workspace(device, tokens, q_heads, kv_heads, Dh, take, max_pages):
    """As _workspace, for the selection of blocks."""
    n = _blocks_bytes(device.index, tokens, q_heads, kv_heads, Dh, take, max_pages)
    return _torch.empty(n, dtype=_torch.uint8, device=device), n


def kv_blocks_bounds_dev(k_pages, bounds, cu, table, lens, k_scale=None, k_group=None,
                         stream=None) -> None:
    """Least and greatest value of the keys of each block (one page of a sequence)
    that the new tokens complete, into bounds [pages, kv_heads, 2, Dh]
    (attnb_kv_blocks_bounds_dev): float32, bfloat16 or float16, for uncoded pages
    their type.  Call it after each append; other arguments as there."""
    dev = k_pages.device
    on = _on(dev, stream)
    if on is not None:
        with on:
            return kv_blocks_bounds_dev(k_pages, bounds, cu, table, lens, k_scale, k_group)
    pg = _pages(k_pages, k_pages, k_scale, k_scale, dev, k_group, k_group)
    check(_lib.attnb_kv_blocks_bounds_dev(pg, _bounds(bounds, pg.num_pages, pg.H, pg.Dh, dev),
                                          _seqs(cu, table, lens, dev), _raw_stream(dev.index)))


def kv_blocks_select_dev(Q, bounds, blocks, cu, table, lens, page_size, keep_first=1, keep_last=1,
                         stream=None) -> None:
    """The blocks that each of Q's tokens [tokens, heads, Dh] attends to, by their
    bounds, into blocks, int32 [tokens, kv_heads, take], ascending, -1 behind the
    last one (attnb_kv_blocks_select_dev): the first keep_first, the last keep_last
    (the token's own is the last), and those that may hold the greatest scores."""
    dev = Q.device
    on = _on(dev, stream)
    if on is not None:
        with on:
            return kv_blocks_select_dev(Q, bounds, blocks, cu, table, lens, page_size, keep_first,
                                        keep_last)
    q = _rows(Q, "Q", dev)
    if bounds.dim() != 4:
        raise ValueError("bounds must be [pages, H, 2, Dh]")
    n, H = bounds.shape[:2]
    b = _bounds(bounds, n, H, q.Dh, dev)
    at, take = _lists(blocks, q.tokens, H, dev), blocks.shape[2]
    sq = _seqs(cu, table, lens, dev)
    ws, size = _blocks_workspace(dev, q.tokens, q.heads, H, q.Dh, take, sq.max_pages)
    check(_lib.attnb_kv_blocks_select_dev(q, b, n, H, page_size, sq, keep_first, keep_last, at,
                                          take, ws.data_ptr(), size, _raw_stream(dev.index)))


def attn_blocks_dev(Q, k_pages, v_pages, O, blocks, cu, table, lens, scale=None, k_scale=None,
                    v_scale=None, stream=None, k_group=None, v_group=None) -> None:
    """attn_paged_dev, causal, over the listed blocks alone (attnb_attn_blocks_dev):
    blocks int32 [tokens, kv_heads, take] as kv_blocks_select_dev writes it, or
    ascending lists of the caller's own, -1 behind the last entry."""
    dev = Q.device
    on = _on(dev, stream)
    if on is not None:
        with on:
            return attn_blocks_dev(Q, k_pages, v_pages, O, blocks, cu, table, lens, scale, k_scale,
                                   v_scale, None, k_group, v_group)
    q, o = _rows(Q, "Q", dev), _rows(O, "O", dev)
    pg = _pages(k_pages, v_pages, k_scale, v_scale, dev, k_group, v_group)
    sq = _seqs(cu, table, lens, dev)
    at, take = _lists(blocks, q.tokens, pg.H, dev), blocks.shape[2]
    ws, size = _workspace(dev, q.heads, pg.H, q.Dh)  # no scores here
    check(_lib.attnb_attn_blocks_dev(q, pg, o, sq, at, take, _scale(scale), ws.data_ptr(), size,
                                     _raw_stream(dev.index)))


class PagedKVCacheDev:
    """A K/V cache for `batch` sequences in one pool of pages, the ragged
    counterpart of KVCacheDev: ``append`` gives each sequence the pages it needs
    and writes its new tokens (quantising them for dtype torch.float8_e4m3fn,
    torch.int8 or torch.uint8, which is 4 bits, and rotating the keys where it is
    given inv_freq), ``attend`` runs the new tokens' queries over everything held.
    With bounds (True, or their dtype for coded pages; bfloat16 there by default)
    ``attend_blocks`` runs them over a few pages of each sequence that it selects.
    Page numbers and lengths are kept on the host and copied to the device when
    they change, to the same addresses (a captured ``attend`` can be replayed after
    later appends of as many tokens); work is enqueued on ``stream`` (default:
    torch's current one), and calls on different streams are ordered by the caller."""

    def __init__(self, batch: int, H: int, Dh: int, num_pages: int, page_size: int = 64,
                 dtype=None, max_tokens: int | None = None, device=None, bounds=False):
        import torch

        if batch <= 0 or num_pages <= 0:
            raise ValueError("batch and num_pages must be positive")
        if page_size not in (16, 32, 64, 128):
            raise ValueError("page_size must be 16, 32, 64 or 128")
        dtype = torch.bfloat16 if dtype is None else dtype
        device = torch.device("cuda", torch.cuda.current_device()) if device is None \
            else torch.device(device)
        self.batch, self.H, self.Dh, self.page_size = batch, H, Dh, page_size
        if dtype == torch.uint8 and Dh % 32:
            raise ValueError("pages of 4 bits need a head size that is a multiple of 32")
        coded = dtype in (torch.float8_e4m3fn, torch.int8, torch.uint8)
        if not isinstance(bounds, bool) and bounds is not None:
            if not coded and bounds != dtype:
                raise ValueError("bounds of uncoded pages have their type")
            if bounds not in (torch.float32, torch.bfloat16, torch.float16):
                raise ValueError("bounds must be float32, bfloat16 or float16")
        most = num_pages * page_size if max_tokens is None else max_tokens
        width = max(1, -(-most // page_size))
        # (as kv_blocks_bounds_dev would, but behind an append that has run)
        if bounds and (width * page_size >= 1 << 30 or batch * width >= 1 << 31):
            raise ValueError("bounds need max_tokens below 2^30, and fewer than 2^31 pages in the table")
        wide = Dh // 2 if dtype == torch.uint8 else Dh
        self.k_pages, self.v_pages = (torch.empty(num_pages, H, page_size, wide, dtype=dtype,
                                                  device=device) for _ in range(2))
        self.k_scale = self.v_scale = self.k_group = self.v_group = self.bounds = None
        if coded:
            self.k_scale, self.v_scale = (torch.empty(num_pages, H, page_size, device=device)
                                          for _ in range(2))
        if dtype == torch.uint8:
            self.k_group, self.v_group = (torch.empty(num_pages, H, page_size, i4_group_bytes(Dh),
                                                      dtype=torch.uint8, device=device)
                                          for _ in range(2))
        if bounds:
            kind = (torch.bfloat16 if coded else dtype) if bounds is True else bounds
            self.bounds = torch.empty(num_pages, H, 2, Dh, dtype=kind, device=device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._held = [[] for _ in range(batch)]
        self.lengths = [0] * batch
        self.table = torch.zeros(batch, width, dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self._cu = [0] * (batch + 1)  # as in cu
        self.cu = torch.zeros(batch + 1, dtype=torch.int32, device=device)
        self._new = None
        # The calls may name any stream: none runs before these fills, nor before what
        # had the memory until now.
        home = torch.cuda.current_stream(self.table.device)
        home.synchronize()
        self._home = home.cuda_stream

    def append(self, k, v, new, stream=None, inv_freq=None, interleaved=False, q=None,
               q_out=None) -> None:
        """k, v: the new tokens of all sequences, packed [sum(new), H, Dh]; new:
        how many each sequence brings (a list of ints).  inv_freq: k is rotated by
        its tokens' positions on the way, and q into q_out (kv_pages_append_rope_dev)."""
        import torch

        new = [int(n) for n in new]
        if len(new) != self.batch or any(n < 0 for n in new):
            raise ValueError("new must give a count for each sequence")
        if k.shape[0] != sum(new) or v.shape[0] != sum(new):
            raise ValueError("k and v must hold sum(new) tokens")
        want = [-(-(n + m) // self.page_size) for n, m in zip(self.lengths, new)]
        if any(w > self.table.shape[1] for w in want):
            raise ValueError("a sequence would outgrow max_tokens")
        if sum(want) - sum(len(h) for h in self._held) > len(self._free):
            raise ValueError("the pool has too few free pages")
        if inv_freq is None and (q is not None or q_out is not None):
            raise ValueError("q is rotated with inv_freq only")
        on = _on(self.table.device, stream) or contextlib.nullcontext()
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        before = [list(h) for h in self._held], list(self._free), self.lengths, self._cu
        for h, w in zip(self._held, want):
            while len(h) < w:
                h.append(self._free.pop())
        self.lengths = [n + m for n, m in zip(self.lengths, new)]
        self._cu = cu
        with on:
            self._use()
            try:
                self._send(self._held != before[0])
                if inv_freq is None:
                    kv_pages_append_dev(k, v, self.k_pages, self.v_pages, self.cu, self.table,
                                        self.lens, self.k_scale, self.v_scale,
                                        k_group=self.k_group, v_group=self.v_group)
                else:
                    kv_pages_append_rope_dev(k, v, self.k_pages, self.v_pages, self.cu, self.table,
                                             self.lens, inv_freq, interleaved, q, q_out,
                                             self.k_scale, self.v_scale, k_group=self.k_group,
                                             v_group=self.v_group)
                if self.bounds is not None:
                    kv_blocks_bounds_dev(self.k_pages, self.bounds, self.cu, self.table, self.lens,
                                         self.k_scale, self.k_group)
            except Exception:  # a refused append changes nothing
                self._held, self._free, self.lengths, self._cu = before
                self._send(True)
                raise
        self._new = new

    def _use(self) -> None:
        """On a stream other than the constructor's: the memory is in use there
        too, and stays taken until that stream is past it."""
        stream = _torch.cuda.current_stream(self.table.device)
        if stream.cuda_stream == self._home or _torch.cuda.is_current_stream_capturing():
            return
        for t in (self.k_pages, self.v_pages, self.k_scale, self.v_scale, self.k_group,
                  self.v_group, self.bounds, self.table, self.lens, self.cu):
            if t is not None:
                t.record_stream(stream)

    def _send(self, table: bool) -> None:
        """Lengths, offsets and (where it changed) the table to the device."""
        import torch

        if table:
            width = self.table.shape[1]
            self.table.copy_(torch.tensor([h + [0] * (width - len(h)) for h in self._held],
                                          dtype=torch.int32))
        self.lens.copy_(torch.tensor(self.lengths, dtype=torch.int32))
        self.cu.copy_(torch.tensor(self._cu, dtype=torch.int32))

    def attend(self, q, o, causal=True, scale=None, stream=None) -> None:
        """o = attention of q [sum(new), heads, Dh], the queries of the tokens
        appended last, over their sequences."""
        self._check_queries(q)
        with _on(self.table.device, stream) or contextlib.nullcontext():
            self._use()
            attn_paged_dev(q, self.k_pages, self.v_pages, o, self.cu, self.table, self.lens,
                           max(self._new), causal, scale, self.k_scale, self.v_scale,
                           k_group=self.k_group, v_group=self.v_group)

    def _check_queries(self, q) -> None:
        if self._new is None:
            raise ValueError("append first: the queries belong to the tokens appended last")
        if q.shape[0] != sum(self._new):
            raise ValueError("q must hold one row for each token appended last")

    def attend_blocks(self, q, o, take: int, keep_first: int = 1, keep_last: int = 1, scale=None,
                      stream=None):
        """As a causal ``attend``, each token and KV head over `take` pages of its
        sequence: the first keep_first, the last keep_last and those that may hold
        the greatest scores (kv_blocks_select_dev).  Returns the page numbers within the
        sequences, int32 [sum(new), H, take]."""
        if self.bounds is None:
            raise ValueError("attend_blocks needs a cache with bounds")
        self._check_queries(q)
        if take < 1:
            raise ValueError("take must be positive")
        with _on(self.table.device, stream) or contextlib.nullcontext():
            self._use()
            blocks = _torch.empty(q.shape[0], self.H, take, dtype=_torch.int32,
                                  device=self.table.device)
            where = self.cu, self.table, self.lens
            kv_blocks_select_dev(q, self.bounds, blocks, *where, self.page_size, keep_first,
                                 keep_last)
            attn_blocks_dev(q, self.k_pages, self.v_pages, o, blocks, *where, scale, self.k_scale,
                            self.v_scale, k_group=self.k_group, v_group=self.v_group)
        return blocks

    def read(self, b: int, k, v, stream=None) -> None:
        """The tokens of sequence b into k, v [lengths[b], H, Dh]."""
        import torch

        if k.shape[0] != self.lengths[b] or v.shape[0] != self.lengths[b]:
            raise ValueError("k and v must hold the sequence's tokens")
        with _on(self.table.device, stream) or contextlib.nullcontext():
            self._use()
            # The length on the device is that of the last append.
            cu = torch.tensor([0, self.lengths[b]], dtype=torch.int32, device=self.table.device)
            kv_pages_read_dev(self.k_pages, self.v_pages, k, v, cu, self.table[b:b + 1], cu[1:],
                              self.k_scale, self.v_scale, k_group=self.k_group,
                              v_group=self.v_group)

    def truncate(self, b: int, length: int) -> None:
        """Keep the first `length` tokens of sequence b (0 gives all its pages
        back); takes effect with the next append."""
        if not 0 <= length <= self.lengths[b]:
            raise ValueError("length must be in [0, current length]")
        keep = -(-length // self.page_size)
        self._free.extend(reversed(self._held[b][keep:]))
        del self._held[b][keep:]
        self.lengths[b] = length
        self._new = None
