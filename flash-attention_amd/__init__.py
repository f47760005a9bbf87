"""ctypes front end of ``csrc/libflash_attention.so`` (MI355X / gfx950).

The directory name carries a hyphen, so load this package by path (see
``load_package`` in ``__graft_entry__.py``); its import name is
``flash_attention_amd``.

The argtypes below are the ones the reference's caller declares
(benchmarks/compare_impls.py:30-40): four ``POINTER(c_uint16)``, five ``c_int``,
``c_void_p`` stream, ``POINTER(c_float)`` elapsed.  There is no CPU fallback:
if the shared library is missing or a call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes as ct
import functools
import os
from typing import NamedTuple

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "csrc", "libflash_attention.so")

HalfPtr = ct.POINTER(ct.c_uint16)
FloatPtr = ct.POINTER(ct.c_float)

EXPORTED_SYMBOLS = (
    "run_tensor_flash_attention",
    "run_tensor_flash_attention_host_half",
    "fa_forward",
    "fa_forward_host_half",
    "fa_forward_host_half_sharded",
    "fa_forward_noalloc",
    "fa_forward_block",
    "fa_forward_general",
    "fa_forward_varlen",
    "fa_forward_block_general",
    "fa_forward_general_host_half",
    "run_naive_attention_host_half",
    "run_cuda_cores_flash_attention_host_half",
    "fa_init_half",
    "fa_device_info",
    "fa_last_error",
    "fa_version",
    "fa_kernel_name",
    "fa_kernel_name_general",
    "fa_kernel_name_general_bh",
    "fa_kernel_name_block_general",
    "fa_split_ways",
    "fa_split_ways_general",
    "fa_set_reserved_cus",
    "fa_get_reserved_cus",
    "fa_debug_reload_env",
    "fa_cache_plan",
    "fa_cache_write",
    "fa_forward_shared_prefix",
    "fa_shared_prefix_workspace",
)

_lib = None


class FlashAttentionError(RuntimeError):
    pass


class _PagedCacheStruct(ct.Structure):  # fa_paged_cache
    _fields_ = [("k", ct.c_void_p), ("v", ct.c_void_p), ("k_strides", ct.c_int64 * 3), ("v_strides", ct.c_int64 * 3),
                ("n_pages", ct.c_int), ("page_size", ct.c_int), ("heads", ct.c_int), ("head_dim", ct.c_int)]


def lib() -> ct.CDLL:
    """Load the HIP library; fail loudly if it has not been built."""
    global _lib
    if _lib is None:
        _lib = bind(LIB_PATH)
    return _lib


def bind(path: str) -> ct.CDLL:
    """dlopen a build of the library and declare its entry points' argument types."""
    if not os.path.exists(path):
        raise FlashAttentionError(
            f"{path} not found: build it with flash-attention_amd/csrc/shared_compile.sh "
            "(there is no CPU fallback)"
        )
    # PyTorch ships a HIP runtime of its own (same SONAME as /opt/rocm's).  Two HIP runtimes in
    # one process do not work, so when torch is installed its copy must be mapped first; the
    # dynamic linker then binds this library to that copy as well.
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    L = ct.CDLL(path)
    sig = [HalfPtr, HalfPtr, HalfPtr, HalfPtr] + [ct.c_int] * 5 + [ct.c_void_p, FloatPtr]
    for name in ("run_tensor_flash_attention", "run_tensor_flash_attention_host_half"):
        getattr(L, name).argtypes = sig
        getattr(L, name).restype = None
    for name in ("fa_forward", "fa_forward_host_half"):
        getattr(L, name).argtypes = sig
        getattr(L, name).restype = ct.c_int
    L.fa_forward_host_half_sharded.argtypes = sig[:-2] + [ct.POINTER(ct.c_int), ct.c_int, FloatPtr]
    L.fa_forward_host_half_sharded.restype = ct.c_int
    L.fa_forward_noalloc.argtypes = sig[:-1]
    L.fa_forward_noalloc.restype = ct.c_int
    L.fa_forward_block.argtypes = (
        [HalfPtr, HalfPtr, HalfPtr, HalfPtr, FloatPtr, FloatPtr, FloatPtr] + [ct.c_int] * 6 + [ct.c_void_p]
    )
    L.fa_forward_block.restype = ct.c_int
    L.fa_forward_general.argtypes = [HalfPtr, HalfPtr, HalfPtr, HalfPtr] + [ct.c_int] * 6 + [ct.c_void_p, FloatPtr]
    L.fa_forward_general.restype = ct.c_int
    L.fa_forward_varlen.argtypes = ([HalfPtr, HalfPtr, HalfPtr, HalfPtr] + [ct.c_int] * 6 +
                                    [ct.POINTER(ct.c_int), ct.POINTER(ct.c_int), ct.c_void_p, FloatPtr])
    L.fa_forward_varlen.restype = ct.c_int
    L.fa_forward_block_general.argtypes = (
        [HalfPtr, HalfPtr, HalfPtr, HalfPtr, FloatPtr, FloatPtr, FloatPtr] + [ct.c_int] * 9 + [ct.c_void_p]
    )
    L.fa_forward_block_general.restype = ct.c_int
    L.fa_forward_general_host_half.argtypes = L.fa_forward_general.argtypes
    L.fa_forward_general_host_half.restype = ct.c_int
    # the sibling libraries' symbols, with the argtypes the reference's caller declares
    # (benchmarks/compare_impls.py:42-58)
    L.run_naive_attention_host_half.argtypes = [HalfPtr] * 4 + [ct.c_int] * 5 + [ct.c_void_p, FloatPtr]
    L.run_naive_attention_host_half.restype = None
    L.run_cuda_cores_flash_attention_host_half.argtypes = [HalfPtr] * 4 + [ct.c_int] * 6 + [ct.c_void_p, FloatPtr]
    L.run_cuda_cores_flash_attention_host_half.restype = None
    L.fa_init_half.argtypes = [HalfPtr, ct.c_size_t, ct.c_ulonglong, ct.c_void_p]
    L.fa_init_half.restype = ct.c_int
    L.fa_device_info.argtypes = [ct.POINTER(ct.c_int), ct.POINTER(ct.c_int), ct.POINTER(ct.c_double)]
    L.fa_device_info.restype = ct.c_int
    L.fa_last_error.argtypes = []
    L.fa_last_error.restype = ct.c_char_p
    L.fa_version.argtypes = []
    L.fa_version.restype = ct.c_char_p
    L.fa_kernel_name.argtypes = [ct.c_int, ct.c_int]
    L.fa_kernel_name.restype = ct.c_char_p
    L.fa_kernel_name_general.argtypes = [ct.c_int, ct.c_int, ct.c_int, ct.c_int]
    L.fa_kernel_name_general.restype = ct.c_char_p
    L.fa_kernel_name_general_bh.argtypes = [ct.c_int] * 5
    L.fa_kernel_name_general_bh.restype = ct.c_char_p
    L.fa_kernel_name_block_general.argtypes = [ct.c_int] * 6
    L.fa_kernel_name_block_general.restype = ct.c_char_p
    L.fa_split_ways.argtypes = [ct.c_int] * 3
    L.fa_split_ways.restype = ct.c_int
    L.fa_split_ways_general.argtypes = [ct.c_int] * 5
    L.fa_split_ways_general.restype = ct.c_int
    L.fa_set_reserved_cus.argtypes = [ct.c_int]
    L.fa_set_reserved_cus.restype = ct.c_int
    L.fa_get_reserved_cus.argtypes = []
    L.fa_get_reserved_cus.restype = ct.c_int
    L.fa_debug_reload_env.argtypes = []
    L.fa_debug_reload_env.restype = None
    vp, i, i64 = ct.c_void_p, ct.c_int, ct.c_int64
    L.fa_cache_plan.argtypes = [vp, vp, vp, i64, vp, vp, vp, vp, vp, vp, i, i, i, i, i, vp, FloatPtr]
    L.fa_cache_plan.restype = i
    L.fa_cache_write.argtypes = [vp, vp, i64, i64, i64, i64, ct.POINTER(_PagedCacheStruct), vp, i, vp, FloatPtr]
    L.fa_cache_write.restype = i
    L.fa_forward_shared_prefix.argtypes = [vp, i64, i64, vp, i64, i64, ct.POINTER(_PagedCacheStruct), vp, i, vp, i64, i, vp, vp,
                                           i, i, i, i, i, ct.c_float, i, vp, ct.c_size_t, vp, FloatPtr]
    L.fa_forward_shared_prefix.restype = i
    L.fa_shared_prefix_workspace.argtypes = [i] * 7
    L.fa_shared_prefix_workspace.restype = ct.c_size_t
    return L


def _check(rc: int) -> None:
    if rc != 0:
        raise FlashAttentionError(f"libflash_attention error {rc}: {lib().fa_last_error().decode()}")


def _np_half_ptr(a: np.ndarray):
    if a.dtype != np.float16 or not a.flags["C_CONTIGUOUS"]:
        raise ValueError("expected a C-contiguous float16 array")
    return a.ctypes.data_as(HalfPtr)


def _dev_half_ptr(t):
    return ct.cast(ct.c_void_p(t.data_ptr()), HalfPtr)


def _dev_float_ptr(t):
    return ct.cast(ct.c_void_p(t.data_ptr()), FloatPtr)


def _stream_handle(stream) -> ct.c_void_p:
    if stream is None:
        return ct.c_void_p(0)
    if isinstance(stream, int):
        return ct.c_void_p(stream)
    return ct.c_void_p(stream.cuda_stream)  # torch.cuda.Stream


def attention_host_half(Q: np.ndarray, K: np.ndarray, V: np.ndarray, tile: int = 64, want_ms: bool = True):
    """Host-pointer path (``run_tensor_flash_attention_host_half``, wrapper.cu:9-35).

    fp16 NumPy arrays of shape [B,H,L,D] in, (fp16 O, kernel-only ms) out."""
    B, H, L, D = Q.shape
    if K.shape != Q.shape or V.shape != Q.shape:
        raise ValueError("Q, K, V must share one [B,H,L,D] shape")
    O = np.empty_like(Q)
    ms = ct.c_float(0.0)
    rc = lib().fa_forward_host_half(
        _np_half_ptr(Q), _np_half_ptr(K), _np_half_ptr(V), _np_half_ptr(O), B, H, L, D, tile, None,
        ct.byref(ms) if want_ms else None,
    )
    _check(rc)
    return O, float(ms.value)


def attention_host_half_sharded(Q: np.ndarray, K: np.ndarray, V: np.ndarray, devices=None, tile: int = 64):
    """The host-pointer path over several GPUs of this node from one process (``fa_forward_host_half_sharded``):
    the flattened B*H axis in contiguous ranges, one per entry of ``devices`` (a list of GPU indices, an int n for
    GPUs 0..n-1, or None for every visible GPU).  Returns (fp16 O, [kernel-only ms of each range])."""
    B, H, L, D = Q.shape
    if K.shape != Q.shape or V.shape != Q.shape:
        raise ValueError("Q, K, V must share one [B,H,L,D] shape")
    O = np.empty_like(Q)
    if devices is None:
        dev_arr, n = None, 0
        n_out = max(1, device_count())
    elif isinstance(devices, int):
        dev_arr, n = None, devices
        n_out = max(1, devices)
    else:
        n = n_out = len(devices)
        dev_arr = (ct.c_int * max(1, n))(*devices)
    ms = (ct.c_float * n_out)()
    rc = lib().fa_forward_host_half_sharded(
        _np_half_ptr(Q), _np_half_ptr(K), _np_half_ptr(V), _np_half_ptr(O), B, H, L, D, tile, dev_arr, n, ms)
    _check(rc)
    return O, [float(x) for x in ms]


def device_count() -> int:
    """GPUs visible to this process (asks torch, which this front end maps first)."""
    import torch

    return torch.cuda.device_count()


def attention(q, k, v, out=None, tile: int = 64, stream=None, timed: bool = False):
    """Device-pointer path (``run_tensor_flash_attention``, wrapper.cu:39-203) on torch
    tensors resident on the GPU.  q,k,v: contiguous fp16 [B,H,L,D].  Returns ``out`` (and
    the kernel-only milliseconds when ``timed``)."""
    import torch

    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise FlashAttentionError("attention() needs GPU tensors; there is no CPU fallback")
    for t in (q, k, v):
        if t.dtype != torch.float16 or not t.is_contiguous():
            raise ValueError("q, k, v must be contiguous float16 tensors")
    B, H, L, D = q.shape
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError("q, k, v must share one [B,H,L,D] shape")
    if out is None:
        out = torch.empty_like(q)
    if stream is None:
        stream = torch.cuda.current_stream(q.device)
    ms = ct.c_float(0.0)
    with torch.cuda.device(q.device):
        rc = lib().fa_forward(
            _dev_half_ptr(q), _dev_half_ptr(k), _dev_half_ptr(v), _dev_half_ptr(out), B, H, L, D, tile,
            _stream_handle(stream), ct.byref(ms) if timed else None,
        )
    _check(rc)
    return (out, float(ms.value)) if timed else out


FLAG_CAUSAL = 1  # FA_FLAG_CAUSAL


def attention_general_host_half(Q: np.ndarray, K: np.ndarray, V: np.ndarray, causal: bool = False):
    """``fa_forward_general_host_half``: fp16 NumPy arrays Q [B,H,Lq,D], K/V [B,H,Lk,D] in, (fp16 O,
    kernel-only ms) out."""
    B, H, Lq, D = Q.shape
    Lk = K.shape[2]
    if K.shape != (B, H, Lk, D) or V.shape != K.shape:
        raise ValueError("K, V must be [B,H,Lk,D] with Q's B, H, D")
    O = np.empty_like(Q)
    ms = ct.c_float(0.0)
    rc = lib().fa_forward_general_host_half(
        _np_half_ptr(Q), _np_half_ptr(K), _np_half_ptr(V), _np_half_ptr(O), B, H, Lq, Lk, D,
        FLAG_CAUSAL if causal else 0, None, ct.byref(ms),
    )
    _check(rc)
    return O, float(ms.value)


def attention_general(q, k, v, causal: bool = False, out=None, stream=None, timed: bool = False):
    """``fa_forward_general``: q [B,H,Lq,D] against k, v [B,H,Lk,D], any Lq, Lk >= 1; ``causal``
    applies the mask of the reference's CPU baseline (testing.cu:74-77; needs Lq == Lk).
    Contiguous fp16 GPU tensors.  Returns ``out`` (and the kernel-only milliseconds when ``timed``)."""
    import torch

    for t in (q, k, v):
        if not t.is_cuda or t.dtype != torch.float16 or not t.is_contiguous():
            raise ValueError("q, k, v must be contiguous float16 GPU tensors; there is no CPU fallback")
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    if k.shape != (B, H, Lk, D) or v.shape != k.shape:
        raise ValueError("k, v must be [B,H,Lk,D] with q's B, H, D")
    if out is None:
        out = torch.empty_like(q)
    if stream is None:
        stream = torch.cuda.current_stream(q.device)
    ms = ct.c_float(0.0)
    with torch.cuda.device(q.device):
        rc = lib().fa_forward_general(
            _dev_half_ptr(q), _dev_half_ptr(k), _dev_half_ptr(v), _dev_half_ptr(out), B, H, Lq, Lk, D,
            FLAG_CAUSAL if causal else 0, _stream_handle(stream), ct.byref(ms) if timed else None,
        )
    _check(rc)
    return (out, float(ms.value)) if timed else out


def attention_varlen(q, k, v, q_len=None, k_len=None, causal: bool = False, out=None, stream=None, timed: bool = False):
    """``fa_forward_varlen``: padded batches.  q [B,H,Lq,D], k, v [B,H,Lk,D] contiguous fp16 GPU tensors; ``q_len`` /
    ``k_len`` int32 GPU tensors of B valid lengths (or None).  Rows of ``out`` from ``q_len[b]`` on are left as
    they are.  Returns ``out`` (and the kernel-only milliseconds when ``timed``)."""
    import torch

    for t in (q, k, v):
        if not t.is_cuda or t.dtype != torch.float16 or not t.is_contiguous():
            raise ValueError("q, k, v must be contiguous float16 GPU tensors; there is no CPU fallback")
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    if k.shape != (B, H, Lk, D) or v.shape != k.shape:
        raise ValueError("k, v must be [B,H,Lk,D] with q's B, H, D")
    for t in (q_len, k_len):
        if t is not None and (not t.is_cuda or t.dtype != torch.int32 or not t.is_contiguous() or t.numel() != B):
            raise ValueError("q_len / k_len must be contiguous int32 GPU tensors of B entries")
    if out is None:
        out = torch.zeros_like(q)
    if stream is None:
        stream = torch.cuda.current_stream(q.device)
    ip = lambda t: ct.cast(ct.c_void_p(t.data_ptr()), ct.POINTER(ct.c_int)) if t is not None else None
    ms = ct.c_float(0.0)
    with torch.cuda.device(q.device):
        rc = lib().fa_forward_varlen(
            _dev_half_ptr(q), _dev_half_ptr(k), _dev_half_ptr(v), _dev_half_ptr(out), B, H, Lq, Lk, D,
            FLAG_CAUSAL if causal else 0, ip(q_len), ip(k_len), _stream_handle(stream), ct.byref(ms) if timed else None,
        )
    _check(rc)
    return (out, float(ms.value)) if timed else out


class BlockState:
    """Carried (o_acc, row_max, row_sum) of the blockwise forward, on the GPU."""

    def __init__(self, BH: int, Lq: int, D: int, device):
        import torch

        self.o_acc = torch.empty((BH, Lq, D), dtype=torch.float32, device=device)
        self.row_max = torch.empty((BH, Lq), dtype=torch.float32, device=device)
        self.row_sum = torch.empty((BH, Lq), dtype=torch.float32, device=device)
        self.first = True


def attention_block(q, k_blk, v_blk, state: BlockState, last: bool, out=None, stream=None):
    """One step of the blockwise forward (``fa_forward_block``): fold the K/V block into
    ``state``; on the ``last`` step write the normalised fp16 output into ``out``."""
    import torch

    B, H, Lq, D = q.shape
    Lk = k_blk.shape[2]
    if k_blk.shape != (B, H, Lk, D) or v_blk.shape != k_blk.shape:
        raise ValueError("k_blk / v_blk must be [B,H,Lk,D]")
    for t in (q, k_blk, v_blk):
        if not t.is_cuda or t.dtype != torch.float16 or not t.is_contiguous():
            raise ValueError("q, k_blk, v_blk must be contiguous float16 GPU tensors")
    if last and out is None:
        out = torch.empty_like(q)
    if stream is None:
        stream = torch.cuda.current_stream(q.device)
    with torch.cuda.device(q.device):
        rc = lib().fa_forward_block(
            _dev_half_ptr(q), _dev_half_ptr(k_blk), _dev_half_ptr(v_blk),
            _dev_half_ptr(out) if out is not None else None,
            _dev_float_ptr(state.o_acc), _dev_float_ptr(state.row_max), _dev_float_ptr(state.row_sum),
            B * H, Lq, Lk, D, int(state.first), int(last), _stream_handle(stream),
        )
    _check(rc)
    state.first = False
    return out


def attention_block_general(q, k_blk, v_blk, state: BlockState, last: bool, causal: bool = False, q_pos0: int = 0,
                            k_pos0: int = 0, out=None, stream=None):
    """One step of the blockwise forward through ``fa_forward_block_general``: any Lq, Lk >= 1, D of
    64, 128 or 256; with ``causal`` key ``k_pos0 + j`` is visible to query ``q_pos0 + i`` iff it is not
    ahead of it, so blocks may be folded in any order."""
    import torch

    B, H, Lq, D = q.shape
    Lk = k_blk.shape[2]
    if k_blk.shape != (B, H, Lk, D) or v_blk.shape != k_blk.shape:
        raise ValueError("k_blk / v_blk must be [B,H,Lk,D]")
    for t in (q, k_blk, v_blk):
        if not t.is_cuda or t.dtype != torch.float16 or not t.is_contiguous():
            raise ValueError("q, k_blk, v_blk must be contiguous float16 GPU tensors")
    if last and out is None:
        out = torch.empty_like(q)
    if stream is None:
        stream = torch.cuda.current_stream(q.device)
    with torch.cuda.device(q.device):
        rc = lib().fa_forward_block_general(
            _dev_half_ptr(q), _dev_half_ptr(k_blk), _dev_half_ptr(v_blk),
            _dev_half_ptr(out) if out is not None else None,
            _dev_float_ptr(state.o_acc), _dev_float_ptr(state.row_max), _dev_float_ptr(state.row_sum),
            B * H, Lq, Lk, D, FLAG_CAUSAL if causal else 0, int(q_pos0), int(k_pos0), int(state.first), int(last),
            _stream_handle(stream),
        )
    _check(rc)
    state.first = False
    return out


class PagedCache:
    """A paged K/V cache (``fa_paged_cache``): ``k`` and ``v`` are float16 or bfloat16 GPU tensors of one shape
    [n_pages, Hkv, page_size, D], with any strides of the first three axes (token-major pages are a permuted view, K and V
    in one pool are slices of it).  page_size a power of two from 16 to 65536, D of 64, 128 or 256.  The tensors are held, not copied."""

    def __init__(self, k, v):
        import torch

        for t in (k, v):
            if not t.is_cuda or t.dtype not in (torch.float16, torch.bfloat16) or t.dim() != 4 or t.stride(3) != 1:
                raise ValueError("k, v must be float16 or bfloat16 GPU tensors [n_pages, Hkv, page_size, D] whose rows are contiguous")
        if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise ValueError("k and v must share shape, dtype and device")
        self.k, self.v, self.dtype, self.device, self.device_index = k, v, k.dtype, k.device, k.device.index
        self.n_pages, self.heads, self.page_size, self.head_dim = k.shape
        # (an axis of one may have any stride, also one that the library would refuse)
        ks, vs = ([D if n == 1 else s for n, s in zip(k.shape[:3], t.stride())] for t, D in ((k, k.shape[3]), (v, k.shape[3])))
        self.c = _PagedCacheStruct(k.data_ptr(), v.data_ptr(), (ct.c_int64 * 3)(*ks), (ct.c_int64 * 3)(*vs),
                                   self.n_pages, self.page_size, self.heads, self.head_dim)
        self.ref = ct.byref(self.c)
        self.dtype_code = 0 if k.dtype == torch.float16 else 1


class CachePlan(NamedTuple):
    """Tables of one serving step, int32 GPU tensors: ``q_start`` [B + 1], ``k_len`` [B], ``slots`` [max_tokens], ``counts``
    [2] (free pages left, requests refused).  ``k_len`` and ``counts[:1]`` are the next step's ``k_len`` and ``free_count``;
    a program keeps two of these and alternates."""

    q_start: object
    k_len: object
    slots: object
    counts: object


def make_cache_plan(B: int, max_tokens: int, device) -> CachePlan:
    """A ``CachePlan``'s tensors for ``B`` requests and up to ``max_tokens`` new tokens a step."""
    import torch

    return CachePlan(*(torch.empty(n, dtype=torch.int32, device=device) for n in (B + 1, B, max_tokens, 2)))


def _raw_stream(torch, stream, index: int) -> int:
    """Handle of ``stream`` (a torch stream, a handle, or None: the current one of GPU ``index``)."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(index)
    return stream if isinstance(stream, int) else stream.cuda_stream


def _allocating_for(torch, stream, device):
    """What a call on ``stream`` allocates (and zeroes) belongs to that stream."""
    import contextlib

    if stream is None:
        return contextlib.nullcontext()
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else stream)


def _run_on(torch, index: int, call, *args, timed: bool = False) -> float:
    """Calls a library function, its elapsed_ms argument last, with GPU ``index`` current; raises on its errors."""
    ms = ct.c_float(0.0) if timed else None
    if torch._C._cuda_getDevice() == index:
        rc = call(*args, ct.byref(ms) if timed else None)
    else:
        with torch.cuda.device(index):
            rc = call(*args, ct.byref(ms) if timed else None)
    if rc:
        _check(rc)
    return ms.value if timed else 0.0


def _int_tensor(torch, t, name: str, index: int, n: int) -> int:
    """Address of a contiguous int32 tensor of ``n`` entries on GPU ``index``."""
    if t.dtype is not torch.int32 or t.get_device() != index or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} entries on the call's GPU")
    return t.data_ptr()


def _table(torch, t, name: str, index: int, rows: int):
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or t.dtype is not torch.int32 or t.get_device() != index or shape[0] != rows or (shape[1] > 1 and stride[1] != 1):
        raise ValueError(f"{name} must be an int32 tensor [{rows}, width] with contiguous rows on the call's GPU")
    return t.data_ptr(), max(stride[0], shape[1]) if rows == 1 else stride[0], shape[1]


def cache_plan(k_len, n_new, block_table, free_pages, free_count, page_size: int, max_tokens: int = None, out: CachePlan = None,
               stream=None, timed: bool = False):
    """``fa_cache_plan``: block table, slot map and lengths of one serving step, on the GPU.  ``k_len``, ``n_new`` [B] keys
    each request holds and adds (negative: drops from its end); ``block_table`` [B, width] and the stack ``free_pages`` are
    updated in place, ``free_count`` [1] counts its pages.  All int32 GPU tensors.  Returns a ``CachePlan`` (``out``, or a
    new one for ``max_tokens`` tokens); a refused request (``n_new`` > 0) keeps its ``k_len``, and attention's output
    means nothing on its rows, which ``q_start`` counts."""
    import torch

    B, dev = k_len.numel(), k_len.get_device()
    if dev < 0:
        raise FlashAttentionError("cache_plan() needs GPU tensors; there is no CPU fallback")
    if out is None:
        if max_tokens is None:
            raise ValueError("cache_plan() needs max_tokens or out")
        with _allocating_for(torch, stream, k_len.device):
            out = make_cache_plan(B, max_tokens, k_len.device)
    elif max_tokens is not None and max_tokens != out.slots.numel():
        raise ValueError("max_tokens must be the size of out.slots")
    table, stride, width = _table(torch, block_table, "block_table", dev, B)
    max_tokens, cap = out.slots.numel(), free_pages.numel()
    ms = _run_on(
        torch, dev, lib().fa_cache_plan, _int_tensor(torch, k_len, "k_len", dev, B), _int_tensor(torch, n_new, "n_new", dev, B), table, stride,
        _int_tensor(torch, free_pages, "free_pages", dev, cap), _int_tensor(torch, free_count, "free_count", dev, 1),
        _int_tensor(torch, out.q_start, "out.q_start", dev, B + 1), _int_tensor(torch, out.k_len, "out.k_len", dev, B),
        _int_tensor(torch, out.slots, "out.slots", dev, max_tokens), _int_tensor(torch, out.counts, "out.counts", dev, 2),
        B, width, page_size, cap, max_tokens, _raw_stream(torch, stream, dev), timed=timed)
    return (out, ms) if timed else out


def _token_rows(t, name: str, heads, cache: "PagedCache"):
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or t.dtype is not cache.dtype or t.get_device() != cache.device_index or shape[2] != cache.head_dim or \
            (heads is not None and shape[1] != heads) or (stride[2] != 1 and t.numel()):
        raise ValueError(f"{name} must be [T, heads, {cache.head_dim}] with contiguous rows, of the cache's dtype and GPU")
    D = shape[2]  # (an axis of one may have any stride)
    return t.data_ptr(), stride[0] if shape[0] > 1 else D, stride[1] if shape[1] > 1 else D


def cache_write(k, v, cache: PagedCache, slots, stream=None, timed: bool = False):
    """``fa_cache_write``: row t of ``k`` and ``v`` [T, Hkv, D] (any token and head strides) goes into slot ``slots[t]`` of the
    cache (int32, a ``CachePlan``'s); negative slots and slots on no page of the cache are skipped."""
    import torch

    T, dev = k.shape[0], cache.device_index
    if v.shape != k.shape:
        raise ValueError("k and v must share one [T, Hkv, D] shape")
    n = slots.numel()
    if n < T:
        raise ValueError("slots must name a slot for every token")
    kp, kt, kh = _token_rows(k, "k", cache.heads, cache)
    vp, vt, vh = _token_rows(v, "v", cache.heads, cache)
    ms = _run_on(torch, dev, lib().fa_cache_write, kp, vp, kt, kh, vt, vh, cache.ref, _int_tensor(torch, slots, "slots", dev, n), T,
                 _raw_stream(torch, stream, dev), timed=timed)
    return ms if timed else None


@functools.lru_cache(maxsize=4096)
def _shared_prefix_workspace(device: int, *sizes) -> int:
    import torch

    with torch.cuda.device(device):
        return lib().fa_shared_prefix_workspace(*sizes)


def attention_shared_prefix(q, cache: PagedCache, q_start, k_len, block_table, prefix_table=None, prefix_len: int = 0,
                            causal: bool = True, scale: float = None, max_k_len: int = None, out=None, stream=None,
                            timed: bool = False):
    """``fa_forward_shared_prefix``: attention of a batch of requests behind one shared prefix.  ``q`` [T, Hq, D] packed new
    tokens (any token and head strides; Hq a multiple of the cache's heads), request b's being rows ``q_start[b]`` to
    ``q_start[b + 1]``; they see the ``prefix_len`` keys on the pages of ``prefix_table`` and the request's own ``k_len[b]``
    keys on the pages of ``block_table[b]``, the new tokens' own among them (already written), with ``causal`` only up to their
    own.  ``max_k_len``: a bound on ``k_len`` that the workspace is made for (default: what the table names).  Rows of
    ``out`` that belong to no request are left as they are (0 in a new one).  Returns ``out`` (and the kernel-only
    milliseconds when ``timed``)."""
    import torch

    dev = cache.device_index
    qp, qt, qh = _token_rows(q, "q", None, cache)
    T, Hq, D = q.shape
    if out is None:
        with _allocating_for(torch, stream, cache.device):
            out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise ValueError("out must have q's shape")
    op, ot, oh = _token_rows(out, "out", Hq, cache)
    B = k_len.numel()
    if Hq % cache.heads:
        raise ValueError("q's heads must be a multiple of the cache's")
    table, stride, width = _table(torch, block_table, "block_table", dev, B)
    if prefix_len:
        if prefix_table is None or prefix_table.numel() * cache.page_size < prefix_len:
            raise ValueError("prefix_table must name the pages of prefix_len keys")
        prefix = _int_tensor(torch, prefix_table, "prefix_table", dev, prefix_table.numel())
    else:
        prefix = None
    room = width * cache.page_size
    max_k = room if max_k_len is None else max(0, min(max_k_len, room))
    handle = _raw_stream(torch, stream, dev)
    n = _shared_prefix_workspace(dev, T, B, Hq, cache.heads, D, prefix_len, max_k)
    if stream is None:
        workspace = torch.empty(n, dtype=torch.uint8, device=cache.device)
    else:
        with _allocating_for(torch, stream, cache.device):
            workspace = torch.empty(n, dtype=torch.uint8, device=cache.device)
    ms = _run_on(
        torch, dev, lib().fa_forward_shared_prefix, qp, qt, qh, op, ot, oh, cache.ref, prefix, prefix_len, table, stride, width,
        _int_tensor(torch, q_start, "q_start", dev, B + 1), _int_tensor(torch, k_len, "k_len", dev, B), T, B, Hq, cache.dtype_code,
        FLAG_CAUSAL if causal else 0, D ** -0.5 if scale is None else scale, max_k, workspace.data_ptr(), n, handle, timed=timed)
    return (out, ms) if timed else out


def init_half(t, seed: int, stream=None) -> None:
    """Fill a GPU fp16 tensor with the throughput driver's pattern
    (benchmark_tensor_flash_attention.cu:34-41)."""
    import torch

    if not t.is_cuda or t.dtype != torch.float16 or not t.is_contiguous():
        raise ValueError("init_half needs a contiguous float16 GPU tensor")
    if stream is None:
        stream = torch.cuda.current_stream(t.device)
    with torch.cuda.device(t.device):
        _check(lib().fa_init_half(_dev_half_ptr(t), t.numel(), seed, _stream_handle(stream)))


def set_reserved_cus(k: int) -> None:
    """``fa_set_reserved_cus``: persistent launches leave ``k`` compute units free for other streams' kernels
    (the transport kernels of a ring's send/recv); 0 restores one workgroup per unit."""
    _check(lib().fa_set_reserved_cus(int(k)))


def reload_env() -> None:
    """Re-read the FA_* environment switches (they are otherwise read once per process).  For tests and A/B runs."""
    lib().fa_debug_reload_env()


def device_info() -> dict:
    cus, khz, peak = ct.c_int(0), ct.c_int(0), ct.c_double(0.0)
    _check(lib().fa_device_info(ct.byref(cus), ct.byref(khz), ct.byref(peak)))
    return {"compute_units": cus.value, "clock_khz": khz.value, "fp16_dense_peak_flops": peak.value}


def mae_mre(ref32: np.ndarray, test16: np.ndarray):
    """Mean absolute error and mean relative error over the reference's non-zero entries, the two figures
    benchmarks/compare_impls.py:66-74 prints."""
    a = np.asarray(ref32, dtype=np.float32).reshape(-1)
    d = np.abs(a - np.asarray(test16).astype(np.float32).reshape(-1))
    nz = a != 0
    return float(d.mean()), (float((d[nz] / np.abs(a[nz])).mean()) if nz.any() else float("nan"))


def attention_flops(B: int, H: int, L: int, D: int) -> float:
    """4*B*H*L^2*D (benchmark_tensor_flash_attention.cu:218)."""
    return 4.0 * B * H * float(L) * float(L) * D
