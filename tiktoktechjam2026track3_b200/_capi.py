"""ctypes binding of libb200tx.so (C-ABI declared in include/b200tx.h).

Follows the reference's binding conventions: the library is loaded lazily, once, under a
lock (transformer_benchmark/native_softmax_bf16.py:16-17, 129-160), every foreign function has
explicit argtypes/restype, and a non-zero status becomes a RuntimeError carrying the library's
own message (transformer_benchmark/cublaslt_linear.py:63-145).

There is no fallback: if the library is missing or the device is not an sm_100 GPU, the call
raises. The wrappers here take torch tensors only to read their pointers, shapes and the current
CUDA stream; all arithmetic happens in the CUDA kernels.
"""

from __future__ import annotations

import ctypes
import struct
import threading
from pathlib import Path
from typing import Optional, Tuple

import torch

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libb200tx.so"

EPI_BIAS = 0
EPI_BIAS_GELU = 1
EPI_RESIDUAL = 2
EPI_RESIDUAL_ZERO = 3
EPI_STORE_F32 = 4
TILE_PAIR = 0x10000

REASON_BAD_INDEX = 3  # of the status word: a position, length or page number lay outside its table
CACHE_BF16 = 0
CACHE_E4M3 = 1

# Every symbol include/b200tx.h declares, with its ctypes signature.
_i64 = ctypes.c_int64
_vp = ctypes.c_void_p


class KVCacheDesc(ctypes.Structure):
    """b2_kv_cache: where a paged cache's keys, values and scales lie."""

    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("pages", _i64), ("kv_heads", _i64),
                ("page_size", _i64), ("head_dim", _i64), ("page_stride", _i64), ("head_stride", _i64),
                ("dtype", ctypes.c_int)]
    device = 0  # index of the GPU that holds them (not part of the C struct)


# The argument structs of the serving entry points: every member is 8 bytes wide, pointers as integers.
ROTARY_ARGS = struct.Struct("13q")
CACHE_APPEND_ARGS = struct.Struct("23q")
CACHE_ATTENTION_ARGS = struct.Struct("11qd4q")
WINDOW_ATTENTION_ARGS = struct.Struct("14qd2q")
SIGNATURES = {
    "b2_abi_version": (ctypes.c_int, []),
    "b2_last_error": (ctypes.c_char_p, []),
    "b2_device_status": (ctypes.c_int, [ctypes.POINTER(ctypes.c_uint32), ctypes.c_int]),
    "b2_device_status_async": (ctypes.c_int, [_vp, _vp]),
    "b2_index_status_async": (ctypes.c_int, [_vp, _vp]),
    "b2_set_wait_limit": (ctypes.c_int, [ctypes.c_uint64]),
    "b2_mask_lengths": (ctypes.c_int, [_vp, _i64, _i64, _vp, _vp, _vp, _vp]),
    "b2_test_set_fault": (ctypes.c_int, [ctypes.c_int]),
    "b2_layernorm_fwd": (
        ctypes.c_int,
        [_vp, ctypes.c_int, _vp, _vp, ctypes.c_float, _vp, _vp, _vp, _i64, _i64, _vp],
    ),
    "b2_add_layernorm_fwd": (
        ctypes.c_int,
        [_vp, _vp, _vp, _vp, ctypes.c_int, _vp, _vp, ctypes.c_float, _vp, _i64, _i64, _vp],
    ),
    "b2_linear_fwd": (
        ctypes.c_int,
        [_vp, _vp, _vp, _i64, _i64, _i64, ctypes.c_int, _vp, _i64, _vp, ctypes.c_int, _vp],
    ),
    "b2_linear_ln_fwd": (
        ctypes.c_int,
        [_vp, _vp, _vp, _i64, _i64, _i64, ctypes.c_int, _vp, _vp, _vp, _vp, ctypes.c_float, _vp, _vp],
    ),
    "b2_linear_ln_plan": (
        ctypes.c_int,
        [_i64, _i64, _i64, ctypes.c_int, ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int),
         ctypes.POINTER(ctypes.c_int)],
    ),
    "b2_attention_fwd": (
        ctypes.c_int,
        [_vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _vp, ctypes.c_int, ctypes.c_float, _vp, _i64, _vp],
    ),
    "b2_attention_rows_fwd": (
        ctypes.c_int,
        [_vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _vp, ctypes.c_int, ctypes.c_float, ctypes.POINTER(_i64),
         ctypes.c_int, _vp, _i64, _vp],
    ),
    "b2_peer_barrier": (ctypes.c_int, [ctypes.POINTER(_vp), ctypes.c_int, ctypes.c_int, ctypes.c_int, _vp]),
    "b2_linear_rs_fwd": (
        ctypes.c_int,
        [_vp, _vp, _vp, _i64, _i64, _i64, ctypes.c_int, ctypes.POINTER(_vp), ctypes.c_int, ctypes.c_int, _i64, _i64,
         _vp, ctypes.c_int, _vp],
    ),
    "b2_linear_bcast_fwd": (
        ctypes.c_int,
        [_vp, _vp, _vp, _i64, _i64, _i64, ctypes.POINTER(_vp), ctypes.c_int, ctypes.c_int, _i64, _i64, ctypes.c_int,
         _vp],
    ),
    "b2_layernorm_gather_fwd": (
        ctypes.c_int, [_vp, _vp, _vp, ctypes.c_float, ctypes.POINTER(_vp), ctypes.c_int, _vp, _i64, _i64, _vp],
    ),
    "b2_rotary_fwd": (ctypes.c_int, [ctypes.c_char_p, _vp]),
    "b2_cache_append_fwd": (ctypes.c_int, [ctypes.c_char_p, _vp]),
    "b2_cache_attention_fwd": (ctypes.c_int, [ctypes.c_char_p, _vp]),
    "b2_window_attention_fwd": (ctypes.c_int, [ctypes.c_char_p, _vp]),
    "b2_cache_attention_workspace": (
        ctypes.c_int, [_i64, _i64, _i64, _i64, _i64, ctypes.c_int, ctypes.POINTER(_i64)],
    ),
}

_lock = threading.Lock()
_lib: Optional[ctypes.CDLL] = None


def load_library() -> ctypes.CDLL:
    """Loads libb200tx.so once and binds every entry point; raises if it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -m tiktoktechjam2026track3_b200.build` "
                "(this package has no CPU or PyTorch fallback)"
            )
        lib = ctypes.CDLL(str(LIB_PATH))
        for name, (restype, argtypes) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = restype
            fn.argtypes = argtypes
        version = lib.b2_abi_version()
        if version != 1:
            raise RuntimeError(f"libb200tx.so ABI version {version}, expected 1")
        _lib = lib
        return lib


def _check(status: int, what: str) -> None:
    if status != 0:
        message = load_library().b2_last_error().decode(errors="replace")
        raise RuntimeError(f"{what} failed with status {status}: {message}")


# The current stream's handle without making a torch.cuda.Stream object for it (0.15 us against 2.3 us of host time a
# call, a quarter of a small kernel's launch); the object's way where this build of torch lacks the query.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)  # without its check for a first use


def _stream_ptr(device: torch.device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _stream_of(device: int) -> int:
    """The current stream's handle of GPU `device`."""
    return _raw_stream(device) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _require(t: torch.Tensor, dtype: torch.dtype, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this package has no CPU path)")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def device_status(clear: bool = True) -> int:
    """Status of the current device (0 = no kernel gave up waiting or met an index outside its table)."""
    lib = load_library()
    out = ctypes.c_uint32(0)
    _check(lib.b2_device_status(ctypes.byref(out), 1 if clear else 0), "b2_device_status")
    return int(out.value)


def mask_lengths(mask: torch.Tensor, kv_len: torch.Tensor, not_prefix: torch.Tensor,
                 row_mask_out: Optional[torch.Tensor] = None) -> None:
    """kv_len[b] = valid keys of row b, not_prefix[b] = 1 where row b is not a prefix (see
    b2_mask_lengths); mask is a contiguous bool [B, S] CUDA tensor."""
    if mask.dtype != torch.bool or mask.dim() != 2:
        raise ValueError("mask must be bool [batch, seq_len]")
    _require(mask, torch.bool, "mask")
    _require(kv_len, torch.int32, "kv_len")
    _require(not_prefix, torch.uint8, "not_prefix")
    batch, seq_len = mask.shape
    if kv_len.numel() < batch or not_prefix.numel() < batch:
        raise ValueError("kv_len and not_prefix need one entry per sequence")
    if row_mask_out is not None:
        _require(row_mask_out, torch.uint8, "row_mask_out")
    _check(load_library().b2_mask_lengths(_ptr(mask), batch, seq_len, _ptr(kv_len), _ptr(row_mask_out),
                                          _ptr(not_prefix), _stream_ptr(mask.device)), "b2_mask_lengths")


def set_wait_limit(limit_ns: int = 0) -> None:
    """Limit of one pipeline wait on the current device in ns (0 = the default 4 s)."""
    _check(load_library().b2_set_wait_limit(int(limit_ns)), "b2_set_wait_limit")


def test_set_fault(fault: int) -> None:
    """Test-only fault selector (see b2_test_set_fault); 0 turns it off."""
    _check(load_library().b2_test_set_fault(int(fault)), "b2_test_set_fault")


class StatusWatch:
    """Checks every forward pass for a kernel pipeline timeout without synchronising.

    `after_forward()` enqueues a copy of the device's status word into pinned host memory behind
    the pass's kernels (b2_device_status_async) and records an event; `check()` reads the copy of
    an earlier pass once its event has completed (never waiting for it unless `wait=True`) and
    raises RuntimeError if a kernel gave up waiting, so a timed-out pass is reported at the latest
    by the next call. The status word is sticky until cleared (b2_device_status(clear=1)), so a
    timeout is never missed, only reported one call late when its copy has not landed yet.

    With `indices` it watches the word of the serving operators' indices too (b2_index_status_async): a position,
    length or page number of any caller on the device that lay outside its table.
    """

    def __init__(self, indices: bool = False) -> None:
        self._indices = indices
        self._host: Optional[torch.Tensor] = None
        self._event: Optional[torch.cuda.Event] = None
        self.status = 0

    def check(self, wait: bool = False) -> int:
        ev = self._event
        if ev is None:
            return 0
        if not wait and not ev.query():
            return 0
        ev.synchronize()
        self._event = None
        value = int(self._host[0].item()) or int(self._host[1].item())
        if value:
            self.status = value
            kernel, site, reason = value >> 16, (value >> 8) & 0xFF, value & 0xFF
            names = {1: "layernorm", 2: "linear", 3: "attention", 4: "peer barrier", 5: "rotary", 6: "cache append",
                     7: "cache attention"}
            what, so = "gave up waiting", "outputs computed since then are not valid"
            if reason == REASON_BAD_INDEX:
                what, so = "met an index outside its table", "what it names was skipped"
            raise RuntimeError(
                f"a {names.get(kernel, kernel)} kernel {what} (status {value:#x}: site {site}, reason "
                f"{reason}); {so}. Clear the status with _capi.device_status(clear=True) after handling it")
        return 0

    def after_forward(self, device: torch.device) -> None:
        if self._host is None:
            self._host = torch.zeros(2, dtype=torch.int32, pin_memory=True)
        if self._event is not None and not self._event.query():
            return  # the previous copy is still in flight: it will report the same sticky word
        self._event = None
        lib = load_library()
        _check(lib.b2_device_status_async(self._host.data_ptr(), _stream_ptr(device)), "b2_device_status_async")
        if self._indices:
            _check(lib.b2_index_status_async(self._host.data_ptr() + 4, _stream_ptr(device)), "b2_index_status_async")
        ev = torch.cuda.Event()
        ev.record(torch.cuda.current_stream(device))
        self._event = ev


def layernorm(
    x: torch.Tensor,
    gamma: torch.Tensor,
    beta: torch.Tensor,
    eps: float,
    y: torch.Tensor,
    resid_out: Optional[torch.Tensor] = None,
    row_mask: Optional[torch.Tensor] = None,
) -> None:
    """y = LayerNorm(x) in bf16 (see b2_layernorm_fwd)."""
    d_model = x.shape[-1]
    rows = x.numel() // d_model
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("x must be float32 or bfloat16")
    _require(x, x.dtype, "x")
    _require(gamma, torch.bfloat16, "gamma")
    _require(beta, torch.bfloat16, "beta")
    _require(y, torch.bfloat16, "y")
    if y.numel() != x.numel():
        raise ValueError("y must have x's shape")
    if resid_out is not None:
        _require(resid_out, torch.float32, "resid_out")
    if row_mask is not None:
        _require(row_mask, torch.uint8, "row_mask")
    status = load_library().b2_layernorm_fwd(
        _ptr(x), 1 if x.dtype == torch.bfloat16 else 0, _ptr(gamma), _ptr(beta), float(eps), _ptr(y),
        _ptr(resid_out), _ptr(row_mask), rows, d_model, _stream_ptr(x.device),
    )
    _check(status, "b2_layernorm_fwd")


ADD_LN_ZERO_ROWS = 1
ADD_LN_ZERO_Y = 2


def add_layernorm(
    resid: torch.Tensor,
    delta: torch.Tensor,
    bias: Optional[torch.Tensor],
    gamma: torch.Tensor,
    beta: torch.Tensor,
    eps: float,
    y: torch.Tensor,
    row_mask: Optional[torch.Tensor] = None,
    flags: int = 0,
) -> None:
    """resid = mask ? resid + delta + bias : (resid | 0); y = LayerNorm(resid) (b2_add_layernorm_fwd)."""
    d_model = resid.shape[-1]
    rows = resid.numel() // d_model
    _require(resid, torch.float32, "resid")
    _require(delta, torch.float32, "delta")
    _require(gamma, torch.bfloat16, "gamma")
    _require(beta, torch.bfloat16, "beta")
    _require(y, torch.bfloat16, "y")
    if delta.numel() != resid.numel() or y.numel() != resid.numel():
        raise ValueError("resid, delta and y must have the same number of elements")
    if bias is not None:
        _require(bias, torch.bfloat16, "bias")
    if row_mask is not None:
        _require(row_mask, torch.uint8, "row_mask")
    status = load_library().b2_add_layernorm_fwd(
        _ptr(resid), _ptr(delta), _ptr(bias), _ptr(row_mask), int(flags), _ptr(gamma), _ptr(beta), float(eps),
        _ptr(y), rows, d_model, _stream_ptr(resid.device),
    )
    _check(status, "b2_add_layernorm_fwd")


def linear(
    a: torch.Tensor,
    w: torch.Tensor,
    bias: Optional[torch.Tensor],
    epilogue: int,
    out: torch.Tensor,
    row_mask: Optional[torch.Tensor] = None,
    tile_n: int = 0,
) -> None:
    """out = epilogue(a @ w.T + bias) (see b2_linear_fwd)."""
    _require(a, torch.bfloat16, "a")
    _require(w, torch.bfloat16, "w")
    m, k = a.shape[0] if a.dim() == 2 else a.numel() // a.shape[-1], a.shape[-1]
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"w has shape {tuple(w.shape)}, expected [n, {k}]")
    if bias is not None:
        _require(bias, torch.bfloat16, "bias")
    out_dtype = torch.bfloat16 if epilogue in (EPI_BIAS, EPI_BIAS_GELU) else torch.float32
    _require(out, out_dtype, "out")
    if out.numel() < m * n:
        raise ValueError("out is too small")
    dst, ldo = out.data_ptr(), out.shape[-1]
    if row_mask is not None:
        _require(row_mask, torch.uint8, "row_mask")
    status = load_library().b2_linear_fwd(
        _ptr(a), _ptr(w), _ptr(bias), m, n, k, int(epilogue), dst, ldo, _ptr(row_mask), int(tile_n),
        _stream_ptr(a.device),
    )
    _check(status, "b2_linear_fwd")


def linear_ln_plan(m: int, n: int, k: int, sm_count: int = 0) -> Optional[Tuple[int, int, bool]]:
    """(tile_n, cluster, recommended) of b2_linear_ln_fwd for an m x n x k problem, or None when n
    has no fused plan (see b2_linear_ln_plan). sm_count 0 asks the current device."""
    lib = load_library()
    tile, cluster, rec = ctypes.c_int(0), ctypes.c_int(0), ctypes.c_int(0)
    status = lib.b2_linear_ln_plan(int(m), int(n), int(k), int(sm_count), ctypes.byref(tile), ctypes.byref(cluster),
                                   ctypes.byref(rec))
    if status == 2:
        return None
    _check(status, "b2_linear_ln_plan")
    return int(tile.value), int(cluster.value), bool(rec.value)


def linear_ln(
    a: torch.Tensor,
    w: torch.Tensor,
    bias: Optional[torch.Tensor],
    resid: torch.Tensor,
    gamma: torch.Tensor,
    beta: torch.Tensor,
    eps: float,
    ln_out: torch.Tensor,
    zero_masked_rows: bool,
    row_mask: Optional[torch.Tensor] = None,
) -> None:
    """resid = mask ? resid + a @ w.T + bias : (0 | resid); ln_out = LayerNorm(resid) (b2_linear_ln_fwd)."""
    _require(a, torch.bfloat16, "a")
    _require(w, torch.bfloat16, "w")
    _require(resid, torch.float32, "resid")
    _require(gamma, torch.bfloat16, "gamma")
    _require(beta, torch.bfloat16, "beta")
    _require(ln_out, torch.bfloat16, "ln_out")
    k = a.shape[-1]
    m = a.numel() // k
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"w has shape {tuple(w.shape)}, expected [n, {k}]")
    if resid.numel() != m * n or ln_out.numel() != m * n or resid.shape[-1] != n:
        raise ValueError(f"resid and ln_out must be [{m}, {n}]")
    if bias is not None:
        _require(bias, torch.bfloat16, "bias")
    if row_mask is not None:
        _require(row_mask, torch.uint8, "row_mask")
    status = load_library().b2_linear_ln_fwd(
        _ptr(a), _ptr(w), _ptr(bias), m, n, k, 1 if zero_masked_rows else 0, _ptr(resid), _ptr(row_mask), _ptr(gamma),
        _ptr(beta), float(eps), _ptr(ln_out), _stream_ptr(a.device),
    )
    _check(status, "b2_linear_ln_fwd")


def attention(
    qkv: torch.Tensor,
    batch: int,
    seq_len: int,
    num_heads: int,
    head_dim: int,
    q_col: int,
    k_col: int,
    v_col: int,
    kv_len: Optional[torch.Tensor],
    causal: bool,
    scale: float,
    ctx: torch.Tensor,
    q_rows=None,
) -> None:
    """ctx = softmax(mask(q k^T * scale)) v per head (see b2_attention_fwd).

    q_rows = (q_begin, q_count), or a list of up to two such ranges in sequence order, computes
    only those query rows of every sequence (b2_attention_rows_fwd).
    """
    _require(qkv, torch.bfloat16, "qkv")
    _require(ctx, torch.bfloat16, "ctx")
    if kv_len is not None:
        _require(kv_len, torch.int32, "kv_len")
        if kv_len.numel() != batch:
            raise ValueError("kv_len must have one entry per sequence")
    lib = load_library()
    if q_rows is None:
        status = lib.b2_attention_fwd(
            _ptr(qkv), qkv.shape[-1], q_col, k_col, v_col, batch, seq_len, num_heads, head_dim, _ptr(kv_len),
            1 if causal else 0, float(scale), _ptr(ctx), ctx.shape[-1], _stream_ptr(qkv.device),
        )
        _check(status, "b2_attention_fwd")
        return
    ranges = [tuple(q_rows)] if isinstance(q_rows[0], int) else [tuple(r) for r in q_rows]
    arr = (_i64 * (2 * len(ranges)))(*[int(v) for r in ranges for v in r])
    status = lib.b2_attention_rows_fwd(
        _ptr(qkv), qkv.shape[-1], q_col, k_col, v_col, batch, seq_len, num_heads, head_dim, _ptr(kv_len),
        1 if causal else 0, float(scale), arr, len(ranges), _ptr(ctx), ctx.shape[-1], _stream_ptr(qkv.device),
    )
    _check(status, "b2_attention_rows_fwd")


PAD_WORDS = 32  # kPadChannels x kMaxPeers uint32 flags per rank


def peer_barrier(pads, rank: int, channel: int, device: torch.device) -> None:
    """Enqueues a cross-GPU barrier on the current stream (see b2_peer_barrier).

    `pads` lists every rank's flag-pad device address (ints) as mapped into this process.
    """
    arr = (_vp * len(pads))(*[int(p) for p in pads])
    status = load_library().b2_peer_barrier(arr, len(pads), int(rank), int(channel), _stream_ptr(device))
    _check(status, "b2_peer_barrier")


def linear_rs(a: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], zero_masked_rows: bool, peer_resid,
              rank: int, rows_per_rank: int, ldo: int, row_mask: Optional[torch.Tensor] = None, tile_n: int = 0) -> None:
    """Residual GEMM whose rows are added into their owner rank's residual (see b2_linear_rs_fwd).

    `peer_resid` lists every rank's residual base address (ints) as mapped into this process.
    """
    _require(a, torch.bfloat16, "a")
    _require(w, torch.bfloat16, "w")
    m, k = a.shape
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError("a and w disagree on K")
    if bias is not None:
        _require(bias, torch.bfloat16, "bias")
    if row_mask is not None:
        _require(row_mask, torch.uint8, "row_mask")
    arr = (_vp * len(peer_resid))(*[int(x) for x in peer_resid])
    status = load_library().b2_linear_rs_fwd(
        _ptr(a), _ptr(w), _ptr(bias), m, n, k, 1 if zero_masked_rows else 0, arr, len(peer_resid), int(rank),
        int(rows_per_rank), int(ldo), _ptr(row_mask), int(tile_n), _stream_ptr(a.device),
    )
    _check(status, "b2_linear_rs_fwd")


def layernorm_gather(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float, y_ranks,
                     row_mask: Optional[torch.Tensor] = None) -> None:
    """LayerNorm of fp32 rows x written as bf16 into every rank's buffer (see b2_layernorm_gather_fwd).

    `y_ranks` lists each rank's destination address (ints) for x's first row.
    """
    _require(x, torch.float32, "x")
    _require(gamma, torch.bfloat16, "gamma")
    _require(beta, torch.bfloat16, "beta")
    if row_mask is not None:
        _require(row_mask, torch.uint8, "row_mask")
    d_model = x.shape[-1]
    rows = x.numel() // d_model
    arr = (_vp * len(y_ranks))(*[int(p) for p in y_ranks])
    status = load_library().b2_layernorm_gather_fwd(
        _ptr(x), _ptr(gamma), _ptr(beta), float(eps), arr, len(y_ranks), _ptr(row_mask), rows, d_model,
        _stream_ptr(x.device),
    )
    _check(status, "b2_layernorm_gather_fwd")


def linear_bcast(a: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], peer_out, rank: int, col_begin: int,
                 ldo: int, tile_n: int = 0) -> None:
    """out = bf16(a @ w.T + bias) into peer_out[rank], columns >= col_begin also into every other
    rank's peer_out (see b2_linear_bcast_fwd). `peer_out` lists device addresses (ints)."""
    _require(a, torch.bfloat16, "a")
    _require(w, torch.bfloat16, "w")
    m, k = a.shape
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError("a and w disagree on K")
    if bias is not None:
        _require(bias, torch.bfloat16, "bias")
    arr = (_vp * len(peer_out))(*[int(x) for x in peer_out])
    status = load_library().b2_linear_bcast_fwd(
        _ptr(a), _ptr(w), _ptr(bias), m, n, k, arr, len(peer_out), int(rank), int(col_begin), int(ldo), int(tile_n),
        _stream_ptr(a.device),
    )
    _check(status, "b2_linear_bcast_fwd")


_BF16, _INT32 = torch.bfloat16, torch.int32


def _elsewhere(t: torch.Tensor, name: str, device: int) -> ValueError:
    if not t.is_cuda:
        return ValueError(f"{name} must be a CUDA tensor (this package has no CPU path)")
    return ValueError(f"{name} must be on cuda:{device} as the call's other tensors, got {t.device}")


def _launch(entry: str, layout: struct.Struct, device: int, *members) -> None:
    """One serving entry point on the current stream of the GPU that holds the call's tensors, made current for it."""
    fn = getattr(_lib or load_library(), entry)
    try:
        args = layout.pack(*members)
    except struct.error as e:
        raise TypeError(f"{entry}: sizes, windows and counts must be 64-bit integers, scales numbers ({e})") from None
    if _current_device() == device:
        status = fn(args, _stream_of(device))
    else:
        with torch.cuda.device(device):
            status = fn(args, _stream_of(device))
    if status:
        _check(status, entry)


def _rows(t: torch.Tensor, name: str, device: int) -> int:
    """Row stride of a bf16 matrix on `device` whose rows are contiguous (a column slice of packed rows is one)."""
    stride = t.stride()
    if len(stride) != 2 or stride[1] != 1 or t.dtype is not _BF16 or t.get_device() != device or device < 0:
        if t.get_device() != device or device < 0:
            raise _elsewhere(t, name, device)
        if t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be {torch.bfloat16}, got {t.dtype}")
        raise ValueError(f"{name} must be 2-D with contiguous rows")
    # A single row's stride may be anything: its length takes the place.
    return stride[0] if t.size(0) > 1 else (t.size(1) + 7) // 8 * 8


def _table(t: torch.Tensor, device: int) -> Tuple[int, int]:
    """(positions, rotary_dim) of a rotary table [positions, rotary_dim / 2, 2]."""
    if t.dim() != 3 or t.size(2) != 2:
        raise ValueError("table must be [positions, rotary_dim / 2, 2]")
    if t.get_device() != device:
        raise _elsewhere(t, "table", device)
    _require(t, torch.float32, "table")
    return t.size(0), 2 * t.size(1)


def _indices(t: torch.Tensor, n: int, name: str, device: int) -> int:
    """Pointer of n contiguous int32 entries on `device`."""
    if t.get_device() != device:
        raise _elsewhere(t, name, device)
    if t.dtype is not _INT32 or not t.is_contiguous():
        _require(t, _INT32, name)
    if t.numel() != n:
        raise ValueError(f"{name} must have {n} entries, got {t.numel()}")
    return t.data_ptr()


def _page_table(t: torch.Tensor, batch: int, device: int) -> Tuple[int, int]:
    """(pointer, pages per sequence) of an int32 page table."""
    if t.dim() != 2 or t.size(0) != batch:
        raise ValueError(f"page_table must be [{batch}, pages], got {tuple(t.shape)}")
    if t.get_device() != device:
        raise _elsewhere(t, "page_table", device)
    if t.dtype is not _INT32 or not t.is_contiguous():
        _require(t, _INT32, "page_table")
    return t.data_ptr(), t.size(1)


def rotary(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, head_dim: int, out: torch.Tensor,
           interleaved: bool = False, inverse: bool = False) -> None:
    """out = the rows of x with every head turned by its row's position (see b2_rotary_fwd)."""
    device = x.get_device()
    ld_x, ld_out = _rows(x, "x", device), _rows(out, "out", device)
    tokens, width = x.size(0), x.size(1)
    if head_dim < 1 or width % head_dim or out.size(0) != tokens or out.size(1) != width:
        raise ValueError(f"x and out must both be [tokens, heads * {head_dim}]")
    most, rotary_dim = _table(table, device)
    _launch(
        "b2_rotary_fwd", ROTARY_ARGS, device, x.data_ptr(), ld_x, tokens, width // head_dim, head_dim, rotary_dim,
        interleaved, inverse, _indices(positions, tokens, "positions", device), table.data_ptr(), most, out.data_ptr(),
        ld_out)


def cache_append(cache: KVCacheDesc, qkv: torch.Tensor, num_heads: int, q_col: int, k_col: int, v_col: int,
                 new_start: torch.Tensor, new_len: torch.Tensor, past_len: torch.Tensor, page_table: torch.Tensor,
                 max_new: int, table: Optional[torch.Tensor] = None, interleaved: bool = False,
                 q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> None:
    """Stores (and with `table` rotates) the new tokens of packed rows qkv (see b2_cache_append_fwd)."""
    device = cache.device
    ld = _rows(qkv, "qkv", device)
    batch, tokens = new_len.numel(), qkv.size(0)
    pages, table_pages = _page_table(page_table, batch, device)
    positions = rotary_dim = ld_q = ld_k = 0
    if table is not None:
        positions, rotary_dim = _table(table, device)
        if q_out is None:
            raise ValueError("a rotation needs q_out")
    if q_out is not None:
        ld_q = _rows(q_out, "q_out", device)
        if table is None or q_out.size(0) != tokens or q_out.size(1) != num_heads * cache.head_dim:
            raise ValueError("q_out needs a table and the shape [tokens, num_heads * head_dim]")
    if k_out is not None:
        ld_k = _rows(k_out, "k_out", device)
        if k_out.size(0) != tokens or k_out.size(1) != cache.kv_heads * cache.head_dim:
            raise ValueError("k_out must be [tokens, kv_heads * head_dim]")
    _launch(
        "b2_cache_append_fwd", CACHE_APPEND_ARGS, device, ctypes.addressof(cache), qkv.data_ptr(), ld, q_col, k_col,
        v_col, tokens, num_heads, batch, _indices(new_start, batch, "new_start", device),
        _indices(new_len, batch, "new_len", device), _indices(past_len, batch, "past_len", device), pages, table_pages,
        max_new, 0 if table is None else table.data_ptr(), positions, rotary_dim, interleaved,
        0 if q_out is None else q_out.data_ptr(), ld_q, 0 if k_out is None else k_out.data_ptr(), ld_k)


def cache_attention_workspace(batch: int, q_len: int, num_heads: int, kv_heads: int, head_dim: int,
                              sm_count: int = 0) -> int:
    """Bytes of cache_attention's workspace (see b2_cache_attention_workspace)."""
    out = _i64(0)
    _check(load_library().b2_cache_attention_workspace(batch, q_len, num_heads, kv_heads, head_dim, sm_count,
                                                       ctypes.byref(out)), "b2_cache_attention_workspace")
    return int(out.value)


def cache_attention(cache: KVCacheDesc, q: torch.Tensor, q_len: int, page_table: torch.Tensor, kv_len: torch.Tensor,
                    window: int, sinks: int, scale: float, out: torch.Tensor, workspace: torch.Tensor) -> None:
    """out = attention of the q_len newest tokens of each sequence over the cache (see b2_cache_attention_fwd)."""
    device = cache.device
    ld_q, ld_out = _rows(q, "q", device), _rows(out, "out", device)
    if workspace.get_device() != device:
        raise _elsewhere(workspace, "workspace", device)
    rows, width = q.size(0), q.size(1)
    batch = kv_len.numel()
    pages, table_pages = _page_table(page_table, batch, device)
    if rows != batch * q_len:
        raise ValueError("q needs q_len rows and kv_len an entry per sequence")
    head_dim = cache.head_dim
    if width % head_dim or out.size(0) != rows or out.size(1) != width:
        raise ValueError("q and out must both be [batch * q_len, heads * head_dim]")
    _launch(
        "b2_cache_attention_fwd", CACHE_ATTENTION_ARGS, device, ctypes.addressof(cache), q.data_ptr(), ld_q, batch, q_len,
        width // head_dim, pages, table_pages, _indices(kv_len, batch, "kv_len", device), window, sinks, scale,
        out.data_ptr(), ld_out, workspace.data_ptr(), workspace.numel())


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: int, seq_len: int, head_dim: int,
                     window: int, sinks: int, kv_len: Optional[torch.Tensor], scale: float, out: torch.Tensor) -> None:
    """out = causal attention with a sliding window and sinks (see b2_window_attention_fwd)."""
    device = q.get_device()
    ld_q, ld_k = _rows(q, "q", device), _rows(k, "k", device)
    ld_v, ld_out = _rows(v, "v", device), _rows(out, "out", device)
    rows, width, k_width = q.size(0), q.size(1), k.size(1)
    if (rows != batch * seq_len or k.size(0) != rows or v.size(0) != rows or out.size(0) != rows or v.size(1) != k_width
            or out.size(1) != width):
        raise ValueError("q, k, v and out must have batch * seq_len rows, k and v alike, out like q")
    if head_dim < 1 or width % head_dim or k_width % head_dim:
        raise ValueError(f"q and k must be whole heads of {head_dim}")
    _launch(
        "b2_window_attention_fwd", WINDOW_ATTENTION_ARGS, device, q.data_ptr(), ld_q, k.data_ptr(), ld_k, v.data_ptr(),
        ld_v, batch, seq_len, width // head_dim, k_width // head_dim, head_dim,
        0 if kv_len is None else _indices(kv_len, batch, "kv_len", device), window, sinks, scale, out.data_ptr(), ld_out)
