"""Operators for answering token by token: rotary positions, a paged key/value cache and the attention over it.

The reference computes whole sequences only (transformer_benchmark/models.py:909-919); these are the parts
that a causal stack needs next to it to go on from what it has read:

  * `rotary_table` / `rotary`: rotary positions, half or interleaved pairs, part of a head, tables scaled
    for contexts longer than the trained one; `inverse=True` is the gradient;
  * `KVCache`: pages of keys and values, bf16, 8-bit codes with one power-of-two scale per page and head, or 4-bit codes
    with a step and a middle for every 32 elements of a token and head. `append` stores (and rotates) the rows of a packed QKV
    projection, `attend` is the attention of the newest token, or few tokens, of every sequence, `read` gives the
    tokens of the cache back as rows;
  * `window_attention`: causal prompt attention with a sliding window and first tokens that stay visible;
  * `packed_attention`: the same for packed sequences of different lengths, whose queries may stand behind keys that a cache
    gave back.

Everything runs in libb200tx.so on the current CUDA stream (include/b200tx.h says what each call takes);
there is no CPU or PyTorch fallback. Lengths, positions and page tables stay on the device and are not read
back: an entry outside its table is skipped by the kernel and reported by a status word of the device
(`_capi.device_status`, `_capi.StatusWatch(indices=True)`); it does not stop other callers.
"""

from __future__ import annotations

import math
from typing import Dict, Optional, Tuple, Union

import torch

from . import _capi

PAGE_SIZES = (16, 32, 64, 128, 256)
CACHE_HEAD_DIMS = (32, 64, 128)  # of KVCache.attend
GROUP = 32  # elements of a head of one token that share a step and a middle in 4 bits


def rotary_table(max_positions: int, rotary_dim: int, base: float = 10000.0, scaling: Optional[Tuple] = None,
                 device: Union[str, torch.device] = "cuda") -> torch.Tensor:
    """cos and sin of every position's angles, fp32 [max_positions, rotary_dim / 2, 2], computed in 64 bits.

    Pair i turns by position * base^(-2i / rotary_dim). `scaling` stretches that for contexts `factor` times longer
    than the trained ones:
      ("linear", factor)             every angle divided by factor (position interpolation);
      ("ntk", factor)                base * factor^(r / (r - 2)): the fastest pair unchanged, the slowest divided by factor;
      ("parts", factor, trained[, slow, fast])  pairs that turn more than `fast` (32) times within the `trained`
          positions unchanged, those that turn less than `slow` (1) times divided by factor, a linear ramp between, and
          cos and sin multiplied by 0.1 ln(factor) + 1.
    """
    if rotary_dim <= 0 or rotary_dim % 16:
        raise ValueError(f"rotary_dim {rotary_dim} must be a positive multiple of 16")
    if max_positions <= 0 or not base > 1.0:
        raise ValueError("max_positions must be positive and base above 1")
    f64 = dict(dtype=torch.float64, device=device)
    gain = 1.0
    kind = scaling[0] if scaling else None
    if kind not in (None, "linear", "ntk", "parts"):
        raise ValueError(f"unknown scaling {kind!r} (linear, ntk, parts)")
    if scaling and len(scaling) not in ((3, 5) if kind == "parts" else (2,)):
        raise ValueError(f"scaling {scaling!r} must be (kind, factor) or ('parts', factor, trained[, slow, fast])")
    factor = float(scaling[1]) if scaling else 1.0
    if not factor >= 1.0:
        raise ValueError("the scaling factor must be at least 1")
    if kind == "ntk":
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    rate = base ** (-torch.arange(0, rotary_dim, 2, **f64) / rotary_dim)
    if kind == "linear":
        rate = rate / factor
    elif kind == "parts":
        trained = float(scaling[2])
        slow, fast = (float(scaling[3]), float(scaling[4])) if len(scaling) > 3 else (1.0, 32.0)
        if not 0 < slow < fast or not trained > 0:
            raise ValueError("a positive trained length and 0 < slow < fast turns are needed")
        turns = trained * rate / (2.0 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        rate = rate * keep + rate / factor * (1.0 - keep)
        gain = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(max_positions, **f64)[:, None] * rate
    return (torch.stack([angle.cos(), angle.sin()], -1) * gain).float().contiguous()


def rotary(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, head_dim: int, *,
           out: Optional[torch.Tensor] = None, interleaved: bool = False, inverse: bool = False) -> torch.Tensor:
    """Rows x [tokens, heads * head_dim] (bf16, any row stride) turned by their positions (int32 [tokens]).

    Pairs are (i, i + rotary_dim / 2) or, interleaved, (2i, 2i + 1) of each head's first rotary_dim elements (the
    table's width); the rest is copied. `out` may be x. `inverse` turns back: the gradient of
    x from that of the output. A row whose position is negative is not written.
    """
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _capi.rotary(x, positions, table, head_dim, out, interleaved, inverse)
    return out


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: int, seq_len: int, head_dim: int, *,
                     window: int = 0, sinks: int = 0, kv_len: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of prompts: query i sees key j <= i iff window == 0, i - j < window or j < sinks.

    q [batch * seq_len, heads * head_dim], k and v [batch * seq_len, kv_heads * head_dim] (bf16, any row strides: they
    may be column ranges of one packed projection). Query head i reads key head i // (heads / kv_heads).
    Rows past kv_len (int32 [batch]) are zeros. scale is head_dim^-0.5 unless given.
    """
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _capi.window_attention(q, k, v, batch, seq_len, head_dim, window, sinks, kv_len,
                           head_dim**-0.5 if scale is None else scale, out)
    return out


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_start: torch.Tensor,
                     kv_start: Optional[torch.Tensor], head_dim: int, *, window: int = 0, sinks: int = 0,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of packed sequences of different lengths: sequence b's queries are rows q_start[b] ... q_start[b + 1] - 1
    of q, its keys and values rows kv_start[b] ... kv_start[b + 1] - 1 of k and v (None: the same rows as its queries).

    Of n_q queries and n_kv keys, query i stands at p = n_kv - n_q + i and sees key j <= p iff window == 0, p - j < window or
    j < sinks; a row that sees none gives zeros. q [rows, heads * head_dim], k and v [rows, kv_heads * head_dim] (bf16, any row
    strides), q_start and kv_start int32 [batch + 1], ascending. Query head i reads key head i // (heads / kv_heads).
    scale is head_dim^-0.5 unless given. Rows of `out` that belong to no sequence are left as they are (made zero in one
    that is made here).
    """
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    _capi.packed_attention(q, k, v, q_start, q_start if kv_start is None else kv_start, head_dim, window, sinks,
                           head_dim**-0.5 if scale is None else scale, out)
    return out


class KVCache:
    """Pages of keys and values, [pages, kv_heads, page_size, head_dim] each, and the operators on them.

    In 8 bits (torch.float8_e4m3fn) a page has one fp32 scale per head, a power of two, in k_scale / v_scale
    [pages, kv_heads]. In 4 bits (torch.uint8, two codes to a byte: [..., head_dim / 2]) k_scale and v_scale are bf16
    [pages, kv_heads, page_size, 2, head_dim / 32]: of every token, the steps of its groups of 32 elements, then their middles
    (include/b200tx.h has the codes' meaning and order). Which pages a sequence owns is the caller's page table,
    int32 [batch, pages of the longest]: token j of sequence b lies in slot j % page_size of page page_table[b, j // page_size].
    `allocate` makes the tensors; the constructor takes the caller's own (k and v may be slices of one
    buffer: their first two strides are free, but alike). `append` and `read` take any head_dim that is a multiple of 16 (4 bits:
    32) up to 256, `attend` 32, 64 and 128.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None) -> None:
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise ValueError("k and v must be alike: [pages, kv_heads, page_size, head_dim] (4 bits: head_dim / 2)")
        if not k.is_cuda or v.device != k.device:
            raise ValueError("k and v must be CUDA tensors on one device (this package has no CPU path)")
        if k.dtype not in (torch.bfloat16, torch.float8_e4m3fn, torch.uint8):
            raise ValueError(f"a cache is bfloat16, float8_e4m3fn or uint8 (4-bit codes), got {k.dtype}")
        four = k.dtype == torch.uint8
        pages, kv_heads, page_size, width = k.shape  # (of a token, in elements of the tensor)
        head_dim = 2 * width if four else width
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size {page_size} must be one of {PAGE_SIZES}")
        if k.stride(3) != 1 or k.stride(2) != width:
            raise ValueError("the tokens of a page and head must be contiguous")
        self.quantised = k.dtype != torch.bfloat16
        if four:
            if head_dim < GROUP or head_dim % GROUP:
                raise ValueError(f"head_dim {head_dim} of a 4-bit cache must be a multiple of {GROUP}")
            shape = (pages, kv_heads, page_size, 2, head_dim // GROUP)
            for s, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                if s is None or s.shape != shape or s.device != k.device:
                    raise ValueError(f"a 4-bit cache needs {name} {list(shape)} next to it")
                _capi._require(s, torch.bfloat16, name)
        elif self.quantised:
            for s, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                if s is None or s.shape != (pages, kv_heads) or s.device != k.device:
                    raise ValueError(f"an 8-bit cache needs {name} [pages, kv_heads] next to it")
                _capi._require(s, torch.float32, name)
        elif k_scale is not None or v_scale is not None:
            raise ValueError("a bfloat16 cache has no scales")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, kv_heads, page_size, head_dim
        each = 2 if four else 1  # elements of the cache in one of the tensor
        page_stride = k.stride(0) if pages > 1 else kv_heads * page_size * width if kv_heads == 1 else kv_heads * k.stride(1)
        scales, groups = (_capi._ptr(k_scale), _capi._ptr(v_scale)), (None, None)
        if four:
            scales, groups = groups, scales
        self._desc = _capi.KVCacheDesc(
            k.data_ptr(), v.data_ptr(), *scales, pages, kv_heads, page_size, head_dim, each * page_stride,
            each * (k.stride(1) if kv_heads > 1 else page_size * width),
            _capi.CACHE_INT4 if four else _capi.CACHE_E4M3 if self.quantised else _capi.CACHE_BF16, *groups)
        self._desc.device = k.get_device()
        self._workspaces: Dict[int, Tuple[int, torch.Tensor]] = {}  # by stream: width times q_len, and what it needs

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.float8_e4m3fn, device: Union[str, torch.device] = "cuda") -> "KVCache":
        if dtype == torch.uint8 and (head_dim < GROUP or head_dim % GROUP):
            raise ValueError(f"head_dim {head_dim} of a 4-bit cache must be a multiple of {GROUP}")
        shape = (pages, kv_heads, page_size, head_dim // 2 if dtype == torch.uint8 else head_dim)
        k = torch.zeros(shape, dtype=dtype, device=device)
        v = torch.zeros(shape, dtype=dtype, device=device)
        if dtype == torch.uint8:
            groups = (*shape[:3], 2, head_dim // GROUP)
            return cls(k, v, *(torch.zeros(groups, dtype=torch.bfloat16, device=device) for _ in range(2)))
        if dtype != torch.float8_e4m3fn:
            return cls(k, v)
        return cls(k, v, torch.ones(shape[:2], device=device), torch.ones(shape[:2], device=device))

    def append(self, qkv: torch.Tensor, num_heads: int, new_start: torch.Tensor, new_len: torch.Tensor,
               past_len: torch.Tensor, page_table: torch.Tensor, max_new: int, *, table: Optional[torch.Tensor] = None,
               interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
               k_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Stores the keys and values of new tokens: rows new_start[b] ... + new_len[b] of the packed projection
        qkv [tokens, (num_heads + 2 kv_heads) * head_dim] (q, k, v side by side) are sequence b's tokens past_len[b] ...

        With a `table` (rotary_table), K is rotated before it is stored and rotated Q is written to q_out (made if
        None) and returned; k_out, if given, receives K as stored but before rounding to 8 or 4 bits. q_out and k_out may be
        qkv's own columns. max_new (host) is at least every new_len.
        """
        d, hk = self.head_dim, self.kv_heads
        if qkv.shape[-1] != (num_heads + 2 * hk) * d:
            raise ValueError(f"qkv must be [tokens, {(num_heads + 2 * hk) * d}], got {tuple(qkv.shape)}")
        if table is not None and q_out is None:
            q_out = torch.empty(qkv.shape[0], num_heads * d, dtype=qkv.dtype, device=qkv.device)
        _capi.cache_append(self._desc, qkv, num_heads, 0, num_heads * d, (num_heads + hk) * d, new_start, new_len,
                           past_len, page_table, max_new, table, interleaved, q_out, k_out)
        return q_out

    def read(self, out_start: torch.Tensor, length: torch.Tensor, start: torch.Tensor, page_table: torch.Tensor,
             max_len: int, *, k_out: Optional[torch.Tensor] = None,
             v_out: Optional[torch.Tensor] = None) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
        """Cached tokens as rows: row out_start[b] + i of k_out and v_out (bf16 [rows, kv_heads * head_dim], either may be
        None) receives the key and the value of sequence b's token start[b] + i, i < length[b]; what 8 or 4 bits hold is
        rounded to bf16. Other rows are left as they are. max_len (host) is at least every length. Returns (k_out, v_out).
        """
        _capi.cache_read(self._desc, out_start, length, start, page_table, max_len, k_out, v_out)
        return k_out, v_out

    def workspace(self, batch: int, num_heads: int, q_len: int = 1) -> torch.Tensor:
        """A zeroed workspace for `attend` calls of up to this many heads times q_len (any batch), for callers that keep
        their own: calls that may run at the same time (other streams, CUDA graphs) need one each."""
        with torch.cuda.device(self.k.device):  # whose SMs it goes by
            n = _capi.cache_attention_workspace(batch, q_len, num_heads, self.kv_heads, self.head_dim)
        return torch.zeros(n, dtype=torch.uint8, device=self.k.device)

    def attend(self, q: torch.Tensor, page_table: torch.Tensor, kv_len: torch.Tensor, *, q_len: int = 1,
               scale: Optional[float] = None, window: int = 0, sinks: int = 0, out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the q_len newest tokens of each sequence over its kv_len cached ones (those included).

        Row b * q_len + t of q [batch * q_len, heads * head_dim] stands at p = kv_len[b] - q_len + t and sees keys
        j <= p with window == 0, p - j < window or j < sinks; a row that sees none gives zeros. Query head i reads key
        head i // (heads / kv_heads). scale is head_dim^-0.5 unless given.
        """
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if workspace is None:
            workspace = self._workspace(q, q_len)
        elif workspace.dtype != torch.uint8 or not workspace.is_cuda or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous uint8 CUDA tensor (see KVCache.workspace)")
        _capi.cache_attention(self._desc, q, q_len, page_table, kv_len, window, sinks,
                              self.head_dim**-0.5 if scale is None else scale, out, workspace)
        return out

    def _workspace(self, q: torch.Tensor, q_len: int) -> torch.Tensor:
        """The current stream's workspace, kept between calls (those of one stream run one after the other) and made
        anew when a call is larger than all before it. A call that is being captured gets one of its own: its memory
        and its zeroing are part of the graph, which may run next to the stream's other calls and outlive the kept one."""
        shape = q.shape
        if q_len < 1 or len(shape) != 2:
            raise ValueError("q must be [batch * q_len, heads * head_dim], q_len at least 1")
        device = self._desc.device
        if _capi._current_device() != device:  # the streams meant are those of the cache's GPU
            with torch.cuda.device(device):
                return self._workspace(q, q_len)
        if torch.cuda.is_current_stream_capturing():
            return self.workspace(shape[0] // q_len, shape[1] // self.head_dim, q_len)
        stream, need = _capi._stream_of(device), shape[1] * q_len
        kept = self._workspaces.get(stream)
        if kept is None or need > kept[0]:
            kept = need, self.workspace(shape[0] // q_len, shape[1] // self.head_dim, q_len)
            self._workspaces[stream] = kept
        return kept[1]
