"""A causal stack that answers token by token: a UserOptimizedTransformer's weights over a paged key/value cache.

The reference's forward (transformer_benchmark/models.py:909-919) computes every position of a whole sequence.
`StreamingTransformer` computes a prompt's positions once, keeps their keys and values, and goes on from there,
one token (or a few) of each sequence at a time:

    stream = StreamingTransformer(model, batch=8, max_tokens=4096, table=rotary_table(4096, 64), window=1024, sinks=4)
    y = stream.prompt(x, lengths)     # [8, S, D]; x's rows past lengths[b] are padding
    y = stream.step(x_next)           # [8, t, D], t new tokens of every sequence
    y = stream.extend(x_more, counts) # [sum(counts), D], counts[b] more tokens of sequence b, packed without padding

Per block: LayerNorm -> packed QKV GEMM -> KVCache.append (positions rotated, keys and values stored) -> window_attention
(prompt), KVCache.attend (step) or KVCache.read and packed_attention (extend) -> out_proj + residual -> LayerNorm -> FFN +
residual, all in libb200tx.so.
Without a table, a window and 8 bits it computes what the model's own causal forward does.
"""

from __future__ import annotations

import functools
from typing import Callable, List, Optional, Sequence

import torch

from . import _capi
from .models import UserOptimizedTransformer
from .serving import CACHE_HEAD_DIMS, KVCache, packed_attention, window_attention


class _Rows:
    """Activation buffers of `rows` tokens."""

    def __init__(self, cfg, rows: int, device: torch.device) -> None:
        d, f = cfg.d_model, cfg.ffn_dim
        self.resid = torch.empty(rows, d, device=device, dtype=torch.float32)
        self.ln = torch.empty(rows, d, device=device, dtype=torch.bfloat16)
        self.qkv = torch.empty(rows, 3 * d, device=device, dtype=torch.bfloat16)
        self.ctx = torch.empty(rows, d, device=device, dtype=torch.bfloat16)
        self.hidden = torch.empty(rows, f, device=device, dtype=torch.bfloat16)


def _plain_tensors(f):
    """f without gradients and with tensors that every autograd mode may write, whatever mode its caller is in."""
    @functools.wraps(f)
    def g(*args, **kwargs):
        with torch.inference_mode(False), torch.no_grad():
            return f(*args, **kwargs)
    return g


class StreamingTransformer:
    """Prompt and step passes of a causal UserOptimizedTransformer over `batch` sequences of up to `max_tokens`.

    table, interleaved: rotary positions (`rotary_table`; None: none, as the model's own forward). window, sinks: each
    token sees the `window` newest tokens and the first `sinks` ones (0: all). dtype: of the cache, float8_e4m3fn,
    bfloat16 or uint8 (4-bit codes). Every pass uses the model's weights as they are: a change since the last one is seen by
    the parameters' storage and version, as in the model's own forward. What is in the cache stays as it was computed.
    """

    @_plain_tensors
    def __init__(self, model: UserOptimizedTransformer, batch: int, max_tokens: int, *,
                 table: Optional[torch.Tensor] = None, interleaved: bool = False, window: int = 0, sinks: int = 0,
                 page_size: int = 64, dtype: torch.dtype = torch.float8_e4m3fn) -> None:
        cfg = model.config
        if not cfg.causal:
            raise ValueError("answering token by token needs a causal model")
        if cfg.head_dim not in CACHE_HEAD_DIMS:
            raise NotImplementedError(f"head_dim {cfg.head_dim} is not supported {CACHE_HEAD_DIMS}")
        if batch <= 0 or max_tokens <= 0 or window < 0 or sinks < 0 or (sinks and not window):
            raise ValueError("batch and max_tokens must be positive, window and sinks not negative, sinks need a window")
        if table is not None and (table.shape[0] < max_tokens or 2 * table.shape[1] > cfg.head_dim):
            raise ValueError("table must have max_tokens positions and at most head_dim / 2 pairs")
        self.model, self.config = model, cfg
        self.batch, self.max_tokens = batch, max_tokens
        self.table, self.interleaved, self.window, self.sinks = table, interleaved, window, sinks
        self.refresh()
        self.device = self.packed[0].w_qkv.device
        pages = -(-max_tokens // page_size)
        # Sequence b owns pages b * pages ... of every layer's cache.
        self.caches: List[KVCache] = [
            KVCache.allocate(batch * pages, cfg.num_heads, cfg.head_dim, page_size, dtype, self.device)
            for _ in range(cfg.num_layers)]
        ints = dict(dtype=torch.int32, device=self.device)
        self.page_table = torch.arange(batch * pages, **ints).view(batch, pages)
        self.past = torch.zeros(batch, **ints)  # tokens in the cache before a pass
        self.total = torch.zeros(batch, **ints)  # and after it
        self.lengths: List[int] = [0] * batch  # the host's copy
        self._starts = {}
        self._workspaces = {}
        self._graphs = {}
        self._status = _capi.StatusWatch()
        self.use_cuda_graph = True

    @_plain_tensors
    def refresh(self) -> None:
        """Reads the model's weights again; a pass does so by itself where a parameter has changed."""
        self.packed = self.model.packed_weights()
        if not self.packed[0].w_qkv.is_cuda or self.packed[0].w_qkv.dtype != torch.bfloat16:
            raise RuntimeError("model weights must be bfloat16 on the GPU: call .to(device, torch.bfloat16)")
        # Their storage, kept until the next refresh: a pass launched before a change is noticed reads it.
        self._held = [p.detach() for p in self.model.parameters()]
        self._graphs = {}

    def reset(self) -> None:
        """Forgets every sequence."""
        self.past.zero_()
        self.total.zero_()
        self.lengths = [0] * self.batch

    def check_device_status(self) -> None:
        """Waits for the last pass and raises RuntimeError if a kernel of it, or an earlier one, gave up waiting."""
        self._status.check(wait=True)

    # ------------------------------------------------------------------ passes
    @torch.no_grad()
    def prompt(self, x: torch.Tensor, lengths: Optional[Sequence[int]] = None) -> torch.Tensor:
        """The prompts of fresh sequences: x [batch, S, D] bf16, rows past lengths[b] padding (outputs there are zero)."""
        self._check(x)
        seq = x.shape[1]
        new = [seq] * self.batch if lengths is None else [int(n) for n in lengths]
        if len(new) != self.batch or min(new) < 0 or max(new) > seq:
            raise ValueError(f"lengths must be {self.batch} numbers in [0, {seq}]")
        if max(new) > self.max_tokens:
            raise ValueError(f"a prompt of {max(new)} tokens does not fit max_tokens {self.max_tokens}")
        self.reset()
        if max(new) == 0:
            return torch.zeros_like(x)
        cfg = self.config
        ints = dict(dtype=torch.int32, device=self.device)
        count = torch.tensor(new, **ints)
        ragged = min(new) < seq
        mask = None
        if ragged:
            mask = (torch.arange(seq, device=self.device)[None, :] < count[:, None]).to(torch.uint8).view(-1)
        rows = _Rows(cfg, self.batch * seq, self.device)

        def attend(cache: KVCache) -> None:
            q, k, v = rows.qkv.split(cfg.d_model, 1)
            cache.append(rows.qkv, cfg.num_heads, self._start(seq), count, self.past, self.page_table, max(new),
                         table=self.table, interleaved=self.interleaved, q_out=q if self.table is not None else None,
                         k_out=k if self.table is not None else None)
            window_attention(q, k, v, self.batch, seq, cfg.head_dim, window=self.window, sinks=self.sinks,
                             kv_len=count if ragged else None, out=rows.ctx)

        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        self._status.check()
        self._with_weights(lambda: self._pass(x.contiguous().view(-1, cfg.d_model), rows, attend, mask,
                                              out.view(-1, cfg.d_model)))
        self.past.copy_(count)
        self.lengths = new
        self._status.after_forward(self.device)
        return out

    @torch.no_grad()
    def step(self, x: torch.Tensor) -> torch.Tensor:
        """The next t tokens of every sequence: x [batch, t, D] bf16 -> [batch, t, D]."""
        self._check(x)
        t = x.shape[1]
        if max(self.lengths) + t > self.max_tokens:
            raise ValueError(f"{max(self.lengths)} + {t} tokens do not fit max_tokens {self.max_tokens}")
        self._status.check()
        out = torch.empty_like(x, memory_format=torch.contiguous_format)

        def launch() -> None:
            if self.use_cuda_graph:
                static_x, static_out, graph = self._graph(t)
                static_x.copy_(x)
                graph.replay()
                out.copy_(static_out)
            else:
                self._step(x.contiguous(), out, _Rows(self.config, self.batch * t, self.device))

        self._with_weights(launch, lambda: self.past.sub_(t))
        self.lengths = [n + t for n in self.lengths]
        self._status.after_forward(self.device)
        return out

    @torch.no_grad()
    def extend(self, x: torch.Tensor, lengths: Sequence[int]) -> torch.Tensor:
        """lengths[b] further tokens of sequence b (0: none), all sequences' rows one after the other without padding: x
        [sum(lengths), D] bf16 -> the same shape. Chunks of a long prompt, a turn of some conversations, or fresh sequences'
        prompts. As in `step`, the tokens see keys and values as the cache holds them.
        """
        cfg = self.config
        new = [int(n) for n in lengths]
        if len(new) != self.batch or min(new) < 0:
            raise ValueError(f"lengths must be {self.batch} numbers, none negative")
        if x.dim() != 2 or x.shape[0] != sum(new) or x.shape[1] != cfg.d_model:
            raise ValueError(f"x must be [{sum(new)}, {cfg.d_model}], got {tuple(x.shape)}")
        self._check_place(x)
        held = [p + n if n else 0 for p, n in zip(self.lengths, new)]  # keys of the sequences that go on
        if max(held) > self.max_tokens:
            raise ValueError(f"{max(held)} tokens do not fit max_tokens {self.max_tokens}")
        if not x.shape[0]:
            return torch.empty_like(x)
        # Behind a window the sinks and the band of the first new token on are read, one after the other: what lies between them
        # no row sees, and distances within the band stay what they are.
        cut = [max(0, p + 1 - self.window - self.sinks) if n and self.window else 0 for p, n in zip(self.lengths, new)]
        q_at, kv_at = [0], [0]
        for n, m, c in zip(new, held, cut):
            q_at.append(q_at[-1] + n)
            kv_at.append(kv_at[-1] + m - c)
        parts = [(r, m if c == 0 else self.sinks, 0) for r, m, c in zip(kv_at, held, cut)]  # first row, tokens, first token
        page_table = self.page_table
        if any(cut):
            parts += [(r + self.sinks, m - c - self.sinks, c + self.sinks) if c else (0, 0, 0)
                      for r, m, c in zip(kv_at, held, cut)]
            page_table = page_table.repeat(2, 1)
        lists = [q_at, kv_at, new, *map(list, zip(*parts))]
        q_start, kv_start, count, read_row, read_len, read_from = torch.tensor(
            sum(lists, []), dtype=torch.int32, device=self.device).split([len(n) for n in lists])
        most = max(n for _, n, _ in parts)
        rows = _Rows(cfg, x.shape[0], self.device)
        k_rows, v_rows = (torch.empty(kv_at[-1], cfg.d_model, dtype=torch.bfloat16, device=self.device) for _ in range(2))

        def attend(cache: KVCache) -> None:
            q = rows.qkv[:, :cfg.d_model]
            cache.append(rows.qkv, cfg.num_heads, q_start[:-1], count, self.past, self.page_table, max(new), table=self.table,
                         interleaved=self.interleaved, q_out=q if self.table is not None else None)
            cache.read(read_row, read_len, read_from, page_table, most, k_out=k_rows, v_out=v_rows)
            packed_attention(q, k_rows, v_rows, q_start, kv_start, cfg.head_dim, window=self.window, sinks=self.sinks,
                             out=rows.ctx)

        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        self._status.check()
        self._with_weights(lambda: self._pass(x.contiguous(), rows, attend, None, out))
        self.past.add_(count)
        self.lengths = [p + n for p, n in zip(self.lengths, new)]
        self._status.after_forward(self.device)
        return out

    # ------------------------------------------------------------------ inside
    def _with_weights(self, launch: Callable[[], None], undo: Callable[[], object] = lambda: None) -> None:
        """launch() with the model's weights as they are (the packed projections are copies, and graphs hold addresses).

        As in the model's forward the launches come first and the comparison of every parameter with the last pass's
        after them (40 us of host time at 12 layers); where one has changed, undo() and launch() again with the new
        ones. The tokens of the first attempt are overwritten, like drafts that were not taken.
        """
        key = self.model._packed_key
        if self.model._packed is not self.packed or key is None or key[0] == "storage":  # known to differ, or not told
            self._follow_weights()
        launch()
        if self.model._weights_key() != self.model._packed_key and self.model.packed_weights() is not self.packed:
            undo()
            self._follow_weights()
            launch()

    def _follow_weights(self) -> None:
        if self.model.packed_weights() is not self.packed:
            self.refresh()
            if self.packed[0].w_qkv.device != self.device:
                raise RuntimeError(f"the model's weights have left {self.device}, where this object's cache is")

    def _check(self, x: torch.Tensor) -> None:
        if x.dim() != 3 or x.shape[0] != self.batch or x.shape[2] != self.config.d_model or x.shape[1] == 0:
            raise ValueError(f"x must be [{self.batch}, tokens, {self.config.d_model}], got {tuple(x.shape)}")
        self._check_place(x)

    def _check_place(self, x: torch.Tensor) -> None:
        if x.device != self.device or x.dtype != torch.bfloat16:
            raise RuntimeError(f"StreamingTransformer computes in bfloat16 on the GPU of its weights, {self.device}")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a pass cannot be captured: it counts tokens on the host and makes buffers that later passes "
                               "use (steps are replayed from graphs of the object's own)")

    def _start(self, rows: int) -> torch.Tensor:
        """First row of every sequence, `rows` rows each."""
        if rows not in self._starts:
            self._starts[rows] = torch.arange(self.batch, dtype=torch.int32, device=self.device) * rows
        return self._starts[rows]

    def _step(self, x: torch.Tensor, out: torch.Tensor, rows: _Rows, count: Optional[torch.Tensor] = None) -> None:
        cfg, t = self.config, x.shape[1]
        key = (t, torch.cuda.is_current_stream_capturing())
        if key not in self._workspaces:  # a graph's calls and eager ones may run at the same time
            self._workspaces[key] = self.caches[0].workspace(self.batch, cfg.num_heads, t)
        workspace = self._workspaces[key]
        torch.add(self.past, t, out=self.total)
        if count is None:
            count = self._counts(t)

        def attend(cache: KVCache) -> None:
            q = rows.qkv[:, :cfg.d_model]
            cache.append(rows.qkv, cfg.num_heads, self._start(t), count, self.past, self.page_table, t, table=self.table,
                         interleaved=self.interleaved, q_out=q if self.table is not None else None)
            cache.attend(q, self.page_table, self.total, q_len=t, window=self.window, sinks=self.sinks, out=rows.ctx,
                         workspace=workspace)

        self._pass(x.view(-1, cfg.d_model), rows, attend, None, out.view(-1, cfg.d_model))
        self.past.copy_(self.total)

    def _counts(self, t: int) -> torch.Tensor:
        key = ("count", t)
        if key not in self._starts:
            self._starts[key] = torch.full((self.batch,), t, dtype=torch.int32, device=self.device)
        return self._starts[key]

    def _graph(self, t: int):
        """Static input, output and the CUDA graph of a step of t tokens."""
        if t not in self._graphs:
            self._capture(t)
        return self._graphs[t][:3]

    @_plain_tensors
    def _capture(self, t: int) -> None:
        x = torch.zeros(self.batch, t, self.config.d_model, device=self.device, dtype=torch.bfloat16)
        out = torch.empty_like(x)
        rows = _Rows(self.config, self.batch * t, self.device)
        self._start(t), self._counts(t)
        self._workspaces[(t, True)] = self.caches[0].workspace(self.batch, self.config.num_heads, t)
        # One eager pass (first use of each kernel sets its attributes outside capture) that stores no token.
        before = self.past.clone()
        self._step(x, out, rows, torch.zeros_like(self.past))
        self.past.copy_(before)
        torch.cuda.current_stream(self.device).synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._step(x, out, rows)
        self._graphs[t] = (x, out, graph, rows)  # the graph writes rows: they live as long as it does

    def _pass(self, x: torch.Tensor, rows: _Rows, attend, mask: Optional[torch.Tensor], out: torch.Tensor) -> None:
        first = self.packed[0]
        _capi.layernorm(x, first.ln1_w, first.ln1_b, first.ln1_eps, rows.ln, resid_out=rows.resid)
        for i, (pb, cache) in enumerate(zip(self.packed, self.caches)):
            if i:
                _capi.layernorm(rows.resid, pb.ln1_w, pb.ln1_b, pb.ln1_eps, rows.ln)
            _capi.linear(rows.ln, pb.w_qkv, pb.b_qkv, _capi.EPI_BIAS, rows.qkv)
            attend(cache)
            _capi.linear(rows.ctx, pb.w_o, pb.b_o, _capi.EPI_RESIDUAL, rows.resid, mask)
            _capi.layernorm(rows.resid, pb.ln2_w, pb.ln2_b, pb.ln2_eps, rows.ln)
            _capi.linear(rows.ln, pb.w_1, pb.b_1, _capi.EPI_BIAS_GELU, rows.hidden)
            _capi.linear(rows.hidden, pb.w_2, pb.b_2, _capi.EPI_RESIDUAL_ZERO, rows.resid, mask)
        fn = self.model.final_norm
        _capi.layernorm(rows.resid, fn.weight, fn.bias, float(fn.eps), out, row_mask=mask)
