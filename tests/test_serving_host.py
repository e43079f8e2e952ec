"""What the serving operators' Python side decides before a launch (no GPU)."""

import re
from pathlib import Path

import pytest
import torch

from tiktoktechjam2026track3_b200 import _capi, serving
from tiktoktechjam2026track3_b200.build import build


class _Queries:
    """Stands for q: [rows, width] on the GPU."""

    device = torch.device("cuda", 0)

    def __init__(self, rows, width):
        self.shape = (rows, width)

    def size(self, i):
        return self.shape[i]


def _cache(monkeypatch, capturing):
    """A cache without tensors whose workspaces are plain lists, on stream 7."""
    cache = object.__new__(serving.KVCache)
    cache.head_dim, cache._workspaces = 64, {}
    monkeypatch.setattr(_capi, "_stream_ptr", lambda device: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(cache, "workspace", lambda *size: list(size), raising=False)
    return cache


def test_a_captured_call_has_a_workspace_of_its_own(monkeypatch):
    """A graph may outlive the workspace that its stream keeps, and run next to the stream's other calls."""
    capturing = [False]
    cache = _cache(monkeypatch, capturing)
    kept = cache._workspace(_Queries(2, 256), 1)
    assert cache._workspace(_Queries(1, 256), 1) is kept  # smaller calls of the stream share it
    capturing[0] = True
    first, second = cache._workspace(_Queries(2, 256), 1), cache._workspace(_Queries(2, 256), 1)
    assert first is not kept and second is not kept and first is not second
    larger = cache._workspace(_Queries(64, 256), 1)
    assert all(larger is not w for _, w in cache._workspaces.values())
    capturing[0] = False
    assert cache._workspace(_Queries(2, 256), 1) is kept


def test_cache_attention_reads_its_pages_past_the_read_only_path():
    """The launch that writes pages and scales may still run when the attention's first CTAs are resident."""
    text = (Path(serving.__file__).parent / "csrc" / "cache_attention.cuh").read_text()
    assert "pdl_wait_previous_grid" in text
    assert not re.search(r"__ldg|ld\.global(\.\w+)*\.nc", text)


@pytest.mark.parametrize("head_dim", [32, 64, 128])
def test_workspace_does_not_grow_with_the_row_blocks(head_dim):
    """64 rows to a key head (four blocks of 16) at a time; more take turns."""
    build()

    def size(q_len, heads, batch=4):
        return _capi.cache_attention_workspace(batch, q_len, heads, 8, head_dim, sm_count=148)

    assert size(1, 8) <= size(2, 64) <= size(4, 64) <= size(8, 64) == size(1024, 64) <= 21 << 20


def test_workspace_is_alike_for_every_batch():
    """Its counters lie at one place for every call: a workspace is either too small, and refused, or right."""
    build()
    sizes = {_capi.cache_attention_workspace(batch, 2, 4 * kv, kv, 64, sm_count=148) for batch in (1, 64, 4096) for kv in (1, 8)}
    assert len(sizes) == 1
