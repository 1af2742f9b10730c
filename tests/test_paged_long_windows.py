"""Windows of chunk attention that reach back to a table's first position or beyond hide nothing, whatever their size:
what the C entry is asked for (on the CPU, with a stand-in for the library)."""
import sys

import pytest
import torch

from lagunalab_amd import _lib, paged

WIDTH = 3  # pages of a table row: 192 positions


@pytest.fixture
def asked(monkeypatch):
    """The windows of the calls made."""
    got = []

    class Library:
        def lq_paged_chunk_workspace_bytes(self, counts, n, hq, kv, width, window):
            got.append(window)
            return 0

        def lq_paged_chunk_attn(self, *a):
            got.append(a[19])
            return 0

    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)
    monkeypatch.setattr(_lib, "on_device", lambda dev: _lib._HERE)
    monkeypatch.setattr(_lib, "raw_stream", lambda dev: 0)
    monkeypatch.setattr(_lib, "load", Library)
    monkeypatch.setattr(paged, "_pool", lambda keys, values: (*keys[0].shape[:2], keys[0].device, [256] * 6))
    return got


@pytest.mark.parametrize("window,want", [
    (None, 0), (1, 1), (191, 191), (192, 0), (193, 0), (1 << 40, 0), (sys.maxsize, 0), (2 ** 64 + 5, 0),
])
def test_the_window_asked_for(asked, window, want):
    keys, values = paged.page_pool(4, 2, device="cpu")
    q, lens = torch.zeros((4, 2, 128), dtype=torch.bfloat16), torch.ones(2, dtype=torch.int32)
    paged.paged_chunk_attention(q, keys, values, torch.zeros((2, WIDTH), dtype=torch.int32), lens, 0.1, window=window)
    assert asked == [want, want]
