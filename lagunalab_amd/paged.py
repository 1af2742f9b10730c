"""A paged 8-bit KV cache: several sessions in one pool (no counterpart in the reference, whose caches
hold one sequence each).

A pool holds the K/V of one layer in pages of 64 positions -- for keys and for values ``(codes uint8
[pages, Hkv, 64, 128], scales bf16 [pages, Hkv, 64, 2], biases)``, every page the contiguous cache's
layout of 64 rows. Row ``b`` of a table (int32 ``[B, width]``, on the device) lists the pages of
sequence ``b`` in order; position ``p`` is slot ``p % 64`` of page ``table[b, p // 64]``.

* :func:`paged_append`, :func:`paged_gather`: rows quantized into the pages, positions read back as bf16;
* :func:`paged_decode_attention`: one new token per sequence, pages that all sequences share read once;
* :func:`copy_pages`: pages copied within the pool;
* :class:`PagedKVCache`: the pool with its page lists -- sequences opened, forked (their pages shared until
  one is written to), trimmed, closed, the pool compacted -- and :class:`PagedBatch`, some of its
  sequences behind the cache protocol of the attention block (``update_and_fetch``, ``attend``).
"""
from __future__ import annotations

import functools
from array import array
import heapq

import torch

from . import _lib
from .prompt_attn import _refuse_grad

PAGE = 64
HEAD_DIM = 128


def page_pool(pages: int, n_kv_heads: int, device="cuda"):
    """An empty pool: ``(keys, values)``, each ``(codes, scales, biases)``."""
    if pages < 1 or n_kv_heads < 1:
        raise ValueError(f"a pool of {pages} pages of {n_kv_heads} heads")
    shape = (pages, n_kv_heads, PAGE)
    return tuple((torch.zeros((*shape, HEAD_DIM), dtype=torch.uint8, device=device),
                  torch.zeros((*shape, HEAD_DIM // 64), dtype=torch.bfloat16, device=device),
                  torch.zeros((*shape, HEAD_DIM // 64), dtype=torch.bfloat16, device=device))
                 for _ in range(2))


def _pool(keys, values):
    """(pages, Hkv, device, the six buffers' pointers) of a checked pool."""
    if len(keys) != 3 or len(values) != 3:
        raise ValueError("a pool's keys and values are (codes, scales, biases)")
    bufs = (*keys, *values)
    lead = keys[0].shape[:2]
    wide, narrow = (*lead, PAGE, HEAD_DIM), (*lead, PAGE, HEAD_DIM // 64)
    for i, t in enumerate(bufs):
        want, dtype = (narrow, torch.bfloat16) if i % 3 else (wide, torch.uint8)
        if t.shape != want or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"pool buffer {tuple(t.shape)} {t.dtype} is not contiguous {want} {dtype}")
    dev = _lib.require_device(*bufs)
    return lead[0], lead[1], dev, [t.data_ptr() for t in bufs]


def _ints(x, n, what, dev, dims=1):
    """An int32 tensor on the pool's device, as the kernels read it (``n``: its first dimension)."""
    if not torch.is_tensor(x) or x.dtype != torch.int32 or x.dim() != dims or x.shape[0] != n:
        raise ValueError(f"{what} must be an int32 tensor with {n} entries or rows, got "
                         f"{(tuple(x.shape), x.dtype) if torch.is_tensor(x) else type(x)}")
    if x.device != dev:
        raise ValueError(f"{what} is on {x.device}, the pool on {dev}")
    return x if x.is_contiguous() or x.stride(-1) == 1 else x.contiguous()


def _table(table, n, dev):
    """(table, entries from one row to the next, entries of a row)."""
    table = _ints(table, n, "table", dev, 2)
    width = table.shape[1]
    if width < 1:
        raise ValueError("table rows of no pages")
    return table, table.stride(0) if n > 1 else width, width


def _counts(counts, B):
    """Host row counts as the C arrays take them."""
    counts = array("i", counts.tolist() if torch.is_tensor(counts) else counts)
    if len(counts) != B:
        raise ValueError(f"{len(counts)} counts for {B} sequences")
    if B and min(counts) < 0:
        raise ValueError(f"negative count in {counts.tolist()}")
    return counts


def _rows(x, T, H, what):
    """Rows [T, H, 128] as the kernels read them: bf16, any token and head strides of 16-byte steps."""
    if x.dtype != torch.bfloat16 or x.shape != (T, H, HEAD_DIM):
        raise ValueError(f"{what} must be bfloat16 {(T, H, HEAD_DIM)}, got {tuple(x.shape)} {x.dtype}")
    st = x.stride()
    if st[2] != 1 or st[0] % 8 or st[1] % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        st = x.stride()
    return x, st[0], st[1]


def _launches(counts):
    """The sequences of a call in launches of at most LQ_MAX_SEQS: (first, how many, rows before, its
    counts' address)."""
    at, ptr = 0, counts.buffer_info()[0]
    for a in range(0, len(counts), _lib.LQ_MAX_SEQS):
        n = min(len(counts) - a, _lib.LQ_MAX_SEQS)
        yield a, n, at, ptr + 4 * a
        at += sum(counts[a:a + n])


def paged_append(k, v, keys, values, table, starts, counts=None):
    """Quantizes rows ``k``, ``v`` (bf16 ``[T, Hkv, 128]``, packed one sequence behind the other) into the
    pages: the ``counts[b]`` rows of sequence ``b`` (host integers; None: as many each) go to its
    positions ``starts[b]``, ``starts[b] + 1``, .. (``starts`` int32 ``[B]`` on the device). Codes, scales
    and biases are those of :func:`lagunalab_amd.quant.quantize`. Rows whose position or page does not
    exist are not stored; no two rows may go to one slot."""
    P, H, dev, ptrs = _pool(keys, values)
    B, T = table.shape[0], k.shape[0]
    if counts is None:
        if B == 0 or T % B:
            raise ValueError(f"{T} rows are not the same number for each of {B} sequences")
        counts = [T // B] * B
    counts = _counts(counts, B)
    if sum(counts) != T:
        raise ValueError(f"counts add up to {sum(counts)}, not to the {T} rows")
    _lib.require_device(k, v, keys[0])
    k, kt, kh = _rows(k, T, H, "k")
    v, vt, vh = _rows(v, T, H, "v")
    table, ts, width = _table(table, B, dev)
    starts = _ints(starts, B, "starts", dev)
    kp, vp, tp, sp = k.data_ptr(), v.data_ptr(), table.data_ptr(), starts.data_ptr()
    lib = _lib.load()
    with _lib.on_device(dev):
        for a, n, at, cp in _launches(counts):
            _lib.check(lib.lq_paged_append(kp + 2 * at * kt, vp + 2 * at * vt, kt, kh, vt, vh, *ptrs, P, H,
                                           HEAD_DIM, tp + 4 * a * ts, ts, width, sp + 4 * a, cp, n,
                                           _lib.raw_stream(dev)), "lq_paged_append")


def paged_gather(keys, values, table, starts, counts):
    """Positions ``starts[b] .. starts[b] + counts[b] - 1`` of each sequence as bf16 rows, packed one
    sequence behind the other: ``(k, v)``, each ``[sum(counts), Hkv, 128]``, as
    :func:`lagunalab_amd.quant.dequantize` gives them. Positions whose page does not exist read as NaN."""
    P, H, dev, ptrs = _pool(keys, values)
    B = table.shape[0]
    counts = _counts(counts, B)
    table, ts, width = _table(table, B, dev)
    starts = _ints(starts, B, "starts", dev)
    out = torch.empty((2, sum(counts), H, HEAD_DIM), dtype=torch.bfloat16, device=dev)
    k, v = out.unbind()
    kp, vp, tp, sp = k.data_ptr(), v.data_ptr(), table.data_ptr(), starts.data_ptr()
    lib = _lib.load()
    with _lib.on_device(dev):
        for a, n, at, cp in _launches(counts) if len(k) else ():
            o = 2 * at * H * HEAD_DIM
            _lib.check(lib.lq_paged_gather(*ptrs, P, H, HEAD_DIM, tp + 4 * a * ts, ts, width, sp + 4 * a, cp,
                                           n, kp + o, vp + o, _lib.raw_stream(dev)), "lq_paged_gather")
    return k, v


@functools.lru_cache(maxsize=1024)
def _decode_workspace(device, B, Hq, Hkv, pages):
    """Bytes of workspace of a decode call (of its shape alone)."""
    need = _lib.load().lq_paged_decode_workspace_bytes(B, Hq, Hkv, pages)
    if need < 0:
        _lib.check(_lib.LQ_EINVAL, "lq_paged_decode_workspace_bytes")
    return need


def paged_decode_attention(q, keys, values, table, lens, scale, shared: int = 0):
    """Attention of one new token per sequence, ``q`` bf16 ``[B, Hq, 1, 128]``, over the first ``lens[b]``
    positions of each (int32 ``[B]`` on the device); returns ``[B, Hq, 1, 128]``. ``shared``: how many
    leading positions lie in the same pages for every sequence that is that long (whole pages of it are
    used): they are read once for the batch. Length 0 gives 0; a length beyond the table's row or a page
    outside the pool gives NaN. The table and the lengths are read by the kernel: a captured call
    follows them."""
    P, H, dev, ptrs = _pool(keys, values)
    if q.dim() != 4 or q.shape[2:] != (1, HEAD_DIM) or q.dtype != torch.bfloat16:
        raise ValueError(f"q must be bfloat16 [B, Hq, 1, {HEAD_DIM}], got {tuple(q.shape)} {q.dtype}")
    _lib.require_device(q, keys[0])
    _refuse_grad(q)
    B, Hq = q.shape[:2]
    if B == 0:
        return torch.empty_like(q)
    if H < 1 or Hq % H or not 1 <= Hq // H <= 16:
        raise ValueError(f"{Hq} query heads are not 1 to 16 per KV head ({H})")
    table, ts, width = _table(table, B, dev)
    lens = _ints(lens, B, "lens", dev)
    pages = int(shared) // PAGE
    if shared < 0 or pages > width:
        raise ValueError(f"{shared} shared positions of table rows of {width} pages")
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    lib = _lib.load()
    with _lib.on_device(dev):
        need = _decode_workspace(dev.index, B, Hq, H, pages)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        out = torch.empty_like(q)
        _lib.check(lib.lq_paged_decode_attn(q.data_ptr(), *ptrs, P, B, Hq, H, HEAD_DIM, table.data_ptr(), ts,
                                            width, lens.data_ptr(), pages, scale, out.data_ptr(),
                                            ws.data_ptr(), need, _lib.raw_stream(dev)),
                   "lq_paged_decode_attn")
    return out


def copy_pages(keys, values, src, dst):
    """Copies pages within a pool: ``src[i]`` to ``dst[i]`` (host integers). A page may be copied to
    several; one that is written twice, or both read and written, is refused."""
    P, H, dev, ptrs = _pool(keys, values)
    src, dst = (array("i", x.tolist() if torch.is_tensor(x) else x) for x in (src, dst))
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} pages to copy to {len(dst)}")
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.lq_copy_pages(*ptrs, P, H, HEAD_DIM, src.buffer_info()[0], dst.buffer_info()[0],
                                     len(src), _lib.raw_stream(dev)), "lq_copy_pages")
