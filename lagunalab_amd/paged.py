"""A paged 8-bit KV cache: several sessions in one pool (no counterpart in the reference, whose caches
hold one sequence each).

A pool holds the K/V of one layer in pages of 64 positions -- for keys and for values ``(codes uint8
[pages, Hkv, 64, 128], scales bf16 [pages, Hkv, 64, 2], biases)``, every page the contiguous cache's
layout of 64 rows. Row ``b`` of a table (int32 ``[B, width]``, on the device) lists the pages of
sequence ``b`` in order; position ``p`` is slot ``p % 64`` of page ``table[b, p // 64]``.

* :func:`paged_append`, :func:`paged_gather`: rows quantized into the pages, positions read back as bf16;
* :func:`paged_append_rotated`: the same from projected rows, queries and keys normed and rotated on the way;
* :func:`paged_decode_attention`: one new token per sequence, pages that all sequences share read once;
* :func:`paged_chunk_attention`: the last rows of each sequence (a token, a verified block, a chunk), over all
  that is before them or within a window;
* :func:`copy_pages`: pages copied within the pool;
* :class:`PagedKVCache`: the pool with its page lists -- sequences opened, forked (their pages shared until
  one is written to), trimmed, closed, the pool compacted -- and :class:`PagedBatch`, some of its
  sequences behind the cache protocol of the attention block (``update_and_fetch``, ``attend``).
"""
from __future__ import annotations

import functools
import heapq
from array import array

import torch

from . import _lib
from .prompt_attn import _refuse_grad, prompt_attention

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


_CODES, _WORDS = torch.uint8, torch.bfloat16


def _pool(keys, values):
    """(pages, Hkv, device, the six buffers' pointers) of a checked pool."""
    if len(keys) != 3 or len(values) != 3:
        raise ValueError("a pool's keys and values are (codes, scales, biases)")
    codes = keys[0]
    at = codes.get_device()
    P, H = codes.shape[:2]
    wide, narrow = (P, H, PAGE, HEAD_DIM), (P, H, PAGE, HEAD_DIM // 64)
    ptrs = []
    for buf in (keys, values):
        want, dtype = wide, _CODES
        for t in buf:
            if t.shape != want or t.dtype is not dtype or not t.is_contiguous():
                raise ValueError(f"pool buffer {tuple(t.shape)} {t.dtype} is not contiguous {want} {dtype}")
            if at < 0 or t.get_device() != at:
                _lib.require_device(*keys, *values)
            ptrs.append(t.data_ptr())
            want, dtype = narrow, _WORDS
    return P, H, codes.device, ptrs


def _length(table):
    """Sequences of a table."""
    if not torch.is_tensor(table) or table.dim() != 2:
        raise ValueError("table must be an int32 tensor [sequences, pages]")
    return table.shape[0]


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


def _even(T, B):
    """As many of T rows for each of B sequences."""
    if B == 0 or T % B:
        raise ValueError(f"{T} rows are not the same number for each of {B} sequences")
    return [T // B] * B


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
    if len(counts) <= _lib.LQ_MAX_SEQS:
        return ((0, len(counts), 0, ptr),) if counts else ()
    return _many_launches(counts, ptr)


def _many_launches(counts, ptr):
    at = 0
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
    B, T = _length(table), k.shape[0]
    counts = _counts(_even(T, B) if counts is None else counts, B)
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


def _norm_weight(w, what):
    if w is None:
        return None
    if w.dtype != torch.bfloat16 or w.shape != (HEAD_DIM,):
        raise ValueError(f"{what} must be bfloat16 [{HEAD_DIM}], got {tuple(w.shape)} {w.dtype}")
    return w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)


def paged_append_rotated(q, k, v, keys, values, table, starts, rotary, counts=None, q_norm=None, k_norm=None,
                         eps=1e-6, fetch=False):
    """:func:`paged_append` of projected rows, with what a layer does to them on the way, for sequences at
    positions of their own: the heads of ``q`` (bf16 ``[T, Hq, 128]``) and ``k`` (``[T, Hkv, 128]``) get their
    RMSNorm (weights bf16 ``[128]``; None: no norm) and the rotation of their positions ``starts[b]``, ``starts[b]
    + 1``, .. (``rotary`` a :class:`lagunalab_amd.rotary.Rotary`, or None), ``v`` is stored as it is. ``q``, ``k``
    and ``v`` may be views into the rows of one projection. Returns the queries (bf16 ``[T, Hq, 128]``); with
    ``fetch`` also the new keys and values as the pages hold them, ``(q, k, v)``.

    Norm, rotation and quantization are in fp32, the angles in 64 bits, with one rounding at the end: queries to
    bf16, keys to 8 bits. (The attention block's own norm and rotation round the normed row to bf16 in between
    and take angles in fp32, off by up to 0.004 radians at 82,671 positions.)"""
    P, H, dev, ptrs = _pool(keys, values)
    B, T = _length(table), k.shape[0]
    counts = _counts(_even(T, B) if counts is None else counts, B)
    if sum(counts) != T:
        raise ValueError(f"counts add up to {sum(counts)}, not to the {T} rows")
    freq = rotary.inv_freq if rotary is not None else None
    _lib.require_device(q, k, v, keys[0], q_norm, k_norm, freq)
    _refuse_grad(q, k, v, *(w for w in (q_norm, k_norm, freq) if w is not None), what="append")
    Hq = q.shape[1] if q.dim() == 3 else -1
    q, qt, qh = _rows(q, T, Hq, "q")
    k, kt, kh = _rows(k, T, H, "k")
    v, vt, vh = _rows(v, T, H, "v")
    q_norm, k_norm = _norm_weight(q_norm, "q_norm"), _norm_weight(k_norm, "k_norm")
    rope = (None, 0, 1.0, False) if freq is None else (freq.data_ptr(), rotary.dims, rotary.mscale,
                                                       rotary.interleaved)
    table, ts, width = _table(table, B, dev)
    starts = _ints(starts, B, "starts", dev)
    out = q.new_empty((T, Hq, HEAD_DIM))
    got = q.new_empty((2, T, H, HEAD_DIM)) if fetch else None
    qp, kp, vp, op = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    gp = got.data_ptr() if fetch else None
    tp, sp = table.data_ptr(), starts.data_ptr()
    run = _lib.load().lq_paged_append_rotated
    with _lib.on_device(dev):
        for a, n, at, cp in _launches(counts):
            g = 2 * at * H * HEAD_DIM
            _lib.check(run(
                qp + 2 * at * qt, kp + 2 * at * kt, vp + 2 * at * vt, qt, qh, kt, kh, vt, vh, _lib.ptr(q_norm),
                _lib.ptr(k_norm), eps, *rope, *ptrs, P, Hq, H, HEAD_DIM, tp + 4 * a * ts, ts, width, sp + 4 * a, cp, n,
                op + 2 * at * Hq * HEAD_DIM, gp + g if fetch else None,
                gp + g + 2 * T * H * HEAD_DIM if fetch else None, _lib.raw_stream(dev)), "lq_paged_append_rotated")
    return (out, *got.unbind()) if fetch else out


def paged_gather(keys, values, table, starts, counts):
    """Positions ``starts[b] .. starts[b] + counts[b] - 1`` of each sequence as bf16 rows, packed one
    sequence behind the other: ``(k, v)``, each ``[sum(counts), Hkv, 128]``, as
    :func:`lagunalab_amd.quant.dequantize` gives them. Positions whose page does not exist read as NaN."""
    P, H, dev, ptrs = _pool(keys, values)
    B = _length(table)
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
    follows them. K and V are the rows that :func:`paged_gather` reads, rounded to bf16, and so are the
    weights (the contiguous cache's fused decode attends to the unrounded values: off by 0.0016 to 0.0018
    of the output against those, where this is by 0.0039 to 0.0045)."""
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


def paged_chunk_attention(q, keys, values, table, lens, scale, counts=None, window=None):
    """Attention of the last rows of each sequence: ``q`` bf16 ``[T, Hq, 128]`` (any token and head strides), packed
    one sequence behind the other, ``counts[b]`` rows of sequence ``b`` (host integers; None: as many each), which
    are the last of its ``lens[b]`` positions (int32 ``[B]`` on the device). A row at position ``p`` sees positions
    ``0 .. p``, or with a ``window`` the last ``window`` of them, itself among them. Returns ``[T, Hq, 128]``. Rows
    at negative positions are 0; a length beyond the table's row makes NaN of its sequence, a page outside the
    pool of the rows that see it. Pages before the window are not read. The table and the lengths are read by the
    kernel: a captured call follows them. K and V are the rows that :func:`paged_gather` reads."""
    P, H, dev, ptrs = _pool(keys, values)
    B = _length(table)
    if q.dim() != 3:
        raise ValueError(f"q must be bfloat16 [T, Hq, {HEAD_DIM}], got {tuple(q.shape)}")
    T, Hq = q.shape[:2]
    counts = _counts(_even(T, B) if counts is None else counts, B)
    if sum(counts) != T:
        raise ValueError(f"counts add up to {sum(counts)}, not to the {T} rows")
    if window is not None and window < 1:
        raise ValueError(f"a window of {window} positions")
    _lib.require_device(q, keys[0])
    _refuse_grad(q)
    q, qt, qh = _rows(q, T, Hq, "q")
    if H < 1 or Hq % H or not 1 <= Hq // H <= 64:
        raise ValueError(f"{Hq} query heads are not 1 to 64 per KV head ({H})")
    table, ts, width = _table(table, B, dev)
    lens = _ints(lens, B, "lens", dev)
    out = q.new_empty((T, Hq, HEAD_DIM))
    qp, op, tp, np = q.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr()
    seen = 0 if window is None or window >= PAGE * width else window  # as long as the table: it hides nothing
    lib = _lib.load()
    with _lib.on_device(dev):
        for a, n, at, cp in _launches(counts):
            need = lib.lq_paged_chunk_workspace_bytes(cp, n, Hq, H, width, seen)
            if need < 0:
                _lib.check(_lib.LQ_EINVAL, "lq_paged_chunk_workspace_bytes")
            ws = keys[0].new_empty(need) if need else None
            _lib.check(lib.lq_paged_chunk_attn(
                qp + 2 * at * qt, qt, qh, *ptrs, P, Hq, H, HEAD_DIM, tp + 4 * a * ts, ts, width, np + 4 * a, cp, n, seen,
                scale, op + 2 * at * Hq * HEAD_DIM, _lib.ptr(ws), need, _lib.raw_stream(dev)), "lq_paged_chunk_attn")
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


class OutOfPages(RuntimeError):
    """The pool has too few free pages for the rows; nothing was changed."""


class PagedKVCache:
    """The K/V of one layer for several sessions, in one pool of pages.

    A session (an int) is opened empty, adopted from a contiguous 8-bit cache, or forked from another,
    whose pages it then shares; a shared page is copied when one of its sessions is about to write to
    it. Pages go back to the pool when their last session is closed or trimmed below them; an append that
    raises leaves its sessions as they were. The lists live on the host; device work runs on the current
    stream, and calls on one cache belong on one stream (a page given back may be taken by the next
    call), outside of captured graphs: a replay would repeat the recorded step on the recorded rows
    (:func:`paged_append` and :func:`paged_decode_attention` can be captured)."""

    def __init__(self, pages: int, n_kv_heads: int, device="cuda"):
        self.keys, self.values = page_pool(pages, n_kv_heads, device)
        self._free = list(range(pages))  # a heap: the lowest page first
        self._uses = [0] * pages
        self._sessions: dict[int, list] = {}  # session -> [its pages, its rows]
        self._next = 0
        self._version = 0  # of the page lists: batches rebuild their tables when it moves

    # ---- sessions

    def open(self) -> int:
        """A new, empty session."""
        self._sessions[self._next] = [[], 0]
        self._next += 1
        return self._next - 1

    def fork(self, session: int) -> int:
        """A session that begins as ``session`` is now, sharing its pages."""
        pages, rows = self._session(session)
        new = self.open()
        self._sessions[new] = [list(pages), rows]
        for p in pages:
            self._uses[p] += 1
        return new

    def adopt(self, cache) -> int:
        """A session of the rows of a contiguous 8-bit cache of one sequence (a ``DequantKVCache`` or
        ``QuantizedKVCache`` of group 64, loaded from a prompt cache for instance): its codes, scales and
        biases are copied as they are."""
        self._outside_graphs()
        keys, values = cache.state
        if keys is None:
            return self.open()
        H = self.keys[0].shape[1]
        n = keys[0].shape[2]
        for t in (keys[0], values[0]):
            if t.dtype != torch.uint8 or t.shape != (1, H, n, HEAD_DIM):
                raise ValueError(f"codes {tuple(t.shape)} {t.dtype} are not those of one sequence of "
                                 f"{H} heads in 8 bits")
        for t in (*keys[1:], *values[1:]):
            if t.shape != (1, H, n, HEAD_DIM // 64) or t.dtype != torch.bfloat16:
                raise ValueError(f"scales or biases {tuple(t.shape)} {t.dtype} are not bfloat16 of groups of 64")
        _lib.require_device(*keys, *values, *self.keys)
        pages = self._take(-(-n // PAGE))
        whole = n // PAGE
        try:
            at = torch.tensor(pages, device=self.keys[0].device)
            for buf, rows in ((self.keys, keys), (self.values, values)):
                for t, x in zip(buf, rows):
                    if whole:
                        t[at[:whole]] = x[0, :, :whole * PAGE].unflatten(1, (whole, PAGE)).transpose(0, 1)
                    if n % PAGE:
                        t[pages[-1], :, :n % PAGE] = x[0, :, whole * PAGE:]
        except BaseException:
            self._give(pages)
            raise
        new = self.open()
        self._sessions[new] = [pages, n]
        return new

    def close(self, session: int):
        """Ends a session and gives its pages back."""
        pages, _ = self._session(session)
        self._give(pages)
        del self._sessions[session]
        self._version += 1

    def trim(self, session: int, n: int) -> int:
        """Drops the last ``n`` rows of a session (rejected drafts); returns how many it had to drop."""
        s = self._session(session)
        n = min(s[1], int(n))
        if n < 0:
            raise ValueError(f"cannot trim {n} rows")
        s[1] -= n
        keep = -(-s[1] // PAGE)
        self._give(s[0][keep:])
        del s[0][keep:]
        self._version += 1
        return n

    def length(self, session: int) -> int:
        return self._session(session)[1]

    def pages(self, session: int) -> list:
        """The session's pages, in order."""
        return list(self._session(session)[0])

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (*self.keys, *self.values))

    def _outside_graphs(self):
        if _lib.capturing(self.keys[0].device):
            raise RuntimeError("sessions move on the host: calls on them cannot be captured into a graph")

    def _session(self, session):
        if session not in self._sessions:
            raise ValueError(f"there is no session {session}")
        return self._sessions[session]

    def _take(self, n):
        if n > len(self._free):
            raise OutOfPages(f"{n} pages are needed, {len(self._free)} of {len(self._uses)} are free")
        got = [heapq.heappop(self._free) for _ in range(n)]
        for p in got:
            self._uses[p] = 1
        return got

    def _give(self, pages):
        for p in pages:
            self._uses[p] -= 1
            if self._uses[p] == 0:
                heapq.heappush(self._free, p)

    def _distinct(self, sessions):
        sessions = list(sessions)
        if len(set(sessions)) != len(sessions):
            raise ValueError(f"a session is listed twice in {sessions}")
        return sessions, [self._session(s) for s in sessions]

    # ---- rows

    def _make_room(self, states, counts):
        """Pages for ``counts`` more rows of each session, written-to pages its own; returns whether a
        page list changed. All or nothing."""
        written = {}  # last pages about to be written to -> their writers so far
        copies, fresh = [], 0
        for (pages, rows), c in zip(states, counts):
            if c and rows % PAGE:
                p = pages[rows // PAGE]
                written[p] = written.get(p, 0) + 1
                if written[p] < self._uses[p]:  # someone keeps it: another session, or a later writer
                    copies.append((pages, rows // PAGE, p))
            if c:
                fresh += max(0, -(-(rows + c) // PAGE) - len(pages))
        new = self._take(len(copies) + fresh)
        if copies:
            dst = new[:len(copies)]
            try:
                copy_pages(self.keys, self.values, [p for _, _, p in copies], dst)
            except BaseException:
                self._give(new)
                raise
            for (pages, i, p), q in zip(copies, dst):
                pages[i] = q
                self._uses[p] -= 1
        at = len(copies)
        for (pages, rows), c in zip(states, counts):
            if c:
                n = max(0, -(-(rows + c) // PAGE) - len(pages))
                pages.extend(new[at:at + n])
                at += n
        return bool(new)

    def _undo_room(self, states):
        """After rows that were not appended: the pages made for them go back (a page copied for its
        writer stays its own)."""
        for pages, rows in states:
            keep = -(-rows // PAGE)
            self._give(pages[keep:])
            del pages[keep:]
        self._version += 1

    def _tables(self, states):
        """(table, lens) of the sessions on the device."""
        if not states:
            empty = torch.zeros((0, 1), dtype=torch.int32, device=self.keys[0].device)
            return empty, empty[:, 0]
        width = max([1] + [len(pages) for pages, _ in states])
        flat = array("i", [0]) * (width * len(states))
        for i, (pages, _) in enumerate(states):
            flat[i * width:i * width + len(pages)] = array("i", pages)
        dev = self.keys[0].device
        table = torch.frombuffer(flat, dtype=torch.int32).to(dev).view(len(states), width)
        return table, torch.tensor([rows for _, rows in states], dtype=torch.int32).to(dev)

    @staticmethod
    def _common(states):
        """Leading positions that lie in the same pages for all sessions (whole pages)."""
        if len(states) < 2:
            return 0
        n = min(rows // PAGE for _, rows in states)
        first = states[0][0]
        for pages, _ in states[1:]:
            if pages[:n] != first[:n]:
                n = next(i for i in range(n) if pages[i] != first[i])
        return n * PAGE

    def _new_rows(self, states, k, v, counts):
        """Host counts of checked rows."""
        T = k.shape[0]
        if counts is None:
            if T % len(states):
                raise ValueError(f"{T} rows are not the same number for each of {len(states)} sessions")
            counts = [T // len(states)] * len(states)
        counts = _counts(counts, len(states)).tolist()
        H = self.keys[0].shape[1]
        if sum(counts) != T or k.shape != (T, H, HEAD_DIM) or v.shape != k.shape:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} are not {sum(counts)} rows of {H} heads")
        if not k.dtype == v.dtype == torch.bfloat16:
            raise ValueError(f"K/V rows must be bfloat16, got {k.dtype} and {v.dtype}")
        _lib.require_device(k, v, self.keys[0])
        return counts

    def _write(self, states, counts, write):
        """What ``write(table, starts)`` gives, which stores ``counts`` new rows of the sessions."""
        self._make_room(states, counts)
        self._version += 1
        try:
            got = write(*self._tables(states))
        except BaseException:
            self._undo_room(states)
            raise
        for s, c in zip(states, counts):
            s[1] += c
        return got

    def append(self, sessions, k, v, counts=None):
        """Appends rows ``k``, ``v`` (bf16 ``[T, Hkv, 128]``, packed one session behind the other,
        ``counts[i]`` each or as many each) to the sessions."""
        self._outside_graphs()
        sessions, states = self._distinct(sessions)
        if not states:
            return
        counts = self._new_rows(states, k, v, counts)
        self._write(states, counts, lambda table, starts: paged_append(k, v, self.keys, self.values, table, starts,
                                                                       counts))

    def append_rotated(self, sessions, q, k, v, rotary, counts=None, q_norm=None, k_norm=None, eps=1e-6, fetch=False):
        """:meth:`append` of projected rows: their heads get norm and rotation at their sessions' positions on the
        way (:func:`paged_append_rotated`). Returns the queries (bf16 ``[T, Hq, 128]``); with ``fetch`` ``(q, k, v)``."""
        self._outside_graphs()
        sessions, states = self._distinct(sessions)
        if not states:
            raise ValueError("no sessions")
        counts = self._new_rows(states, k, v, counts)
        return self._write(states, counts, lambda table, starts: paged_append_rotated(
            q, k, v, self.keys, self.values, table, starts, rotary, counts, q_norm, k_norm, eps, fetch))

    def rows(self, sessions):
        """All rows of the sessions as bf16, packed: ``(k, v)``, each ``[sum of lengths, Hkv, 128]``."""
        self._outside_graphs()
        _, states = self._distinct(sessions)
        table, lens = self._tables(states)
        return paged_gather(self.keys, self.values, table, torch.zeros_like(lens), [n for _, n in states])

    def attention(self, sessions, q, scale):
        """Attention of one new token per session over its rows: ``q`` bf16 ``[B, Hq, 1, 128]``."""
        self._outside_graphs()
        _, states = self._distinct(sessions)
        table, lens = self._tables(states)
        return paged_decode_attention(q, self.keys, self.values, table, lens, scale,
                                      shared=self._common(states))

    def chunk_attention(self, sessions, q, scale, counts=None, window=None):
        """Attention of the last rows of each session, ``q`` bf16 ``[T, Hq, 128]`` packed one session behind the
        other, ``counts[i]`` each or as many each, over all before them or a window (:func:`paged_chunk_attention`)."""
        self._outside_graphs()
        sessions, states = self._distinct(sessions)
        counts = _counts(_even(q.shape[0], len(states)) if counts is None else counts, len(states)).tolist()
        for s, (_, rows), c in zip(sessions, states, counts):
            if rows < c:
                raise ValueError(f"session {s} of {rows} rows is shorter than its {c} queries")
        table, lens = self._tables(states)
        return paged_chunk_attention(q, self.keys, self.values, table, lens, scale, counts, window)

    def batch(self, sessions, window=None, rotates=False) -> "PagedBatch":
        """The sessions as the cache of a model call with one row of the batch for each. ``window``: of a
        sliding-window layer, whose rows see that many positions, themselves among them. ``rotates``: the attention
        block leaves norm and rotation to the append, and the sessions may be of different lengths."""
        return PagedBatch(self, sessions, window, rotates)

    # ---- pages

    def compact(self) -> int:
        """Moves pages in use to the front of the pool; returns how many there are."""
        self._outside_graphs()
        live = [p for p, n in enumerate(self._uses) if n]
        n = len(live)
        holes = [p for p in range(n) if not self._uses[p]]
        moved = dict(zip(live[n - len(holes):], holes))
        if moved:
            copy_pages(self.keys, self.values, list(moved), list(moved.values()))
            for s in self._sessions.values():
                s[0][:] = [moved.get(p, p) for p in s[0]]
            for p, q in moved.items():
                self._uses[q], self._uses[p] = self._uses[p], 0
            self._free = list(range(n, len(self._uses)))
            self._version += 1
        return n

    def resize(self, pages: int):
        """A pool of ``pages`` pages: compacted, then copied into new buffers."""
        self._outside_graphs()
        used = len(self._uses) - len(self._free)
        if pages < max(used, 1):
            raise ValueError(f"{used} pages are in use: the pool cannot have {pages}")
        self.compact()
        keys, values = page_pool(pages, self.keys[0].shape[1], self.keys[0].device)
        for t, x in zip((*keys, *values), (*self.keys, *self.values)):
            t[:used] = x[:used]
        self.keys, self.values = keys, values
        self._uses = self._uses[:used] + [0] * (pages - used)
        self._free = list(range(used, pages))
        self._version += 1


class PagedBatch:
    """Sessions of a :class:`PagedKVCache` behind the cache protocol of the attention block
    (``update_and_fetch`` -> ``fused_step`` -> ``attend``; ``laguna_mlx/laguna.py:94-111``), row ``b`` of a
    call being session ``b``. Steps of one row run :func:`paged_decode_attention`, the pages that all
    sessions share read once; longer ones (prompts, chunks) read the sessions' rows back and run
    :func:`lagunalab_amd.prompt_attn.prompt_attention`, causal. What is attended are the quantized rows,
    as with ``DequantKVCache``. ``offset`` needs sessions of one length (the block's rotary embedding has
    one position per call); the layers are full-attention ones (:meth:`make_mask`).

    With a ``window`` the layers are sliding-window ones: every step runs :func:`paged_chunk_attention`. With
    ``rotates`` the block hands its projections to :meth:`append_rotated`, each session is at a position of its own,
    and steps of more than one row run :func:`paged_chunk_attention` too, which copies nothing."""

    fused_step = True

    def __init__(self, cache: PagedKVCache, sessions, window=None, rotates=False):
        if window is not None and window < 1:
            raise ValueError(f"a window of {window} positions")
        self.cache = cache
        self.sessions, _ = cache._distinct(sessions)
        self.window, self.rotates = window, bool(rotates)
        self._seen = -1

    def _states(self):
        return [self.cache._session(s) for s in self.sessions]

    def _refresh(self, states):
        if self._seen != self.cache._version:
            self._table, self._lens = self.cache._tables(states)
            self._shared = self.cache._common(states)
            self._seen = self.cache._version

    def update_and_fetch(self, keys, values):
        """Appends ``keys``, ``values`` (bf16 ``[B, Hkv, L, 128]``) to the sessions; returns them (attention
        goes through :meth:`attend`)."""
        self.cache._outside_graphs()
        B, H, L, D = keys.shape
        if B != len(self.sessions) or (H, D) != (self.cache.keys[0].shape[1], HEAD_DIM) \
                or values.shape != keys.shape:
            raise ValueError(f"keys {tuple(keys.shape)} and values {tuple(values.shape)} are not rows of "
                             f"{len(self.sessions)} sessions of {self.cache.keys[0].shape[1]} heads")
        if not keys.dtype == values.dtype == torch.bfloat16:
            raise ValueError(f"K/V rows must be bfloat16, got {keys.dtype} and {values.dtype}")
        _lib.require_device(keys, values, self.cache.keys[0])
        k, v = (t.transpose(1, 2).reshape(B * L, H, D) for t in (keys, values))
        self._write(L, lambda: paged_append(k, v, self.cache.keys, self.cache.values, self._table, self._lens, [L] * B))
        return keys, values

    def append_rotated(self, queries, keys, values, rotary, q_norm=None, k_norm=None, eps=1e-6):
        """Appends projected rows (bf16 ``[B, L, heads, 128]``, any strides) to the sessions, queries and keys normed
        and rotated at each session's positions on the way (:func:`paged_append_rotated`); returns the queries
        ``[B, Hq, L, 128]`` for :meth:`attend`."""
        self.cache._outside_graphs()
        B, L, H, D = keys.shape
        if B != len(self.sessions) or (H, D) != (self.cache.keys[0].shape[1], HEAD_DIM) \
                or values.shape != keys.shape or queries.shape[:2] != (B, L):
            raise ValueError(f"queries {tuple(queries.shape)}, keys {tuple(keys.shape)} and values "
                             f"{tuple(values.shape)} are not rows of {len(self.sessions)} sessions of "
                             f"{self.cache.keys[0].shape[1]} heads")
        if not queries.dtype == keys.dtype == values.dtype == torch.bfloat16:
            raise ValueError(f"rows must be bfloat16, got {queries.dtype}, {keys.dtype} and {values.dtype}")
        _lib.require_device(queries, keys, values, self.cache.keys[0])
        q, k, v = (t.flatten(0, 1) for t in (queries, keys, values))
        got = self._write(L, lambda: paged_append_rotated(
            q, k, v, self.cache.keys, self.cache.values, self._table, self._lens, rotary, [L] * B, q_norm, k_norm, eps))
        return got.view(queries.shape).transpose(1, 2)

    def _write(self, L, write):
        """What ``write()`` gives, which stores L new rows of each session."""
        states = self._states()
        if self.cache._make_room(states, [L] * len(states)):
            self.cache._version += 1
        try:
            self._refresh(states)
            got = write()
            lens = self._lens + L
        except BaseException:
            self.cache._undo_room(states)
            raise
        for s in states:
            s[1] += L
        self._lens = lens
        self.cache._version += 1  # other batches of these sessions hold old lengths
        self._seen = self.cache._version
        return got

    def attend(self, queries, scale):
        """Attention of the step's rows, ``queries`` bf16 ``[B, Hq, L, 128]``: the last ``L`` positions of
        each session, causal, within the window."""
        self.cache._outside_graphs()
        B, Hq, L, D = queries.shape
        if B != len(self.sessions):
            raise ValueError(f"{B} rows of queries for {len(self.sessions)} sessions")
        states = self._states()
        if any(n < L for _, n in states):
            raise ValueError(f"sessions shorter than the step of {L} rows")
        self._refresh(states)
        q = queries.to(torch.bfloat16)
        keys, values = self.cache.keys, self.cache.values
        # single tokens by the decode kernels, which take up to 16 query heads per KV head
        if self.window is not None or (self.rotates and (L > 1 or Hq > 16 * keys[0].shape[1])):
            out = paged_chunk_attention(q.transpose(1, 2).reshape(B * L, Hq, D), keys, values, self._table, self._lens,
                                        scale, [L] * B, self.window)
            out = out.view(B, L, Hq, D).transpose(1, 2)
        elif L == 1:
            out = paged_decode_attention(q, keys, values, self._table, self._lens, scale, shared=self._shared)
        else:
            lens = [n for _, n in states]
            k, v = paged_gather(keys, values, self._table, torch.zeros_like(self._lens), lens)
            out = prompt_attention(q.transpose(1, 2).reshape(B * L, Hq, D), k, v, [L] * B, scale, k_lens=lens)
            out = out.view(B, L, Hq, D).transpose(1, 2)
        return out.to(queries.dtype)

    @property
    def offset(self) -> int:
        lens = {n for _, n in self._states()}
        if len(lens) > 1:
            raise ValueError(f"sessions of different lengths {sorted(lens)} have no common offset")
        return lens.pop() if lens else 0

    def make_mask(self, N, return_array=False, window_size=None):
        """The mask of a step of ``N`` rows. :meth:`attend` is causal over all rows, or those of the batch's
        window, whatever the mask: another window is refused, unless neither leaves out any of the rows. Sessions of
        different lengths have no array for a mask: "causal" stands for it, of a single row None."""
        from .cache import create_attention_mask
        lens = [n for _, n in self._states()] if self.rotates else [self.offset]
        rows = max(lens, default=0) + N
        if min(rows, rows if window_size is None else window_size) != min(rows, self.window or rows):
            if self.window is not None:
                raise ValueError(f"the batch has a window of {self.window} positions, its layer one of {window_size}")
            raise ValueError(f"a window of {window_size} positions ends before the {rows} rows: paged "
                             "batches are for full-attention layers")
        if self.rotates and not return_array:
            return None if N == 1 else "causal"
        return create_attention_mask(N, offset=self.offset, return_array=return_array, window_size=window_size)

    def is_trimmable(self):
        return True

    def trim(self, n):
        """Drops the last ``n`` rows of every session (at most as many as the shortest has)."""
        n = min([int(n)] + [rows for _, rows in self._states()])
        for s in self.sessions:
            self.cache.trim(s, n)
        return n

    def empty(self):
        return all(n == 0 for _, n in self._states())

    @property
    def nbytes(self):
        """Bytes of the pages that the sessions use, shared ones once."""
        per_page = self.cache.nbytes // len(self.cache._uses)
        return per_page * len({p for pages, _ in self._states() for p in pages})
