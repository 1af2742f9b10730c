"""Attention of the last rows of sequences over a paged cache (``paged_chunk_attention``) against attention in 64
bits over the rows that the pages hold: layouts, counts, lengths and windows where blocks, tiles and parts begin
and end; what masked positions, free slots and other sequences' pages hold; captured calls, streams, refusals."""
import ctypes as C

import pytest
import torch

from lagunalab_amd import _lib, paged
from lagunalab_amd.paged import paged_append, paged_chunk_attention, paged_gather
from paged_util import D, PAGE, fill_pool, make_table, randn, write_rows

pytestmark = pytest.mark.gpu
SCALE = D ** -0.5


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def held(buf, ids, n):
    """The first n positions of a sequence (pages ids) as bf16 holds them, in 64 bits [n, Hkv, 128], on the pool's
    device."""
    at = torch.arange(n, device=buf[0].device)
    pages, slots = ids.to(at.device).long()[at // PAGE], at % PAGE
    c, s, b = (t[pages, :, slots] for t in buf)
    s, b = (x.double().repeat_interleave(64, dim=-1) for x in (s, b))
    return (c.double() * s + b).to(torch.bfloat16).double()


def exact(q, pool, table, lens, counts, window, scale):
    """(out, bound) of packed rows q, in 64 bits on the pool's device. The bound: weights rounded to bf16 (2^-8
    each, in the weighted values and in their sum), the output too, scores summed in fp32 (128 2^-24 of the
    products' magnitudes, through the exponential in weights and sum; the hardware's exp2 and the sums over keys
    are within the factor)."""
    hq, kv = q.shape[1], pool[0][0].shape[1]
    G, a = hq // kv, 0
    q = q.double()
    out, bound = torch.zeros_like(q), torch.full_like(q, 1e-30)
    for b, (n, c) in enumerate(zip(lens, counts)):
        if c and n:
            k, v = (held(buf, table[b], n) for buf in pool)
            p = torch.arange(n - c, n, device=q.device)[:, None]
            j = torch.arange(n, device=q.device)
            seen = (j <= p) & (j > p - (window or 1 << 40))
            none = ~seen.any(1)
            seen = seen.repeat_interleave(G, 0)
            for h in range(kv):
                x = q[a:a + c, h * G:(h + 1) * G].reshape(c * G, D)
                kh, vh = k[:, h].contiguous(), v[:, h].contiguous()
                s = (x @ kh.t().contiguous() * scale).masked_fill(~seen, float("-inf"))
                w = torch.softmax(s, 1).nan_to_num(0.0)
                o, size = w @ vh, w @ vh.abs()
                mag = (x.abs() @ kh.abs().t().contiguous() * abs(scale)).masked_fill(~seen, 0).amax(1, keepdim=True)
                slack = 2 * 2.0 ** -8 + 4 * (128 * 2.0 ** -24 * mag + 2.0 ** -18)
                out[a:a + c, h * G:(h + 1) * G] = o.view(c, G, D)
                bound[a:a + c, h * G:(h + 1) * G] = (size * slack + o.abs() * 2.0 ** -8 + 1e-30).view(c, G, D)
            out[a:a + c][none] = 0
        a += c
    return out, bound


def assert_within(got, want, bound, what=""):
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = ((got.double() - want).abs() / bound).max().item() if got.numel() else 0.0
    assert off <= 1.0, f"{what}: {off:.3f} times the bound"


def sessions(g, kv, lens, dev, kstd=1.0, vstd=1.0, spare=0):
    """A pool whose used slots hold quantized rows, all others NaN scales and biases; its table."""
    table, pages = make_table(g, lens, 0, width_spare=spare)
    pool = fill_pool(g, pages, kv, dev)
    for b, n in enumerate(lens):
        if n:
            write_rows(pool, table[b], randn(g, n, kv, D, std=kstd), randn(g, n, kv, D, std=vstd))
    return pool, table


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def check(dev, hq, kv, lens, counts, window, scale=SCALE, qstd=1.0, what="", **kw):
    g = gen(1000 * hq + sum(lens) + sum(counts))
    pool, table = sessions(g, kv, lens, dev, **kw)
    q = randn(g, sum(counts), hq, D, std=qstd).to(dev)
    got = paged_chunk_attention(q, *pool, table.to(dev), ints(lens, dev), scale, counts, window=window)
    assert_within(got, *exact(q, pool, table, lens, counts, window, scale), what)


@pytest.mark.parametrize("window", [None, 1, 63, 64, 65, 200])
@pytest.mark.parametrize("hq,kv", [(32, 8), (6, 1), (3, 3), (48, 8), (64, 1), (10, 2)])
def test_chunks_of_any_place(dev, hq, kv, window):
    """Ends and starts in, at and around pages; nothing new, one row, blocks; all that there is, less, more."""
    for lens, counts in (([1], [1]), ([64, 65, 63, 128], [1, 1, 1, 1]), ([5, 0, 64, 200, 129], [5, 0, 64, 2, 66]),
                         ([300, 131, 1, 257], [17, 0, 1, 130]), ([700], [333]), ([90, 3, 64], [100, 5, 65])):
        check(dev, hq, kv, lens, counts, window, what=f"{lens} {counts}")


@pytest.mark.parametrize("hq,kv,lens,counts,window", [
    (32, 8, [5005], [5], None), (48, 8, [4099], [8], None), (48, 8, [20011, 300, 7], [8, 3, 7], None),
    (32, 8, [9000], [512], None), (48, 8, [3000], [1031], 512), (16, 2, [2500, 2500], [700, 64], None),
    (8, 8, [6000], [1], 512), (64, 8, [700] * 40, [3] * 40, None), (48, 8, [64 * i + i for i in range(64)], [1] * 64, 512),
    (32, 8, list(range(0, 4000, 61))[:64], list(range(64)), 300), (32, 8, [4099], [4099], None),
    (4, 4, [30000], [2], 29000), (128, 2, [1500, 90], [9, 90], None),
])
def test_long_chunks(dev, hq, kv, lens, counts, window):
    counts = [min(n, c) for n, c in zip(lens, counts)]
    check(dev, hq, kv, lens, counts, window)


@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("counts", [[1, 3, 2], [70, 1, 40]])
@pytest.mark.parametrize("scale,qstd,kstd,vstd", [(-SCALE, 1, 1, 1), (0.0, 1, 1, 1), (1.0, 1, 1, 1), (SCALE, 30, 1, 1),
                                                  (SCALE, 1, 1, 1e-6), (SCALE, 1e4, 1e4, 1), (SCALE, 1, 1, 1e30)])
def test_scales(dev, scale, qstd, kstd, vstd, counts, window):
    check(dev, 12, 2, [400, 77, 130], counts, window, scale, qstd=qstd, kstd=kstd, vstd=vstd)


def test_rows_of_a_projection_and_more_sequences_than_a_launch(dev):
    g = gen(5)
    lens = [3 + 7 * i for i in range(100)]
    counts = [i % 4 for i in range(100)]
    pool, table = sessions(g, 2, lens, dev)
    wide = randn(g, sum(counts), 12 * D + 24).to(dev)
    q = wide[:, 2 * D:10 * D].unflatten(1, (8, D))
    got = paged_chunk_attention(q, *pool, table.to(dev), ints(lens, dev), SCALE, counts)
    assert_within(got, *exact(q, pool, table, lens, counts, None, SCALE), "strided")
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(paged_chunk_attention(heads_first, *pool, table.to(dev), ints(lens, dev), SCALE, counts), got)
    odd = torch.cat([wide[:, :1], wide], 1)[:, 1:][:, 2 * D:10 * D].unflatten(1, (8, D))  # 2-byte aligned rows
    assert torch.equal(paged_chunk_attention(odd, *pool, table.to(dev), ints(lens, dev), SCALE, counts), got)


def test_as_many_rows_each_without_counts(dev):
    g = gen(6)
    lens = [70, 9, 300]
    pool, table = sessions(g, 2, lens, dev)
    q = randn(g, 6, 4, D).to(dev)
    args = (*pool, table.to(dev), ints(lens, dev), SCALE)
    assert torch.equal(paged_chunk_attention(q, *args), paged_chunk_attention(q, *args, [2, 2, 2]))
    none = paged_chunk_attention(q[:0], *args, [0, 0, 0], window=5)
    assert none.shape == (0, 4, D)


@pytest.mark.parametrize("counts", [[1, 1], [6, 1], [150, 90]])
def test_rows_before_the_first_position_are_zero(dev, counts):
    g = gen(7)
    lens = [n // 2 for n in counts]
    pool, table = sessions(g, 2, [max(1, n) for n in lens], dev)
    q = randn(g, sum(counts), 4, D).to(dev)
    got = paged_chunk_attention(q, *pool, table.to(dev), ints(lens, dev), SCALE, counts)
    assert_within(got, *exact(q, pool, table, lens, counts, None, SCALE))
    at = 0
    for n, c in zip(lens, counts):
        assert (got[at:at + c - n] == 0).all()
        at += c


@pytest.mark.parametrize("window", [None, 70])
@pytest.mark.parametrize("counts", [[2, 4], [90, 130], [3, 130]])
@pytest.mark.parametrize("what", ["k nan", "k inf", "v nan", "v inf"])
def test_positions_that_a_row_does_not_see_do_not_reach_it(dev, what, counts, window):
    """A row of the pool that is not finite, at a position that some rows of the block see and others do not."""
    g = gen(8)
    lens = [201, 330]
    pool, table = sessions(g, 2, lens, dev)
    hq = 6
    q = randn(g, sum(counts), hq, D).to(dev)
    args = (table.to(dev), ints(lens, dev), SCALE, counts)
    clean = paged_chunk_attention(q, *pool, *args, window=window)
    for b, at in ((0, lens[0] - 1), (1, lens[1] - counts[1] // 2), (1, lens[1] - counts[1] - 60)):
        spoiled = [tuple(t.clone() for t in buf) for buf in pool]
        page, slot = int(table[b, at // PAGE]), at % PAGE
        spoiled[what[0] == "v"][1][page, 1, slot, 1] = float(what[2:])  # a group of the second head
        got = paged_chunk_attention(q, *spoiled, *args, window=window)
        first = sum(counts[:b]) + at - (lens[b] - counts[b])  # the first row that sees it
        last = sum(counts[:b + 1]) if window is None else min(sum(counts[:b + 1]), first + window)
        first = max(first, sum(counts[:b]))
        sees = torch.zeros(len(q), dtype=torch.bool, device=dev)
        sees[first:max(first, last)] = True
        assert torch.equal(got[~sees], clean[~sees]), (b, at)
        assert torch.equal(got[sees][:, :hq // 2], clean[sees][:, :hq // 2])  # the other head
        if what[0] == "v":
            assert torch.equal(got[sees][:, hq // 2:, :64], clean[sees][:, hq // 2:, :64])  # the other group
            assert not torch.isfinite(got[sees][:, hq // 2:, 64:]).any()
        else:
            assert not torch.isfinite(got[sees][:, hq // 2:]).any()


@pytest.mark.parametrize("counts", [[1, 2, 1], [50, 70, 5], [300, 2, 1]])
def test_bad_lengths_and_pages(dev, counts):
    g = gen(9)
    lens = [310, 400, 130]
    pool, table = sessions(g, 2, lens, dev)
    q = randn(g, sum(counts), 8, D).to(dev)
    clean = paged_chunk_attention(q, *pool, table.to(dev), ints(lens, dev), SCALE, counts)
    ends = [sum(counts[:i + 1]) for i in range(3)]
    for n in (-1, PAGE * table.shape[1] + 1, -2 ** 31, 2 ** 31 - 1):
        got = paged_chunk_attention(q, *pool, table.to(dev), ints([lens[0], n, lens[2]], dev), SCALE, counts)
        assert torch.isnan(got[ends[0]:ends[1]]).all()
        assert torch.equal(got[:ends[0]], clean[:ends[0]]) and torch.equal(got[ends[1]:], clean[ends[1]:])
    for bad in (-1, pool[0][0].shape[0], 2 ** 31 - 1):
        spoiled = table.clone()
        spoiled[0, 2] = bad  # positions 128 .. 191
        got = paged_chunk_attention(q, *pool, spoiled.to(dev), ints(lens, dev), SCALE, counts)
        see = max(0, 128 - (lens[0] - counts[0]))  # the first row that does
        assert torch.isnan(got[see:ends[0]]).all()
        assert torch.equal(got[:see], clean[:see]) and torch.equal(got[ends[0]:], clean[ends[0]:])
        # pages wholly before the window are not looked at
        got = paged_chunk_attention(q, *pool, spoiled.to(dev), ints([310, 400, 130], dev), SCALE, counts, window=30)
        ok = paged_chunk_attention(q, *pool, table.to(dev), ints([310, 400, 130], dev), SCALE, counts, window=30)
        hidden = [i for i in range(ends[0]) if lens[0] - counts[0] + i - 29 > 191 or lens[0] - counts[0] + i < 128]
        assert torch.equal(got[hidden], ok[hidden]) and torch.equal(got[ends[0]:], ok[ends[0]:])


@pytest.mark.parametrize("counts,window", [([1, 1, 1], 100), ([5, 2, 9], None), ([120, 1, 60], None), ([70, 80, 3], 33)])
def test_captured_calls_follow_lengths_and_tables(dev, counts, window):
    g = gen(10)
    lens = [700, 300, 1100]
    pool, table = sessions(g, 2, lens, dev)
    q = randn(g, sum(counts), 12, D).to(dev)
    q_in, t_in, n_in = q.clone(), table.to(dev), ints(lens, dev)
    out = paged_chunk_attention(q_in, *pool, t_in, n_in, SCALE, counts, window=window)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_chunk_attention(q_in, *pool, t_in, n_in, SCALE, counts, window=window)
    order = torch.tensor([1, 2, 0])
    for step in range(4):
        now = [max(0, n - 97 * step) for n in (lens if step % 2 == 0 else [lens[i] for i in order])]
        rows = table if step % 2 == 0 else table[order]
        q_in.copy_(q.flip(0) if step == 3 else q)
        t_in.copy_(rows)
        n_in.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        want = paged_chunk_attention(q_in, *pool, t_in, n_in, SCALE, counts, window=window)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert_within(out, *exact(q_in, pool, rows, now, counts, window, SCALE), f"step {step}")


def test_two_streams_at_once(dev):
    g = gen(11)
    lens, counts = [5000, 2000], [3, 200]
    pool, table = sessions(g, 8, lens, dev)
    qs = [randn(g, 203, 32, D).to(dev) for _ in range(2)]
    args = (*pool, table.to(dev), ints(lens, dev), SCALE, counts)
    want = [paged_chunk_attention(q, *args) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(paged_chunk_attention(qs[i], *args))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_the_same_every_time(dev):
    g = gen(12)
    lens, counts = [5000, 900, 64, 3000], [16, 300, 1, 5]
    pool, table = sessions(g, 8, lens, dev)
    q = randn(g, sum(counts), 48, D).to(dev)
    args = (*pool, table.to(dev), ints(lens, dev), SCALE, counts)
    first = paged_chunk_attention(q, *args)
    for _ in range(5):
        assert torch.equal(paged_chunk_attention(q, *args), first)


def test_pages_beyond_32_bit_offsets(dev):
    pages, kv = 67000, 8
    pool = [(torch.empty((pages, kv, PAGE, D), dtype=torch.uint8, device=dev),
             torch.empty((pages, kv, PAGE, 2), dtype=torch.bfloat16, device=dev),
             torch.empty((pages, kv, PAGE, 2), dtype=torch.bfloat16, device=dev)) for _ in range(2)]
    g = gen(13)
    lens = [300, 120, 500]
    table = torch.zeros((3, 8), dtype=torch.int32)
    table[0, :5] = torch.arange(66990, 66995)
    table[1, :2] = torch.tensor([3, 66999])
    table[2] = torch.arange(66000, 66800, 100)
    for b, n in enumerate(lens):
        write_rows(pool, table[b], randn(g, n, kv, D), randn(g, n, kv, D))
    for counts in ([1, 2, 1], [40, 100, 3]):
        q = randn(g, sum(counts), 32, D).to(dev)
        got = paged_chunk_attention(q, *pool, table.to(dev), ints(lens, dev), SCALE, counts)
        assert_within(got, *exact(q, pool, table, lens, counts, None, SCALE))


def test_nothing_behind_the_outputs_is_touched(dev):
    """The C entry on buffers with room behind them: outputs, and a workspace of exactly the bytes asked for."""
    g = gen(14)
    lib = _lib.load()
    for lens, counts, hq in (([300, 70], [3, 1], 4), ([900, 70], [200, 61], 12)):
        kv, T = 2, sum(counts)
        pool, table = sessions(g, kv, lens, dev)
        q = randn(g, T, hq, D).to(dev)
        cn = (C.c_int32 * len(counts))(*counts)
        need = lib.lq_paged_chunk_workspace_bytes(cn, len(counts), hq, kv, table.shape[1], 0)
        ws = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=dev)
        out = torch.full((T + 8, hq, D), 7.0, dtype=torch.bfloat16, device=dev)
        t_d, n_d = table.to(dev), ints(lens, dev)
        _lib.check(lib.lq_paged_chunk_attn(
            q.data_ptr(), hq * D, D, *(t.data_ptr() for buf in pool for t in buf), pool[0][0].shape[0], hq, kv, D,
            t_d.data_ptr(), t_d.stride(0), t_d.shape[1], n_d.data_ptr(), cn, len(counts), 0, SCALE, out.data_ptr(),
            ws.data_ptr(), need, _lib.raw_stream(dev)), "lq_paged_chunk_attn")
        assert (out[T:] == 7.0).all() and (ws[need:] == 0xA5).all()
        assert_within(out[:T], *exact(q, pool, table, lens, counts, None, SCALE))
